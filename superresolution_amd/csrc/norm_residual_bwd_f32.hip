// The row kernels of the fused block norm's backward pass for fp32 maps (norm_residual_bwd.h).
#include "norm_residual_bwd.h"

int srhip_norm::rows_f32(const NormBwdParams& p, const Plan& q, hipStream_t stream) { return dispatch<float>(p, q, stream); }
