// The row kernels of the fused block norm's backward pass for bf16 maps (norm_residual_bwd.h).
#include "norm_residual_bwd.h"

int srhip_norm::rows_bf16(const NormBwdParams& p, const Plan& q, hipStream_t stream) { return dispatch<__bf16>(p, q, stream); }
