// The row kernels of the fused block norm's backward pass for fp32 maps (norm_residual_bwd.h).
#include "norm_residual_bwd.h"

int srhip_norm::rows_f32(int c, bool ck, bool mapg, const NormBwdParams* p, Plan& q, hipStream_t stream)
{
    return rows_of<float, false>(c, ck, mapg, p, q, stream);
}
