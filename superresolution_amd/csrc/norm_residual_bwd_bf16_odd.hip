// The row kernels of the fused block norm's backward pass for bf16 maps whose channel count is no multiple of a vector (norm_residual_bwd.h).
#include "norm_residual_bwd.h"

int srhip_norm::rows_bf16_odd(int c, bool ck, bool mapg, const NormBwdParams* p, Plan& q, hipStream_t stream)
{
    return rows_of<__bf16, true>(c, ck, mapg, p, q, stream);
}
