// The row kernels of the fused block norm's backward pass for bf16 maps (norm_residual_bwd.h).
#include "norm_residual_bwd.h"

int srhip_norm::rows_bf16(int c, bool ck, bool mapg, const NormBwdParams* p, Plan& q, hipStream_t stream)
{
    return rows_of<__bf16, false>(c, ck, mapg, p, q, stream);
}
