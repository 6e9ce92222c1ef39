// Backward of the fused block norm (norm_residual.hip): from h, the sum r and the gradients dr, dn of r and n, with
// hhat, rhat the normalised rows (mean and 1 / sqrt(var + eps) taken again from the row in registers),
//
//   q  = dn * w_pre,    dR = dr + rstd_r (q - mean q - rhat mean(q rhat))         dx = dR
//   dp = s act(g) dR,   u = dp * w_post,  dh = rstd_h (u - mean u - hhat mean(u hhat))
//   dw_pre = sum dn rhat, db_pre = sum dn, dw_post = sum dp hhat, db_post = sum dp      (sums over rows)
//   dg = s act'(g) sum dR p,  ds = sum dR act(g) p                                       (rms: without the means)
//
// One pass: h, r, dr, dn are read once and dx, dh written once, a row in the registers of its lanes.  h and r may be 8-bit
// checkpoints, decoded as they are loaded.  A work-group keeps the sums over its rows in registers (fp32), adds its row
// groups' at the end through LDS and writes them to its own place of the workspace; a second launch adds those in a fixed
// order.  No atomics: results repeat bit for bit.  Bound by HBM.
#include "norm_residual.h"

namespace {

struct NormBwdParams {
    const char *h, *r, *dr, *dn, *gate;
    const unsigned char *h_scales, *r_scales;   // of checkpoints, or null: maps
    const float *post_w, *post_b, *pre_w, *scale_ptr;
    char *dx, *dh, *dgate;
    float* partial;                             // [work-groups][4 c + 4]: dw_post, db_post, dw_pre, db_pre, ds; or the results
    float* gate_partial;                        // [items][c]; or the result
    float *dpost_w, *dpost_b, *dpre_w, *dpre_b, *dscale;
    long long rows, rows_per_gate, seg_rows;    // an item is seg_rows rows of one gate's
    long long items;
    int segs;                                   // items per gate
    int c, groups, layer, post, pre, gate_mode, gate_f32, sigmoid, need_p, direct;
    float scale, eps, inv_c;
};

// Sums `acc` of the work-group's row groups, channel by channel, into out (times `factor` and, where the gate's activation
// is in the way, its derivative at the gate g).  Every thread calls it.
template <class C>
__device__ __forceinline__ void flush_rows(float* tile, const float* acc, float* out, const int c, const float factor, const float* gate,
                                           const bool sigmoid)
{
    const int t = threadIdx.x % C::TPR, rg = threadIdx.x / C::TPR;
    __syncthreads();   // the tile's last readers are done
#pragma unroll
    for (int v = 0; v < C::V; ++v)
#pragma unroll
        for (int k = 0; k < C::VEC; ++k) tile[rg * C::CMAX + (v * C::TPR + t) * C::VEC + k] = acc[v * C::VEC + k];
    __syncthreads();
    for (int i = threadIdx.x; i < C::CMAX && i < c; i += C::THREADS) {
        float s = tile[i];
        for (int k = 1; k < C::RPB; ++k) s += tile[k * C::CMAX + i];
        s *= factor;
        if (gate != nullptr && sigmoid) { const float g = sigmoid_f32(gate[i]); s *= g * (1.0f - g); }
        out[i] = s;
    }
}

template <class C, bool CK>
struct SavedRow {
    using T = typename C::T;
    rows_u32x4 q[C::V];
    // a row of a map, or of a checkpoint (words 0, 1: codes, word 3: scale byte)
    __device__ __forceinline__ void load(const char* p, const unsigned char* scales, const long long row, const int c, const int groups, const int* c0, const int* nv)
    {
        if (CK && scales != nullptr) {
#pragma unroll
            for (int v = 0; v < C::V; ++v) {
                const unsigned char* codes = (const unsigned char*)p + row * c + c0[v];
                unsigned w[2] = {0u, 0u};
                if (nv[v] >= C::VEC) __builtin_memcpy(w, codes, C::VEC);
                else
#pragma unroll
                    for (int k = 0; k < C::VEC; ++k)
                        if (k < nv[v]) w[k >> 2] |= (unsigned)codes[k] << (8 * (k & 3));
                q[v][0] = w[0]; q[v][1] = w[1]; q[v][2] = 0u;
                q[v][3] = nv[v] > 0 ? scales[row * groups + c0[v] / kCk8Group] : 0u;
            }
        } else {
#pragma unroll
            for (int v = 0; v < C::V; ++v) q[v] = load_row16<T>(p + (row * c + c0[v]) * RowVec<T>::SIZE, nv[v]);
        }
    }
    __device__ __forceinline__ void unpack(const unsigned char* scales, float* f) const
    {
        if (CK && scales != nullptr) {
#pragma unroll
            for (int v = 0; v < C::V; ++v)
#pragma unroll
                for (int k = 0; k < C::VEC / 4; ++k) ck8_unpack4(q[v][k], ck8_scale(q[v][3]), f + v * C::VEC + 4 * k);
        } else {
#pragma unroll
            for (int v = 0; v < C::V; ++v) RowVec<T>::unpack(q[v], f + v * C::VEC);
        }
    }
};

template <class C, bool CK>
__global__ __launch_bounds__(C::THREADS) void norm_residual_bwd_kernel(const NormBwdParams p)
{
    using T = typename C::T;
    constexpr int SIZE = RowVec<T>::SIZE, VEC = C::VEC, E = C::E;
    __shared__ float scratch[row_sum_scratch<C>()];
    __shared__ float tile[C::THREADS * E];
    RowSum<C> sum{scratch, 0};
    const int t = threadIdx.x % C::TPR, rg = threadIdx.x / C::TPR;
    int c0[C::V], nv[C::V];
    float wpost[E], bpost[E], wpre[E], g[E];
    float a_wpost[E], a_bpost[E], a_wpre[E], a_bpre[E], a_g[E], a_s = 0.0f;
#pragma unroll
    for (int v = 0; v < C::V; ++v) {
        c0[v] = (v * C::TPR + t) * VEC;
        nv[v] = p.c - c0[v];
        load_params<C>(p.post_w, c0[v], nv[v], 1.0f, wpost + v * VEC);
        load_params<C>(p.post_b, c0[v], nv[v], 0.0f, bpost + v * VEC);
        load_params<C>(p.pre_w, c0[v], nv[v], 1.0f, wpre + v * VEC);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) { g[j] = 1.0f; a_wpost[j] = a_bpost[j] = a_wpre[j] = a_bpre[j] = a_g[j] = 0.0f; }
    const float scale = p.scale_ptr ? *p.scale_ptr : p.scale;

    for (long long item = blockIdx.x; item < p.items; item += gridDim.x) {
        const long long s = item / p.segs;
        const long long r0 = s * p.rows_per_gate + (item - s * p.segs) * p.seg_rows;
        const long long r1 = r0 + p.seg_rows < (s + 1) * p.rows_per_gate ? r0 + p.seg_rows : (s + 1) * p.rows_per_gate;
        if (p.gate_mode == SRHIP_GATE_ROWS) {
#pragma unroll
            for (int v = 0; v < C::V; ++v) load_params<C>((const float*)p.gate + s * p.c, c0[v], nv[v], 0.0f, g + v * VEC);
            if (p.sigmoid)
#pragma unroll
                for (int j = 0; j < E; ++j) g[j] = sigmoid_f32(g[j]);
#pragma unroll
            for (int j = 0; j < E; ++j) a_g[j] = 0.0f;
        }
        for (long long base = r0; base < r1; base += C::RPB) {
            const bool live = base + rg < r1;
            const long long row = live ? base + rg : r1 - 1;   // lanes behind the item's last row work on it too and add nothing
            const long long at = row * p.c;
            SavedRow<C, CK> qh, qr;
            rows_u32x4 qdr[C::V], qdn[C::V], qg[C::V];
            if (p.need_p) qh.load(p.h, p.h_scales, row, p.c, p.groups, c0, nv);
            if (p.pre) {
                qr.load(p.r, p.r_scales, row, p.c, p.groups, c0, nv);
#pragma unroll
                for (int v = 0; v < C::V; ++v) qdn[v] = load_row16<T>(p.dn + (at + c0[v]) * SIZE, nv[v]);
            }
            if (p.dr)
#pragma unroll
                for (int v = 0; v < C::V; ++v) qdr[v] = load_row16<T>(p.dr + (at + c0[v]) * SIZE, nv[v]);
            if (p.gate_mode == SRHIP_GATE_MAP) {
                if (p.gate_f32) {
#pragma unroll
                    for (int v = 0; v < C::V; ++v) load_params<C>((const float*)p.gate + at, c0[v], nv[v], 0.0f, g + v * VEC);
                } else {
#pragma unroll
                    for (int v = 0; v < C::V; ++v) qg[v] = load_row16<T>(p.gate + (at + c0[v]) * SIZE, nv[v]);
#pragma unroll
                    for (int v = 0; v < C::V; ++v) RowVec<T>::unpack(qg[v], g + v * VEC);
                }
                if (p.sigmoid)
#pragma unroll
                    for (int j = 0; j < E; ++j) g[j] = sigmoid_f32(g[j]);
            }

            // ---- the norm behind the sum: dR
            float d[E];
#pragma unroll
            for (int j = 0; j < E; ++j) d[j] = 0.0f;
            if (p.pre) {
                float r[E], dn[E], mean, rstd, m1 = 0.0f, m2 = 0.0f;
                qr.unpack(p.r_scales, r);
#pragma unroll
                for (int v = 0; v < C::V; ++v) RowVec<T>::unpack(qdn[v], dn + v * VEC);
                row_statistics<C>(sum, r, nv, p.layer, p.inv_c, p.eps, mean, rstd);
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    r[j] = (r[j] - mean) * rstd;
                    if (live) { a_wpre[j] += dn[j] * r[j]; a_bpre[j] += dn[j]; }
                    d[j] = dn[j] * wpre[j];           // 0 where the channel does not exist
                    m1 += d[j];
                    m2 += d[j] * r[j];
                }
                sum.two(m1, m2);
                m1 = p.layer ? m1 * p.inv_c : 0.0f;
                m2 *= p.inv_c;
#pragma unroll
                for (int j = 0; j < E; ++j) d[j] = rstd * (d[j] - m1 - r[j] * m2);
            }
            if (p.dr) {
                float dr[E];
#pragma unroll
                for (int v = 0; v < C::V; ++v) RowVec<T>::unpack(qdr[v], dr + v * VEC);
#pragma unroll
                for (int j = 0; j < E; ++j) d[j] += dr[j];
            }
#pragma unroll
            for (int v = 0; v < C::V; ++v) {
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (k >= nv[v]) d[v * VEC + k] = 0.0f;
                if (live) store_row16<T>(p.dx + (at + c0[v]) * SIZE, RowVec<T>::pack(d + v * VEC), nv[v]);
            }
            if (!p.dh) continue;

            // ---- gate, scale and the norm in front of them: dh
            float h[E], mean = 0.0f, rstd = 1.0f;
            if (p.need_p) qh.unpack(p.h_scales, h);
            if (p.post) {
                row_statistics<C>(sum, h, nv, p.layer, p.inv_c, p.eps, mean, rstd);
#pragma unroll
                for (int j = 0; j < E; ++j) h[j] = (h[j] - mean) * rstd;
            }
            if (p.need_p) {
                float dg[E];
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    dg[j] = d[j] * (h[j] * wpost[j] + bpost[j]);   // dR p
                    if (live) a_s += j % VEC < nv[j / VEC] ? dg[j] * g[j] : 0.0f;
                }
                if (p.gate_mode == SRHIP_GATE_ROWS) {
                    if (live)
#pragma unroll
                        for (int j = 0; j < E; ++j) a_g[j] += dg[j];
                } else if (p.gate_mode == SRHIP_GATE_MAP) {
#pragma unroll
                    for (int j = 0; j < E; ++j) dg[j] *= scale * (p.sigmoid ? g[j] * (1.0f - g[j]) : 1.0f);
                    if (live) {
#pragma unroll
                        for (int v = 0; v < C::V; ++v) {
                            if (p.gate_f32) {
#pragma unroll
                                for (int k = 0; k < VEC; ++k)
                                    if (k < nv[v]) ((float*)p.dgate)[at + c0[v] + k] = dg[v * VEC + k];
                            } else {
                                store_row16<T>(p.dgate + (at + c0[v]) * SIZE, RowVec<T>::pack(dg + v * VEC), nv[v]);
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < E; ++j) d[j] *= scale * g[j];      // dp
            if (p.post) {
                float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    if (live) { a_wpost[j] += d[j] * h[j]; a_bpost[j] += d[j]; }
                    d[j] *= wpost[j];
                    m1 += d[j];
                    m2 += d[j] * h[j];
                }
                sum.two(m1, m2);
                m1 = p.layer ? m1 * p.inv_c : 0.0f;
                m2 *= p.inv_c;
#pragma unroll
                for (int j = 0; j < E; ++j) d[j] = rstd * (d[j] - m1 - h[j] * m2);
            }
            if (live)
#pragma unroll
                for (int v = 0; v < C::V; ++v) store_row16<T>(p.dh + (at + c0[v]) * SIZE, RowVec<T>::pack(d + v * VEC), nv[v]);
        }
        if (p.gate_mode == SRHIP_GATE_ROWS) {
            const bool whole = p.segs == 1;   // the item holds every row of its gate: the sum is the result
            flush_rows<C>(tile, a_g, p.gate_partial + item * p.c, p.c, whole ? scale : 1.0f, whole ? (const float*)p.gate + s * p.c : nullptr,
                          p.sigmoid);
        }
    }

    float* out = p.partial + (long long)blockIdx.x * (4 * p.c + 4);
    if (p.post) {
        flush_rows<C>(tile, a_wpost, p.direct ? p.dpost_w : out, p.c, 1.0f, nullptr, false);
        if (p.dpost_b) flush_rows<C>(tile, a_bpost, p.direct ? p.dpost_b : out + p.c, p.c, 1.0f, nullptr, false);
    }
    if (p.pre) {
        flush_rows<C>(tile, a_wpre, p.direct ? p.dpre_w : out + 2 * p.c, p.c, 1.0f, nullptr, false);
        if (p.dpre_b) flush_rows<C>(tile, a_bpre, p.direct ? p.dpre_b : out + 3 * p.c, p.c, 1.0f, nullptr, false);
    }
    if (p.dscale) {
        __syncthreads();
        a_s = lanes_sum<64>(a_s);
        if ((threadIdx.x & 63) == 0) tile[threadIdx.x >> 6] = a_s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int k = 1; k < C::THREADS / 64; ++k) a_s += tile[k];
            *(p.direct ? p.dscale : out + 4 * p.c) = a_s;
        }
    }
}

// Adds the work-groups' sums: 64 columns to a block, 16 thread groups taking every 16th partial, then their sums in order.
// Blocks: 4 vectors x ceil(c / 64), the scale's, then ceil(c / 64) for every gate of more than one item.
__global__ __launch_bounds__(1024) void norm_residual_bwd_sums_kernel(const NormBwdParams p, const int nwg, const int cblocks)
{
    __shared__ float red[16][64];
    const int col = threadIdx.x & 63, part = threadIdx.x >> 6;
    const float* src;
    float* dst;
    long long n = nwg, stride = 4ll * p.c + 4;
    float factor = 1.0f;
    const long long b = blockIdx.x;
    int ch;
    if (b < 4ll * cblocks) {
        const int which = (int)(b / cblocks);
        ch = (int)(b % cblocks) * 64 + col;
        dst = which == 0 ? p.dpost_w : which == 1 ? p.dpost_b : which == 2 ? p.dpre_w : p.dpre_b;
        src = p.partial + which * p.c;
    } else if (b == 4ll * cblocks) {
        ch = col == 0 ? 0 : p.c;   // one column
        dst = p.dscale;
        src = p.partial + 4 * p.c;
    } else {
        const long long s = (b - 4ll * cblocks - 1) / cblocks;
        ch = (int)((b - 4ll * cblocks - 1) % cblocks) * 64 + col;
        dst = (float*)p.dgate + s * p.c;
        src = p.gate_partial + s * p.segs * p.c;
        n = p.segs;
        stride = p.c;
        factor = p.scale_ptr ? *p.scale_ptr : p.scale;
        if (p.sigmoid && ch < p.c) { const float g = sigmoid_f32(((const float*)p.gate)[s * p.c + ch]); factor *= g * (1.0f - g); }
    }
    if (dst == nullptr) return;   // uniform over the block
    float s = 0.0f;
    if (ch < p.c)
#pragma unroll 4
        for (long long k = part; k < n; k += 16) s += src[k * stride + ch];
    red[part][col] = s;
    __syncthreads();
    if (part == 0 && ch < p.c) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += red[k][col];
        dst[ch] = s * factor;
    }
}

// How the rows are cut into items and work-groups: a function of the shape alone (and of the device's CUs), so that the
// workspace can be sized before the call.
struct Plan {
    long long items, seg_rows;
    int segs, grid, rpb, threads;
};
Plan plan_of(const srhip_norm_residual_bwd_args* a)
{
    Plan q;
    const int tpr = a->c <= 16 ? 2 : a->c <= 32 ? 4 : a->c <= 64 ? 8 : a->c <= 128 ? 16 : a->c <= 256 ? 32 : a->c <= 512 ? 64
                    : a->c <= 1024 ? 128 : a->c <= 2048 ? 256 : 512;
    q.threads = tpr <= 256 ? 256 : tpr;
    q.rpb = q.threads / tpr;
    const long long passes = (a->rows + q.rpb - 1) / q.rpb;
    const long long cus = srhip_num_cus(), resident = cus * (768 / q.threads > 0 ? 768 / q.threads : 1);
    // A work-group's partial sums (4 c floats written, and read again) weigh as much as one or two of its rows: eight
    // passes to a work-group at least, once every CU has one.
    long long grid = passes / 8;
    if (grid < cus) grid = passes < cus ? passes : cus;
    if (grid > resident) grid = resident;
    const long long gates = a->gate_mode == SRHIP_GATE_ROWS ? a->rows / a->rows_per_gate : 1;
    const long long per_gate = a->rows / gates;
    long long segs = (grid + gates - 1) / gates;
    const long long most = (per_gate + q.rpb - 1) / q.rpb;
    if (segs > most) segs = most;
    q.seg_rows = (((per_gate + segs - 1) / segs) + q.rpb - 1) / q.rpb * q.rpb;
    q.segs = (int)((per_gate + q.seg_rows - 1) / q.seg_rows);
    q.items = gates * q.segs;
    q.grid = (int)(q.items < grid ? q.items : grid);
    return q;
}

template <class C>
int launch(NormBwdParams p, const Plan& q, const long long gates, hipStream_t stream)
{
    if (p.h_scales || p.r_scales) hipLaunchKernelGGL((norm_residual_bwd_kernel<C, true>), dim3(q.grid), dim3(C::THREADS), 0, stream, p);
    else hipLaunchKernelGGL((norm_residual_bwd_kernel<C, false>), dim3(q.grid), dim3(C::THREADS), 0, stream, p);
    const int rc = srhip_check_launch("norm_residual_bwd_kernel");
    if (rc != SRHIP_OK || p.direct) return rc;   // one work-group (one item a gate) writes the results itself
    const int cblocks = srhip_div_up(p.c, 64);
    const bool gate_sums = p.gate_mode == SRHIP_GATE_ROWS && q.segs > 1;
    const long long blocks = 4ll * cblocks + 1 + (gate_sums ? gates * cblocks : 0);
    hipLaunchKernelGGL(norm_residual_bwd_sums_kernel, dim3((unsigned)blocks), dim3(1024), 0, stream, p, q.grid, cblocks);
    return srhip_check_launch("norm_residual_bwd_sums_kernel");
}

template <class T>
int dispatch(const NormBwdParams& p, const Plan& q, const long long gates, hipStream_t s)
{
    constexpr int K = 8 / RowVec<T>::VEC;   // vectors for 8 channels
    if (p.c <= 16) return launch<RowCfg<T, 2, K>>(p, q, gates, s);
    if (p.c <= 32) return launch<RowCfg<T, 4, K>>(p, q, gates, s);
    if (p.c <= 64) return launch<RowCfg<T, 8, K>>(p, q, gates, s);
    if (p.c <= 128) return launch<RowCfg<T, 16, K>>(p, q, gates, s);
    if (p.c <= 256) return launch<RowCfg<T, 32, K>>(p, q, gates, s);
    if (p.c <= 512) return launch<RowCfg<T, 64, K>>(p, q, gates, s);
    if (p.c <= 1024) return launch<RowCfg<T, 128, K>>(p, q, gates, s);
    if (p.c <= 2048) return launch<RowCfg<T, 256, K>>(p, q, gates, s);
    if (p.c <= 4096) return launch<RowCfg<T, 512, K>>(p, q, gates, s);
    return launch<RowCfg<T, 512, 2 * K>>(p, q, gates, s);
}

}  // namespace

static int bad_shape(const srhip_norm_residual_bwd_args* a)
{
    SRHIP_REQUIRE(a, "norm_residual_bwd: null pointer");
    SRHIP_REQUIRE(a->rows >= 0 && a->c >= 1 && a->c <= SRHIP_NORM_MAX_C, "norm_residual_bwd: bad shape (%lld rows of %d channels; 1 .. %d channels)", a->rows, a->c, SRHIP_NORM_MAX_C);
    SRHIP_REQUIRE(a->gate_mode >= SRHIP_GATE_NONE && a->gate_mode <= SRHIP_GATE_MAP, "norm_residual_bwd: unknown gate mode %d", a->gate_mode);
    SRHIP_REQUIRE(a->rows == 0 || a->gate_mode != SRHIP_GATE_ROWS || (a->rows_per_gate >= 1 && a->rows % a->rows_per_gate == 0), "norm_residual_bwd: %lld rows are not a multiple of %lld rows per gate", a->rows, a->rows_per_gate);
    return SRHIP_OK;
}

extern "C" {

SRHIP_API size_t srhip_norm_residual_bwd_workspace_bytes(const srhip_norm_residual_bwd_args* a)
{
    if (bad_shape(a) != SRHIP_OK || a->rows == 0) return 0;
    const Plan q = plan_of(a);
    return ((size_t)q.grid * (4 * (size_t)a->c + 4) + (a->gate_mode == SRHIP_GATE_ROWS && q.segs > 1 ? (size_t)q.items * a->c : 0)) * sizeof(float);
}

SRHIP_API int srhip_norm_residual_bwd(const srhip_norm_residual_bwd_args* a, void* stream)
{
    const int rc = bad_shape(a);
    if (rc != SRHIP_OK) return rc;
    SRHIP_REQUIRE(a->dtype == SRHIP_DT_BF16 || a->dtype == SRHIP_DT_F32, "norm_residual_bwd: unknown type %d", a->dtype);
    SRHIP_REQUIRE(a->kind == SRHIP_NORM_LAYER || a->kind == SRHIP_NORM_RMS, "norm_residual_bwd: unknown norm %d", a->kind);
    SRHIP_REQUIRE(a->eps >= 0.0f, "norm_residual_bwd: eps must not be negative");
    SRHIP_REQUIRE(a->rows >= 1, "norm_residual_bwd: no rows");
    SRHIP_REQUIRE(a->dx && (a->dr || a->pre), "norm_residual_bwd: null pointer");
    SRHIP_REQUIRE(!a->pre || (a->r && a->dn && a->pre_weight && a->dpre_weight), "norm_residual_bwd: the norm behind the sum needs r, dn, its weight and room for its gradient");
    SRHIP_REQUIRE(a->dh || (!a->post && a->gate_mode == SRHIP_GATE_NONE && !a->dscale), "norm_residual_bwd: a gate, a scale or a post norm without a branch");
    SRHIP_REQUIRE(!a->post || (a->post_weight && a->dpost_weight), "norm_residual_bwd: the post norm needs its weight and room for its gradient");
    SRHIP_REQUIRE(a->gate_mode == SRHIP_GATE_NONE || (a->gate && a->dgate), "norm_residual_bwd: null gate");
    const int need_p = a->dh && (a->post || a->gate_mode != SRHIP_GATE_NONE || a->dscale);
    SRHIP_REQUIRE(!need_p || a->h, "norm_residual_bwd: null branch");
    SRHIP_REQUIRE(a->workspace, "norm_residual_bwd: null workspace");
    const Plan q = plan_of(a);
    NormBwdParams p;
    p.h = (const char*)a->h; p.r = (const char*)a->r; p.dr = (const char*)a->dr; p.dn = (const char*)a->dn; p.gate = (const char*)a->gate;
    p.h_scales = (const unsigned char*)a->h_scales; p.r_scales = (const unsigned char*)a->r_scales;
    p.post_w = a->post ? a->post_weight : nullptr; p.post_b = a->post ? a->post_bias : nullptr; p.pre_w = a->pre ? a->pre_weight : nullptr;
    p.scale_ptr = a->scale_ptr;
    p.dx = (char*)a->dx; p.dh = (char*)a->dh; p.dgate = (char*)a->dgate;
    p.partial = (float*)a->workspace;
    p.gate_partial = q.segs > 1 ? p.partial + (size_t)q.grid * (4 * (size_t)a->c + 4) : (float*)a->dgate;
    p.dpost_w = a->post ? a->dpost_weight : nullptr; p.dpost_b = a->post ? a->dpost_bias : nullptr;
    p.dpre_w = a->pre ? a->dpre_weight : nullptr; p.dpre_b = a->pre ? a->dpre_bias : nullptr;
    p.dscale = a->dscale;
    p.rows = a->rows;
    p.rows_per_gate = a->gate_mode == SRHIP_GATE_ROWS ? a->rows_per_gate : a->rows;
    p.seg_rows = q.seg_rows; p.items = q.items; p.segs = q.segs;
    p.c = a->c; p.groups = srhip_div_up(a->c, kCk8Group); p.layer = a->kind == SRHIP_NORM_LAYER; p.post = a->post; p.pre = a->pre;
    p.gate_mode = a->gate_mode; p.gate_f32 = a->dtype != SRHIP_DT_F32 && a->gate_f32; p.sigmoid = a->gate_sigmoid;
    p.need_p = need_p; p.direct = q.grid == 1;
    p.scale = a->scale; p.eps = a->eps; p.inv_c = 1.0f / (float)a->c;
    const long long gates = a->rows / p.rows_per_gate;
    return a->dtype == SRHIP_DT_BF16 ? dispatch<__bf16>(p, q, gates, (hipStream_t)stream) : dispatch<float>(p, q, gates, (hipStream_t)stream);
}

}  // extern "C"
