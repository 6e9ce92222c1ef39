// Backward of the fused block norm (norm_residual.hip): from h, the sum r and the gradients dr, dn of r and n, with
// hhat, rhat the normalised rows (mean and 1 / sqrt(var + eps) taken again from the row in registers),
//
//   q  = dn * w_pre,    dR = dr + rstd_r (q - mean q - rhat mean(q rhat))         dx = dR
//   dp = s act(g) dR,   u = dp * w_post,  dh = rstd_h (u - mean u - hhat mean(u hhat))
//   dw_pre = sum dn rhat, db_pre = sum dn, dw_post = sum dp hhat, db_post = sum dp      (sums over rows)
//   dg = s act'(g) sum dR p,  ds = sum dR act(g) p                                       (rms: without the means)
//
// One pass: h, r, dr, dn are read once and dx, dh written once, a row in the registers of its lanes, the next row's loads
// under way meanwhile.  h and r may be 8-bit checkpoints, decoded as they are loaded.  A gate that is constant over an item's
// rows leaves the sums: with A1 = sum dR hhat and A0 = sum dR over the item,
//   dw_post = sum over items of s act(g) A1,  db_post: A0,  dg = s act'(g) (w A1 + b A0),  ds = sum over channels act(g) (w A1 + b A0)
// so that two sums per channel serve four gradients.  (A gate map: A1, A0 of act(g) dR; dg is written row by row.)
// A work-group keeps its sums in registers (fp32), adds its row groups' through LDS and writes them to its own place of the
// workspace; a second launch adds those in a fixed order.  No atomics: results repeat bit for bit.  Bound by HBM.
#pragma once
#include "norm_residual.h"

namespace srhip_norm {

struct NormBwdParams {
    const char *h, *r, *dr, *dn, *gate;
    const unsigned char *h_scales, *r_scales;   // of checkpoints, or null: maps
    const float *post_w, *post_b, *pre_w, *scale_ptr;
    char *dx, *dh, *dgate;
    float* wg_sums;                             // [work-groups][2][c]: dw_pre, db_pre
    float* item_sums;                           // [items][2][c]: A1, A0
    float* item_scale;                          // [items]: the item's part of ds
    float *dpost_w, *dpost_b, *dpre_w, *dpre_b, *dscale;
    long long rows, rows_per_gate, seg_rows;    // an item is seg_rows rows of one gate's
    long long items;
    int segs;                                   // items per gate
    int c, groups, layer, post, pre, gate_mode, gate_f32, sigmoid, need_h, item_flush;
    float scale, eps, inv_c;
};

// act(gate) of a channel, and its derivative
__device__ __forceinline__ float gate_value(const NormBwdParams& p, const long long s, const int ch, float& slope)
{
    slope = 1.0f;
    if (p.gate_mode != SRHIP_GATE_ROWS) return 1.0f;
    const float g = ((const float*)p.gate)[s * p.c + ch];
    if (!p.sigmoid) return g;
    const float a = sigmoid_f32(g);
    slope = a * (1.0f - a);
    return a;
}

// Adds `acc` over the work-group's row groups, channel by channel, and hands (channel, sum) to `put`; every thread calls it.
template <class C, class F>
__device__ __forceinline__ void sum_row_groups(float* tile, const float* acc, const int c, F&& put)
{
    const int t = threadIdx.x % C::TPR;
    if constexpr (C::RPB == 1) {
#pragma unroll
        for (int j = 0; j < C::E; ++j) {
            const int ch = (j / C::VEC * C::TPR + t) * C::VEC + j % C::VEC;
            if (ch < c) put(ch, acc[j]);
        }
    } else {
        // the groups of one wave by lane moves, the waves (or, of wider rows, the groups) through LDS
        constexpr int PARTS = C::TPR <= 64 ? C::THREADS / 64 : C::RPB;
        const int part = C::TPR <= 64 ? threadIdx.x >> 6 : threadIdx.x / C::TPR;
        __syncthreads();   // the tile's last readers are done
#pragma unroll
        for (int j = 0; j < C::E; ++j) {
            const float v = C::TPR < 64 ? same_place_sum<C::TPR>(acc[j]) : acc[j];
            if (C::TPR >= 64 || (threadIdx.x & 63) < C::TPR) tile[part * C::CMAX + (j / C::VEC * C::TPR + t) * C::VEC + j % C::VEC] = v;
        }
        __syncthreads();
        for (int ch = threadIdx.x; ch < C::CMAX && ch < c; ch += C::THREADS) {
            float s = tile[ch];
#pragma unroll
            for (int k = 1; k < PARTS; ++k) s += tile[k * C::CMAX + ch];
            put(ch, s);
        }
    }
}
template <class C>
constexpr int row_groups_tile() { return C::RPB == 1 ? C::THREADS / 64 : C::CMAX * (C::TPR <= 64 ? C::THREADS / 64 : C::RPB); }

template <class C, bool CK>
struct SavedRow {
    using T = typename C::T;
    rows_u32x4 q[C::V];
    // a row of a map, or of a checkpoint (words 0, 1: codes, word 3: scale byte)
    __device__ __forceinline__ void load(const char* p, const unsigned char* scales, const long long row, const int c, const int groups, const int* c0, const int* nv, const bool whole)
    {
        if (CK && scales != nullptr) {
            const unsigned char* codes = (const unsigned char*)p + row * c;
            const unsigned char* sb = scales + row * groups;
#pragma unroll
            for (int v = 0; v < C::V; ++v) {
                unsigned w[2] = {0u, 0u};
                if (whole || nv[v] >= C::VEC) __builtin_memcpy(w, codes + c0[v], C::VEC);
                else
#pragma unroll
                    for (int k = 0; k < C::VEC; ++k)
                        if (k < nv[v]) w[k >> 2] |= (unsigned)codes[c0[v] + k] << (8 * (k & 3));
                q[v][0] = w[0]; q[v][1] = w[1]; q[v][2] = 0u;
                q[v][3] = whole || nv[v] > 0 ? sb[c0[v] / kCk8Group] : 0u;
            }
        } else {
            load_row<C>(p + row * c * RowVec<T>::SIZE, c0, nv, whole, q);
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
            unpack_row<C>(q, f);
        }
    }
};

// what a lane reads of a row
template <class C, bool CK, bool MAPG>
struct RawRow {
    SavedRow<C, CK> h, r;
    rows_u32x4 dr[C::V], dn[C::V], g[MAPG ? C::V : 1];
    __device__ __forceinline__ void load(const NormBwdParams& p, const long long row, const int* c0, const int* nv, const bool whole)
    {
        const long long at = row * p.c * RowVec<typename C::T>::SIZE;
        if (p.need_h) h.load(p.h, p.h_scales, row, p.c, p.groups, c0, nv, whole);
        if (p.pre) {
            r.load(p.r, p.r_scales, row, p.c, p.groups, c0, nv, whole);
            load_row<C>(p.dn + at, c0, nv, whole, dn);
        }
        if (p.dr) load_row<C>(p.dr + at, c0, nv, whole, dr);
        if constexpr (MAPG)
            if (!p.gate_f32) load_row<C>(p.gate + at, c0, nv, whole, g);
    }
};

template <class C, bool CK, bool MAPG>
__global__ __launch_bounds__(C::THREADS) void norm_residual_bwd_kernel(const NormBwdParams p)
{
    using T = typename C::T;
    constexpr int SIZE = RowVec<T>::SIZE, VEC = C::VEC, E = C::E;
    __shared__ float scratch[row_sum_scratch<C>()];
    __shared__ float tile[row_groups_tile<C>()];
    RowSum<C> sum{scratch, 0};
    const int t = threadIdx.x % C::TPR, rg = threadIdx.x / C::TPR;
    const bool whole = p.c == C::CMAX;
    int c0[C::V], nv[C::V];
#pragma unroll
    for (int v = 0; v < C::V; ++v) {
        c0[v] = (v * C::TPR + t) * VEC;
        nv[v] = p.c - c0[v];
    }
    float wpre[E], sw[E];   // sw: scale (and, constant over an item, the gate) times the post norm's weight
    float sb[MAPG ? E : 1];
    float a_w[E], a_b[E], a1[E], a0[E];
    load_params<C>(p.pre_w, c0, nv, 1.0f, wpre);
    const float scale = p.scale_ptr ? *p.scale_ptr : p.scale;
    if constexpr (MAPG) {
        load_params<C>(p.post_w, c0, nv, 1.0f, sw);
        load_params<C>(p.post_b, c0, nv, 0.0f, sb);
#pragma unroll
        for (int j = 0; j < E; ++j) { sw[j] *= scale; sb[j] *= scale; }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) a_w[j] = a_b[j] = 0.0f;

    for (long long item = blockIdx.x; item < p.items; item += gridDim.x) {
        const long long s = item / p.segs;
        const long long r0 = s * p.rows_per_gate + (item - s * p.segs) * p.seg_rows;
        const long long end = (s + 1) * p.rows_per_gate;
        const long long r1 = r0 + p.seg_rows < end ? r0 + p.seg_rows : end;
        // the next row's loads run ahead of the row at work, but where 16 elements a lane leave no registers for them
        constexpr bool AHEAD = E <= 8;
        RawRow<C, CK, MAPG> next;
        // lanes behind the item's last row work on it too and add nothing
        if (AHEAD) next.load(p, r0 + rg < r1 ? r0 + rg : r1 - 1, c0, nv, whole);
        if constexpr (!MAPG) {
            load_params<C>(p.post_w, c0, nv, 1.0f, sw);
#pragma unroll
            for (int j = 0; j < E; ++j) sw[j] *= scale;
            if (p.gate_mode == SRHIP_GATE_ROWS) {
                float g[E];
                load_params<C>((const float*)p.gate + s * p.c, c0, nv, 0.0f, g);
#pragma unroll
                for (int j = 0; j < E; ++j) sw[j] *= p.sigmoid ? sigmoid_f32(g[j]) : g[j];
            }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) a1[j] = a0[j] = 0.0f;
        for (long long base = r0; base < r1; base += C::RPB) {
            const bool live = base + rg < r1;
            const long long row = live ? base + rg : r1 - 1;
            const long long at = row * p.c * SIZE;
            if (!AHEAD) next.load(p, row, c0, nv, whole);
            const RawRow<C, CK, MAPG> raw = next;
            if (AHEAD && base + C::RPB < r1) next.load(p, base + C::RPB + rg < r1 ? base + C::RPB + rg : r1 - 1, c0, nv, whole);

            float r[E], h[E], d[E], rstd_r = 1.0f, rstd_h = 1.0f;
            if (p.pre) raw.r.unpack(p.r_scales, r);
            if (p.need_h) raw.h.unpack(p.h_scales, h);
            normalise<C>(sum, p.pre, r, p.post, h, nv, p.layer, p.inv_c, p.eps, rstd_r, rstd_h);

            // ---- the norm behind the sum: dR
#pragma unroll
            for (int j = 0; j < E; ++j) d[j] = 0.0f;
            if (p.dr) unpack_row<C>(raw.dr, d);
            if (p.pre) {
                float q[E], m1 = 0.0f, m2 = 0.0f;
                unpack_row<C>(raw.dn, q);
                if (live)
#pragma unroll
                    for (int j = 0; j < E; ++j) { a_w[j] += q[j] * r[j]; a_b[j] += q[j]; }
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    q[j] *= wpre[j];
                    m1 += q[j];
                    m2 += q[j] * r[j];
                }
                sum.two(m1, m2);
                m1 = p.layer ? -rstd_r * (m1 * p.inv_c) : 0.0f;
                m2 = -rstd_r * (m2 * p.inv_c);
#pragma unroll
                for (int j = 0; j < E; ++j) d[j] = rstd_r * q[j] + (m2 * r[j] + (d[j] + m1));
                zero_absent<C>(d, nv);
            }
            if (live) store_row<C>(p.dx + at, c0, nv, whole, d);
            if (!p.dh) continue;

            // ---- gate, scale and the norm in front of them: dh
            if constexpr (MAPG) {
                float g[E];
                if (p.gate_f32) load_gate_f32<C>(p.gate + row * p.c * 4, c0, nv, g);
                else unpack_row<C>(raw.g, g);
                if (p.sigmoid)
#pragma unroll
                    for (int j = 0; j < E; ++j) g[j] = sigmoid_f32(g[j]);
                float dg[E];
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    dg[j] = d[j] * (h[j] * sw[j] + sb[j]);
                    if (p.sigmoid) dg[j] *= g[j] * (1.0f - g[j]);
                    d[j] *= g[j];
                }
                if (live) {
                    if (p.gate_f32) {
#pragma unroll
                        for (int j = 0; j < E; ++j)
                            if (j % VEC < nv[j / VEC]) ((float*)p.dgate)[row * p.c + c0[j / VEC] + j % VEC] = dg[j];
                    } else {
                        store_row<C>(p.dgate + at, c0, nv, whole, dg);
                    }
                }
            }
            if (p.need_h && live)
#pragma unroll
                for (int j = 0; j < E; ++j) { a1[j] += d[j] * h[j]; a0[j] += d[j]; }
#pragma unroll
            for (int j = 0; j < E; ++j) d[j] *= sw[j];
            if (p.post) {
                float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    m1 += d[j];
                    m2 += d[j] * h[j];
                }
                sum.two(m1, m2);
                m1 = p.layer ? -rstd_h * (m1 * p.inv_c) : 0.0f;
                m2 = -rstd_h * (m2 * p.inv_c);
#pragma unroll
                for (int j = 0; j < E; ++j) d[j] = rstd_h * d[j] + (m2 * h[j] + m1);
            }
            if (live) store_row<C>(p.dh + at, c0, nv, whole, d);
        }
        if (p.item_flush) {
            float* out = p.item_sums + item * 2 * p.c;
            float part = 0.0f;
            sum_row_groups<C>(tile, a1, p.c, [&](const int ch, const float v) {
                float slope;
                out[ch] = v;
                if (p.dscale) part += v * gate_value(p, s, ch, slope) * (p.post_w ? p.post_w[ch] : 1.0f);
            });
            sum_row_groups<C>(tile, a0, p.c, [&](const int ch, const float v) {
                float slope;
                out[p.c + ch] = v;
                if (p.dscale && p.post_b) part += v * gate_value(p, s, ch, slope) * p.post_b[ch];
            });
            if (p.dscale) {
                part = lanes_sum<64>(part);
                __syncthreads();
                if ((threadIdx.x & 63) == 0) tile[threadIdx.x >> 6] = part;
                __syncthreads();
                if (threadIdx.x == 0) {
                    for (int k = 1; k < C::THREADS / 64; ++k) part += tile[k];
                    p.item_scale[item] = part;
                }
            }
        }
    }
    if (p.pre) {
        float* out = p.wg_sums + (long long)blockIdx.x * 2 * p.c;
        sum_row_groups<C>(tile, a_w, p.c, [&](const int ch, const float v) { out[ch] = v; });
        sum_row_groups<C>(tile, a_b, p.c, [&](const int ch, const float v) { out[p.c + ch] = v; });
    }
}

// How the rows are cut into items and work-groups
struct Plan {
    long long items, seg_rows;
    int segs, grid, rpb, threads;
};

template <class C, bool CK>
void launch_rows(const NormBwdParams& p, const Plan& q, hipStream_t stream)
{
    if (p.gate_mode == SRHIP_GATE_MAP) hipLaunchKernelGGL((norm_residual_bwd_kernel<C, CK, true>), dim3(q.grid), dim3(C::THREADS), 0, stream, p);
    else hipLaunchKernelGGL((norm_residual_bwd_kernel<C, CK, false>), dim3(q.grid), dim3(C::THREADS), 0, stream, p);
}
template <class C>
int launch(const NormBwdParams& p, const Plan& q, hipStream_t stream)
{
    if (p.h_scales || p.r_scales) launch_rows<C, true>(p, q, stream);
    else launch_rows<C, false>(p, q, stream);
    return srhip_check_launch("norm_residual_bwd_kernel");
}

template <class T>
int dispatch(const NormBwdParams& p, const Plan& q, hipStream_t s)
{
    constexpr int K = 8 / RowVec<T>::VEC;   // vectors for 8 channels
    if (p.c <= 16) return launch<RowCfg<T, 2, K>>(p, q, s);
    if (p.c <= 32) return launch<RowCfg<T, 4, K>>(p, q, s);
    if (p.c <= 64) return launch<RowCfg<T, 8, K>>(p, q, s);
    if (p.c <= 128) return launch<RowCfg<T, 16, K>>(p, q, s);
    if (p.c <= 256) return launch<RowCfg<T, 32, K>>(p, q, s);
    if (p.c <= 512) return launch<RowCfg<T, 64, K>>(p, q, s);
    if (p.c <= 1024) return launch<RowCfg<T, 128, K>>(p, q, s);
    if (p.c <= 2048) return launch<RowCfg<T, 256, K>>(p, q, s);
    if (p.c <= 4096) return launch<RowCfg<T, 512, K>>(p, q, s);
    return launch<RowCfg<T, 512, 2 * K>>(p, q, s);
}

// the two map types are compiled side by side
int rows_bf16(const NormBwdParams& p, const Plan& q, hipStream_t stream);
int rows_f32(const NormBwdParams& p, const Plan& q, hipStream_t stream);

}  // namespace srhip_norm
