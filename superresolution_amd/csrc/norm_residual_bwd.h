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
#include <atomic>

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

// Gradient of a gate that is constant over rows, from their sums A1 and A0; f: scale times the derivative of its activation
__device__ __forceinline__ float gate_gradient(const NormBwdParams& p, const int ch, const float f, const float a1, const float a0)
{
    const float w = p.post_w ? p.post_w[ch] * a1 : a1;
    return f * (p.post_b ? w + p.post_b[ch] * a0 : w);   // (no bias: nothing is added, an infinite A0 does not matter)
}

// Adds `acc` over the work-group's row groups, channel by channel, and hands (channel, sum) to `put`; every thread calls it.
template <class C, class F>
__device__ __forceinline__ void sum_row_groups(float* tile, const Lane<C>& l, const float* acc, const int c, F&& put)
{
    if constexpr (C::RPB == 1) {
#pragma unroll
        for (int j = 0; j < C::E; ++j)
            if (l.mine(j)) put(l.c0[j / C::VEC] + j % C::VEC, acc[j]);
    } else {
        // the groups of one wave by lane moves, the waves (or, of wider rows, the groups) through LDS
        constexpr int PARTS = C::TPR <= 64 ? C::THREADS / 64 : C::RPB;
        const int part = C::TPR <= 64 ? threadIdx.x >> 6 : threadIdx.x / C::TPR;
        __syncthreads();   // the tile's last readers are done
#pragma unroll
        for (int j = 0; j < C::E; ++j) {
            const float v = C::TPR < 64 ? same_place_sum<C::TPR>(acc[j]) : acc[j];
            if ((C::TPR >= 64 || (threadIdx.x & 63) < C::TPR) && l.mine(j)) tile[part * C::CMAX + l.c0[j / C::VEC] + j % C::VEC] = v;
        }
        __syncthreads();
        for (int ch = threadIdx.x; ch < c; ch += C::THREADS) {
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
    rows_u32x4 q[C::V];
    // a lane's part of a row of a map, or of a checkpoint (words 0, 1: codes, word 3: scale byte)
    __device__ __forceinline__ void load(const char* p, const unsigned char* scales, const long long pass, const NormBwdParams& np, const Lane<C>& l, const unsigned back, const unsigned back_rows)
    {
        if (CK && scales != nullptr) {
            const unsigned char* codes = (const unsigned char*)p + pass * np.c;
            const unsigned char* sb = scales + pass * np.groups;
#pragma unroll
            for (int v = 0; v < C::V; ++v) {
                unsigned w[2] = {0u, 0u};
                __builtin_memcpy(w, codes + (size_t)(l.e[v] - back), C::VEC);
                q[v][0] = w[0]; q[v][1] = w[1];
                // (a vector that was moved to end with the row can lie across two groups: two scales)
                const unsigned sr = (l.rg - back_rows) * np.groups;
                q[v][3] = sb[(size_t)(sr + (unsigned)(l.c0[v] + C::VEC - 1) / kCk8Group)];
                q[v][2] = C::ODD ? sb[(size_t)(sr + (unsigned)l.c0[v] / kCk8Group)] : 0u;
            }
        } else {
            load_row<C>(p + pass * np.c * C::SIZE, l, back, q);
        }
    }
    __device__ __forceinline__ void unpack(const unsigned char* scales, const Lane<C>& l, float* f) const
    {
        if (CK && scales != nullptr) {
#pragma unroll
            for (int v = 0; v < C::V; ++v)
#pragma unroll
                for (int k = 0; k < C::VEC; k += 4) {
                    float g[4];
                    ck8_unpack4(q[v][k / 4], ck8_scale(q[v][3]), g);
                    if constexpr (C::ODD) {
                        float a[4];
                        ck8_unpack4(q[v][k / 4], ck8_scale(q[v][2]), a);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if ((l.c0[v] + k + i) / kCk8Group < (l.c0[v] + C::VEC - 1) / kCk8Group) g[i] = a[i];
                    }
#pragma unroll
                    for (int i = 0; i < 4 && k + i < C::VEC; ++i) f[v * C::VEC + k + i] = g[i];
                }
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
    // pass: first row; lanes behind the item's last row (`left` rows from the first on) work on it too and add nothing
    __device__ __forceinline__ void load(const NormBwdParams& p, const long long pass, const long long left, const Lane<C>& l)
    {
        const unsigned back_rows = l.rg < left ? 0u : (unsigned)(l.rg - (int)(left - 1)), back = back_rows * p.c;
        const long long at = pass * p.c * C::SIZE;
        if (p.need_h) h.load(p.h, p.h_scales, pass, p, l, back, back_rows);
        if (p.pre) {
            r.load(p.r, p.r_scales, pass, p, l, back, back_rows);
            load_row<C>(p.dn + at, l, back, dn);
        }
        if (p.dr) load_row<C>(p.dr + at, l, back, dr);
        if constexpr (MAPG)
            if (!p.gate_f32) load_row<C>(p.gate + at, l, back, g);
    }
};

// Waves to a SIMD that the registers are to leave room for: four of the kernel that decodes short bf16 rows (it needs 137
// registers left alone, and at 128, nine of them spilled, 64 channels of four crops take 587 us instead of 617), three with a
// gate map (two crops: 469 us instead of 532; of fp32 maps 138 us instead of 74, they are left alone), else what the compiler
// arrives at (the same on maps: 684 us for 681).
template <class C, bool CK, bool MAPG, bool SINGLE>
constexpr int min_waves() { return C::SIZE == 2 && C::TPR <= 64 && !SINGLE ? (MAPG ? 3 : CK ? 4 : 1) : 1; }

// SINGLE: a few rows, one item; its work-group writes the results and there is no second launch.  A kernel of its own: in the others
// these writes cost 4 to 28 registers, and fp32 rows of odd width with a gate map their second wave to a SIMD (3 x 135 x 241 rows
// of 99: 106 us instead of 73, from checkpoints 94 instead of 68).
template <class C, bool CK, bool MAPG, bool SINGLE>
__global__ __launch_bounds__(C::THREADS, (min_waves<C, CK, MAPG, SINGLE>())) void norm_residual_bwd_kernel(const NormBwdParams p)
{
    constexpr int SIZE = C::SIZE, VEC = C::VEC, E = C::E;
    __shared__ float scratch[row_sum_scratch<C>()];
    __shared__ float tile[row_groups_tile<C>()];
    RowSum<C> sum{scratch, 0};
    const Lane<C> l(p.c);
    float wpre[E], sw[E];   // sw: scale and gate, constant over an item, times the post norm's weight; of a gate map the weight alone
    float sb[MAPG ? E : 1]; // a gate map: the post norm's bias
    float a_w[E], a_b[E], a1[E], a0[E];
    load_params<C>(p.pre_w, l, 1.0f, wpre);
    const float scale = p.scale_ptr ? *p.scale_ptr : p.scale;
    if constexpr (MAPG) {
        load_params<C>(p.post_w, l, 1.0f, sw);
        load_params<C>(p.post_b, l, 0.0f, sb);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) a_w[j] = a_b[j] = 0.0f;

    for (long long item = blockIdx.x; item < p.items; item += gridDim.x) {
        const long long s = item / p.segs;
        const long long r0 = s * p.rows_per_gate + (item - s * p.segs) * p.seg_rows;
        const long long end = (s + 1) * p.rows_per_gate;
        const long long r1 = r0 + p.seg_rows < end ? r0 + p.seg_rows : end;
        // A work-group that holds one or two rows loads the next one ahead (16000 rows of 4096: 188 us, without 218), and so does
        // one that decodes (64 channels of four crops from checkpoints: 621 us, without 673).  Otherwise, with many rows in
        // flight, it gains nothing and costs registers; with 16 elements a lane there are none left for it.
        constexpr bool AHEAD = (C::TPR > 64 || CK) && E <= 8;
        RawRow<C, CK, MAPG> next;
        if (AHEAD) next.load(p, r0, r1 - r0, l);
        if constexpr (!MAPG) {
            load_params<C>(p.post_w, l, 1.0f, sw);
#pragma unroll
            for (int j = 0; j < E; ++j) sw[j] *= scale;
            if (p.gate_mode == SRHIP_GATE_ROWS) {
                float g[E];
                load_params<C>((const float*)p.gate + s * p.c, l, 0.0f, g);
#pragma unroll
                for (int j = 0; j < E; ++j) sw[j] *= p.sigmoid ? sigmoid_f32(g[j]) : g[j];
            }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) a1[j] = a0[j] = 0.0f;
        for (long long base = r0; base < r1; base += C::RPB) {
            const bool live = l.rg < r1 - base;
            const long long at = base * p.c * SIZE;
            if (!AHEAD) next.load(p, base, r1 - base, l);
            const RawRow<C, CK, MAPG> raw = next;
            if (AHEAD && base + C::RPB < r1) next.load(p, base + C::RPB, r1 - base - C::RPB, l);

            float r[E], h[E], d[E], rstd_r = 1.0f, rstd_h = 1.0f;
            if (p.pre) raw.r.unpack(p.r_scales, l, r);
            if (p.need_h) raw.h.unpack(p.h_scales, l, h);
            normalise<C>(sum, l, p.pre, r, p.post, h, p.layer, p.inv_c, p.eps, rstd_r, rstd_h);

            // ---- the norm behind the sum: dR
            if (p.dr) unpack_row<C>(raw.dr, d);
            else
#pragma unroll
                for (int j = 0; j < E; ++j) d[j] = 0.0f;
            if (p.pre) {
                float q[E];
                unpack_row<C>(raw.dn, q);
                if (live)
#pragma unroll
                    for (int j = 0; j < E; ++j) { a_w[j] += q[j] * r[j]; a_b[j] += q[j]; }
#pragma unroll
                for (int j = 0; j < E; ++j) q[j] *= wpre[j];
                float m1 = 0.0f, m2 = lane_sum<C>(l, [&](int j) { return q[j] * r[j]; });
                if (p.layer) m1 = lane_sum<C>(l, [&](int j) { return q[j]; });
                sum.two(m1, m2);
                m1 = -rstd_r * (m1 * p.inv_c);
                m2 = -rstd_r * (m2 * p.inv_c);
#pragma unroll
                for (int j = 0; j < E; ++j) d[j] = rstd_r * q[j] + (m2 * r[j] + (d[j] + m1));
            }
            if (live) store_row<C>(p.dx + at, l, d);
            if (!p.dh) continue;

            // ---- gate, scale and the norm in front of them: dh
            if constexpr (MAPG) {
                float g[E];
                if (p.gate_f32) load_gate_f32<C>(p.gate + base * p.c * 4, l, live ? 0u : (unsigned)((l.rg - (int)(r1 - base - 1)) * p.c), g);
                else unpack_row<C>(raw.g, g);
                if (p.sigmoid)
#pragma unroll
                    for (int j = 0; j < E; ++j) g[j] = sigmoid_f32(g[j]);
                float dg[E];
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    dg[j] = scale * d[j] * (h[j] * sw[j] + sb[j]);   // (the scale outside: an infinite one meets no bias of 0)
                    if (p.sigmoid) dg[j] *= g[j] * (1.0f - g[j]);
                    d[j] *= g[j];
                }
                if (live) {
                    if (p.gate_f32) {
#pragma unroll
                        for (int j = 0; j < E; ++j)
                            if (l.in[j / VEC]) ((float*)p.dgate + base * p.c)[l.e[j / VEC] + j % VEC] = dg[j];
                    } else {
                        store_row<C>(p.dgate + at, l, dg);
                    }
                }
            }
            if (p.need_h && live)
#pragma unroll
                for (int j = 0; j < E; ++j) { a1[j] += d[j] * h[j]; a0[j] += d[j]; }
#pragma unroll
            for (int j = 0; j < E; ++j) d[j] = MAPG ? d[j] * scale * sw[j] : d[j] * sw[j];
            if (p.post) {
                float m1 = 0.0f, m2 = lane_sum<C>(l, [&](int j) { return d[j] * h[j]; });
                if (p.layer) m1 = lane_sum<C>(l, [&](int j) { return d[j]; });
                sum.two(m1, m2);
                m1 = -rstd_h * (m1 * p.inv_c);
                m2 = -rstd_h * (m2 * p.inv_c);
#pragma unroll
                for (int j = 0; j < E; ++j) d[j] = rstd_h * d[j] + (m2 * h[j] + m1);
            }
            if (live) store_row<C>(p.dh + at, l, d);
        }
        if (p.item_flush) {
            float* out = p.item_sums + item * 2 * p.c;
            float part = 0.0f;
            sum_row_groups<C>(tile, l, a1, p.c, [&](const int ch, const float v) {
                float slope;
                const float gv = gate_value(p, s, ch, slope);
                out[ch] = v;
                if (p.dscale) part += v * gv * (p.post_w ? p.post_w[ch] : 1.0f);
                if constexpr (SINGLE)
                    if (p.dpost_w) p.dpost_w[ch] = scale * (gv * v);
            });
            sum_row_groups<C>(tile, l, a0, p.c, [&](const int ch, const float v) {
                float slope;
                const float gv = gate_value(p, s, ch, slope);
                out[p.c + ch] = v;
                if (p.dscale && p.post_b) part += v * gv * p.post_b[ch];
                if constexpr (SINGLE) {
                    if (p.dpost_b) p.dpost_b[ch] = scale * (gv * v);
                    if (p.gate_mode == SRHIP_GATE_ROWS)   // out[ch] is this thread's own
                        ((float*)p.dgate)[ch] = gate_gradient(p, ch, scale * slope, out[ch], v);
                }
            });
            if (p.dscale) {
                part = lanes_sum<64>(part);
                __syncthreads();
                if ((threadIdx.x & 63) == 0) tile[threadIdx.x >> 6] = part;
                __syncthreads();
                if (threadIdx.x == 0) {
                    for (int k = 1; k < C::THREADS / 64; ++k) part += tile[k];
                    *(SINGLE ? p.dscale : p.item_scale + item) = part;
                }
            }
        }
    }
    if (p.pre) {
        float* out = p.wg_sums + (long long)blockIdx.x * 2 * p.c;
        sum_row_groups<C>(tile, l, a_w, p.c, [&](const int ch, const float v) { (SINGLE ? p.dpre_w : out)[ch] = v; });
        sum_row_groups<C>(tile, l, a_b, p.c, [&](const int ch, const float v) {
            if (!SINGLE) out[p.c + ch] = v;
            else if (p.dpre_b) p.dpre_b[ch] = v;
        });
    }
}

// How the rows are cut into items and work-groups
struct Plan {
    long long items, seg_rows;
    int segs, grid, rpb;
};

// Calls f with the configuration of a row of c channels: the narrowest group of lanes that holds it.
template <class T, bool ODD, class F>
int with_rows(const int c, F&& f)
{
    constexpr int K = 8 / RowVec<T>::VEC;   // vectors for 8 channels
    if (ODD && c < RowVec<T>::VEC) return f(RowCfg<RowOne<T>, 8, 1, false>{});
    if (c <= 16) return f(RowCfg<RowVec<T>, 2, K, ODD>{});
    if (c <= 32) return f(RowCfg<RowVec<T>, 4, K, ODD>{});
    if (c <= 64) return f(RowCfg<RowVec<T>, 8, K, ODD>{});
    if (c <= 128) return f(RowCfg<RowVec<T>, 16, K, ODD>{});
    if (c <= 256) return f(RowCfg<RowVec<T>, 32, K, ODD>{});
    if (c <= 512) return f(RowCfg<RowVec<T>, 64, K, ODD>{});
    if (c <= 1024) return f(RowCfg<RowVec<T>, 128, K, ODD>{});
    if (c <= 2048) return f(RowCfg<RowVec<T>, 256, K, ODD>{});
    if (c <= 4096) return f(RowCfg<RowVec<T>, 512, K, ODD>{});
    return f(RowCfg<RowVec<T>, 512, 2 * K, ODD>{});
}

// How many work-groups of the call's kernel a CU holds, and their rows; asked of the runtime once per kernel and device.
template <class C, bool CK, bool MAPG>
void shape_of(Plan& q)
{
    static std::atomic<int> fit[kSrhipMaxDevices];
    const int dev = srhip_current_device();
    int n = fit[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, norm_residual_bwd_kernel<C, CK, MAPG, false>, C::THREADS, 0) != hipSuccess || n < 1) n = 1;
        fit[dev].store(n, std::memory_order_relaxed);
    }
    q.grid = n;
    q.rpb = C::RPB;
}
template <class C, bool CK, bool MAPG>
int shape_or_launch(const NormBwdParams* p, Plan& q, hipStream_t stream)
{
    if (p == nullptr) {
        shape_of<C, CK, MAPG>(q);
        return SRHIP_OK;
    }
    if (q.items == 1) hipLaunchKernelGGL((norm_residual_bwd_kernel<C, CK, MAPG, true>), dim3(1), dim3(C::THREADS), 0, stream, *p);
    else hipLaunchKernelGGL((norm_residual_bwd_kernel<C, CK, MAPG, false>), dim3(q.grid), dim3(C::THREADS), 0, stream, *p);
    return srhip_check_launch("norm_residual_bwd_kernel");
}
template <class T, bool ODD>
int rows_of(const int c, const bool ck, const bool mapg, const NormBwdParams* p, Plan& q, hipStream_t stream)
{
    return with_rows<T, ODD>(c, [&](auto cfg) {
        using C = decltype(cfg);
        if (ck) return mapg ? shape_or_launch<C, true, true>(p, q, stream) : shape_or_launch<C, true, false>(p, q, stream);
        return mapg ? shape_or_launch<C, false, true>(p, q, stream) : shape_or_launch<C, false, false>(p, q, stream);
    });
}

// Compiled side by side, by map type and whether channels come in whole vectors.  p null: the kernel's shape into q (grid =
// work-groups to a CU); otherwise its launch as q says.
int rows_bf16(int c, bool ck, bool mapg, const NormBwdParams* p, Plan& q, hipStream_t stream);
int rows_bf16_odd(int c, bool ck, bool mapg, const NormBwdParams* p, Plan& q, hipStream_t stream);
int rows_f32(int c, bool ck, bool mapg, const NormBwdParams* p, Plan& q, hipStream_t stream);
int rows_f32_odd(int c, bool ck, bool mapg, const NormBwdParams* p, Plan& q, hipStream_t stream);

}  // namespace srhip_norm
