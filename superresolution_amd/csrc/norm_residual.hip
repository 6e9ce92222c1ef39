// The norms around a residual block, with its gate and residual scale, in one pass over the rows of a channels-last map:
//
//   p = N_post(h) = (h - mean h) / sqrt(var h + eps) * w + b          (layer; rms: h / sqrt(mean h^2 + eps) * w; none: h)
//   r = x + s * act(g) * p                                            (the residual sum: what the next block adds to)
//   n = N_pre(r)                                                      (what the next block reads)
//
// Layer by layer this is LayerNorm (core/arch/CAMixerSR.py:29-37), a gated map (core/arch/RepRFN.py:233-235), a scaled
// residual sum (core/models/model.py:33) and LayerNorm again: ten passes over maps of which four or five are left.
// n is the norm of the unrounded sum.  All arithmetic in fp32, each output rounded once.
//
// Bound by HBM: x, h (and a gate map) are read once, r and n written once, a row stays in the registers of its lanes.
#include <atomic>

#include "norm_residual.h"

namespace {

struct NormParams {
    const char* x;
    const char* h;
    const char* gate;
    const float *post_w, *post_b, *pre_w, *pre_b, *scale_ptr;
    char* r;
    char* n;
    long long rows, rows_per_gate;
    long long wg_rows, wg_step;   // a work-group takes wg_rows rows, or (wg_step > 0) wg_rows of every wg_step
    int c, layer, post, pre, gate_mode, gate_f32, sigmoid;
    float scale, eps, inv_c;
};

// MAPG: the gate is a map.  Otherwise it is constant over runs of rows and held, times the scale, in registers.  It multiplies the
// norm's result, weight and bias together, not the two on their own: an infinite gate is then an infinite term, as in the formula,
// and not infinity times a bias of 0 or the difference of two infinities.
template <class C, bool MAPG>
__global__ __launch_bounds__(C::THREADS) void norm_residual_kernel(const NormParams p)
{
    constexpr int SIZE = C::SIZE, E = C::E;
    __shared__ float scratch[row_sum_scratch<C>()];
    RowSum<C> sum{scratch, 0};
    const Lane<C> l(p.c);
    float wpost[E], bpost[E], wpre[E], bpre[E], g[E];   // g: scale times gate
    load_params<C>(p.pre_w, l, 1.0f, wpre);
    load_params<C>(p.pre_b, l, 0.0f, bpre);
    load_params<C>(p.post_w, l, 1.0f, wpost);
    load_params<C>(p.post_b, l, 0.0f, bpost);
    const float scale = p.scale_ptr ? *p.scale_ptr : p.scale;
    long long gate_end = 0;   // first row that the gate held in registers does not belong to
#pragma unroll
    for (int j = 0; j < E; ++j) g[j] = scale;

    const long long first = blockIdx.x * p.wg_rows, last = p.wg_step || p.wg_rows > p.rows - first ? p.rows : first + p.wg_rows;
    for (long long base = first; base < last; base += p.wg_step ? p.wg_step : C::RPB) {
        // lanes behind the last row work on it too and store nothing
        const bool live = l.rg < p.rows - base;
        const unsigned back = live ? 0u : (unsigned)((l.rg - (int)(p.rows - base - 1)) * p.c);
        const long long at = base * p.c * SIZE;
        rows_u32x4 qx[C::V], qh[C::V], qg[C::V];
        load_row<C>(p.x + at, l, back, qx);
        if (p.h) load_row<C>(p.h + at, l, back, qh);
        if constexpr (MAPG) {
            if (p.gate_f32) load_gate_f32<C>(p.gate + base * p.c * 4, l, back, g);
            else load_row<C>(p.gate + at, l, back, qg);
        } else if (p.gate_mode == SRHIP_GATE_ROWS && live && base + l.rg >= gate_end) {   // rows of a lane only grow
            const long long s = (base + l.rg) / p.rows_per_gate;
            gate_end = (s + 1) * p.rows_per_gate;
            load_params<C>((const float*)p.gate + s * p.c, l, 0.0f, g);
#pragma unroll
            for (int j = 0; j < E; ++j) g[j] = scale * (p.sigmoid ? sigmoid_f32(g[j]) : g[j]);
        }

        float r[E];
        unpack_row<C>(qx, r);
        if (p.h) {
            float h[E];
            unpack_row<C>(qh, h);
            if (p.post) normalise<C>(sum, l, h, p.layer, p.inv_c, p.eps);
            if constexpr (MAPG) {
                if (!p.gate_f32) unpack_row<C>(qg, g);
                if (p.sigmoid)
#pragma unroll
                    for (int j = 0; j < E; ++j) g[j] = sigmoid_f32(g[j]);
#pragma unroll
                for (int j = 0; j < E; ++j) g[j] *= scale;
            }
#pragma unroll
            for (int j = 0; j < E; ++j) r[j] += g[j] * (h[j] * wpost[j] + bpost[j]);
            if (live) store_row<C>(p.r + at, l, r);
        }
        if (p.pre) {
            normalise<C>(sum, l, r, p.layer, p.inv_c, p.eps);
#pragma unroll
            for (int j = 0; j < E; ++j) r[j] = r[j] * wpre[j] + bpre[j];
            if (live) store_row<C>(p.n + at, l, r);
        }
    }
}

template <class C, bool MAPG>
int launch_rows(NormParams p, hipStream_t stream)
{
    const long long passes = (p.rows + C::RPB - 1) / C::RPB;
    long long grid;
    if (C::TPR <= 64 && C::E <= 8) {
        // Short rows: eight passes to a work-group, enough to pay for its parameters, and as many work-groups as that makes
        // (64 channels of four 1024^2 crops: 389 us; 4, 16, 32 passes 436, 412, 433 us; work-groups that stay resident and
        // stride over the rows 432 us).  A launch has fewer than 2^32 threads: of more rows (2^32 of one channel) more to a work-group.
        constexpr long long kMost = (1ll << 32) / C::THREADS - 1;
        const long long per = passes <= 8 * kMost ? 8 : (passes + kMost - 1) / kMost;
        p.wg_rows = per * C::RPB;
        p.wg_step = 0;
        grid = (passes + per - 1) / per;
    } else {
        // Long rows: the work-groups that fit the device at once stride over the rows (16000 rows of 4096: 108 us, of eight
        // rows to a work-group 125 us: the last of them leave the device half empty).
        static std::atomic<int> fit[kSrhipMaxDevices];
        const int dev = srhip_current_device();
        int n = fit[dev].load(std::memory_order_relaxed);
        if (n == 0) {
            if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, norm_residual_kernel<C, MAPG>, C::THREADS, 0) != hipSuccess || n < 1) n = 1;
            fit[dev].store(n, std::memory_order_relaxed);
        }
        grid = (long long)srhip_num_cus() * n < passes ? (long long)srhip_num_cus() * n : passes;
        p.wg_rows = C::RPB;
        p.wg_step = grid * C::RPB;
    }
    hipLaunchKernelGGL((norm_residual_kernel<C, MAPG>), dim3((unsigned)grid), dim3(C::THREADS), 0, stream, p);
    return srhip_check_launch("norm_residual_kernel");
}
template <class C>
int launch(const NormParams& p, hipStream_t stream)
{
    return p.gate_mode == SRHIP_GATE_MAP ? launch_rows<C, true>(p, stream) : launch_rows<C, false>(p, stream);
}

// the narrowest group of lanes that holds a row
template <class T, bool ODD>
int dispatch(const NormParams& p, hipStream_t s)
{
    constexpr int K = 8 / RowVec<T>::VEC;   // vectors for 8 channels
    if (ODD && p.c < RowVec<T>::VEC) return launch<RowCfg<RowOne<T>, 8, 1, false>>(p, s);
    if (p.c <= 16) return launch<RowCfg<RowVec<T>, 2, K, ODD>>(p, s);
    if (p.c <= 32) return launch<RowCfg<RowVec<T>, 4, K, ODD>>(p, s);
    if (p.c <= 64) return launch<RowCfg<RowVec<T>, 8, K, ODD>>(p, s);
    if (p.c <= 128) return launch<RowCfg<RowVec<T>, 16, K, ODD>>(p, s);
    if (p.c <= 256) return launch<RowCfg<RowVec<T>, 32, K, ODD>>(p, s);
    if (p.c <= 512) return launch<RowCfg<RowVec<T>, 64, K, ODD>>(p, s);
    if (p.c <= 1024) return launch<RowCfg<RowVec<T>, 64, 2 * K, ODD>>(p, s);
    if (p.c <= 2048) return launch<RowCfg<RowVec<T>, 256, K, ODD>>(p, s);
    if (p.c <= 4096) return launch<RowCfg<RowVec<T>, 256, 2 * K, ODD>>(p, s);
    return launch<RowCfg<RowVec<T>, 512, 2 * K, ODD>>(p, s);
}
template <class T>
int dispatch(const NormParams& p, hipStream_t s)
{
    return p.c % RowVec<T>::VEC ? dispatch<T, true>(p, s) : dispatch<T, false>(p, s);
}

}  // namespace

extern "C" SRHIP_API int srhip_norm_residual_fwd(const srhip_norm_residual_args* a, void* stream)
{
    SRHIP_REQUIRE(a, "norm_residual: null pointer");
    SRHIP_REQUIRE(a->rows >= 0 && a->c >= 1 && a->c <= SRHIP_NORM_MAX_C, "norm_residual: bad shape (%lld rows of %d channels; 1 .. %d channels)", a->rows, a->c, SRHIP_NORM_MAX_C);
    SRHIP_REQUIRE(a->dtype == SRHIP_DT_BF16 || a->dtype == SRHIP_DT_F32, "norm_residual: unknown type %d", a->dtype);
    SRHIP_REQUIRE(a->kind == SRHIP_NORM_LAYER || a->kind == SRHIP_NORM_RMS, "norm_residual: unknown norm %d", a->kind);
    SRHIP_REQUIRE(a->gate_mode >= SRHIP_GATE_NONE && a->gate_mode <= SRHIP_GATE_MAP, "norm_residual: unknown gate mode %d", a->gate_mode);
    SRHIP_REQUIRE(a->eps >= 0.0f, "norm_residual: eps must not be negative");
    if (a->rows == 0) return SRHIP_OK;   // (pointers of empty maps may be null)
    SRHIP_REQUIRE(a->h || a->pre, "norm_residual: neither a branch nor a norm behind the sum");
    SRHIP_REQUIRE(a->h || (!a->post && a->gate_mode == SRHIP_GATE_NONE), "norm_residual: a gate or a post norm without a branch");
    SRHIP_REQUIRE(a->x && (!a->h || a->r) && (!a->pre || (a->n && a->pre_weight)) && (!a->post || a->post_weight), "norm_residual: null pointer");
    SRHIP_REQUIRE(a->gate_mode == SRHIP_GATE_NONE || a->gate, "norm_residual: null gate");
    SRHIP_REQUIRE(a->gate_mode != SRHIP_GATE_ROWS || (a->rows_per_gate >= 1 && a->rows % a->rows_per_gate == 0), "norm_residual: %lld rows are not a multiple of %lld rows per gate", a->rows, a->rows_per_gate);
    NormParams p;
    p.x = (const char*)a->x; p.h = (const char*)a->h; p.gate = (const char*)a->gate;
    p.post_w = a->post ? a->post_weight : nullptr; p.post_b = a->post ? a->post_bias : nullptr;
    p.pre_w = a->pre ? a->pre_weight : nullptr; p.pre_b = a->pre ? a->pre_bias : nullptr;
    p.scale_ptr = a->scale_ptr;
    p.r = (char*)a->r; p.n = (char*)a->n;
    p.rows = a->rows; p.rows_per_gate = a->rows_per_gate;
    p.c = a->c; p.layer = a->kind == SRHIP_NORM_LAYER; p.post = a->post; p.pre = a->pre;
    p.gate_mode = a->gate_mode; p.gate_f32 = a->dtype != SRHIP_DT_F32 && a->gate_f32; p.sigmoid = a->gate_sigmoid;
    p.scale = a->scale; p.eps = a->eps; p.inv_c = 1.0f / (float)a->c;
    return a->dtype == SRHIP_DT_BF16 ? dispatch<__bf16>(p, (hipStream_t)stream) : dispatch<float>(p, (hipStream_t)stream);
}
