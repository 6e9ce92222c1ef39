// Weight gradient of a pointwise layer (1x1 convolution, core/models/model_final.py:237-246 under loss.backward()) of any width
// as one GEMM over the pixels, from an 8-bit checkpoint of its input or from the bf16 map itself:
//
//   dW[co][ci] = sum over pixels of dz[pixel][co] * x[pixel][ci],    db[co] = sum over pixels of dz[pixel][co]
//
// Few outputs (cout x cin), a long contraction (up to millions of pixels), both operands pixel-major: a work-group takes a
// 128 x 128 block of outputs and a run of pixels, so that every map is read once per 128 channels of the other one.  32 pixels
// at a time travel HBM -> registers, a step ahead of LDS (two steps ahead measured the same); codes are decoded there, once, to bf16 (exact); then
// to one of two LDS buffers, from which ds_read_b64_tr_b16 takes the MFMA operands (8 pixels of one channel to a lane).  Four
// waves own 64 x 64 outputs each (2 x 2 tiles of 32 x 32: four operand reads for four MFMAs, LDS and matrix unit even).
// LDS rows are 288 bytes, so that the four rows of a transposing read lie in different banks.
//
// The runs' partial blocks (fp32) are added by a second launch in a fixed order; a single run writes the result.
// Measured from checkpoints, beside the centre tap of conv3x3_wgrad.hip with its 64 x 64 slice pairs: 160 -> 112 channels, 65 k
// pixels 21 us (49), a million 109 us = 3.6 TB/s (262); 256 -> 192, a million 204 us = 3.3 TB/s (485).  Short maps are bound by
// their few dependent steps and the partial sums (65 k pixels: nine steps and 16 MB, 16 us, and 5 us for the launch that adds
// them), long ones by the LDS traffic of the operand reads beside HBM.
#include "rows_util.h"

namespace {

constexpr int kBlock = 128, kStep = 32, kRow = 288;   // outputs of a block's side, pixels of a step, bytes of an LDS row
constexpr int kThreads = 256;
typedef __attribute__((ext_vector_type(8))) __bf16 pw_bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 pw_bf16x4;

struct PwParams {
    const char *x, *scales, *dz;
    float *dw, *db;            // [runs][cout][cin] and [runs][cout] partial sums, or the result
    long long npix, run;       // pixels, pixels of a run (a multiple of kStep)
    int cin, xs, xg, cout, zs; // channels that count and channels per pixel; xg: scale bytes per pixel
    int nci, blocks, runs;     // blocks along cin, in all
};

__device__ __forceinline__ pw_bf16x4 read_tr(const char* p)
{
    typedef __attribute__((address_space(3))) pw_bf16x4* lds4;
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)p);
}

template <bool X8>
__global__ __launch_bounds__(kThreads, 2) void wgrad1x1_kernel(const PwParams p)
{
    __shared__ __attribute__((aligned(16))) char lds[2][2][kStep * kRow];   // [buffer][x, dz]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the blocks of a run one after the other on one XCD (work-group i runs on XCD i % 8), whose L2 then holds what they share
    const int group = (int)blockIdx.x / (8 * p.blocks), rest = (int)blockIdx.x % (8 * p.blocks);
    const int run = group * 8 + (rest & 7), block = rest >> 3;
    if (run >= p.runs) return;
    const int ci0 = block % p.nci * kBlock, co0 = block / p.nci * kBlock;
    const long long first = (long long)run * p.run;
    const long long end = first + p.run < p.npix ? first + p.run : p.npix;
    const int steps = (int)((end - first + kStep - 1) / kStep);

    // ---- staging roles: x 16 channels of a pixel, dz 8 channels of two pixels
    const int xpx = tid >> 3, xc = (tid & 7) * 16, zpx = tid >> 4, zc = (tid & 15) * 8;
    const bool xin0 = ci0 + xc < p.xs, xin1 = ci0 + xc + 8 < p.xs, zin = co0 + zc < p.zs;
    rows_u32x4 qx[2], qz[2];
    unsigned sb = 0;
    const rows_u32x4 zero = {0u, 0u, 0u, 0u};
    float bias[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) bias[k] = 0.0f;
    const bool want_bias = p.db != nullptr && ci0 == 0;

    auto load = [&](const int step) {
        const long long base = first + (long long)step * kStep;
        const long long px = base + xpx;
        const bool live = px < end;
        if (X8) {
            qx[0] = live && xin0 ? load16(p.x + px * p.xs + ci0 + xc) : zero;
            sb = live && xin0 ? (unsigned)((const unsigned char*)p.scales)[px * p.xg + (ci0 + xc) / kCk8Group] : 0u;
        } else {
            qx[0] = live && xin0 ? load16(p.x + (px * p.xs + ci0 + xc) * 2) : zero;
            qx[1] = live && xin1 ? load16(p.x + (px * p.xs + ci0 + xc + 8) * 2) : zero;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long long pz = base + zpx + 16 * j;
            qz[j] = pz < end && zin ? load16(p.dz + (pz * p.zs + co0 + zc) * 2) : zero;
        }
    };
    auto store = [&](const int buf) {
        char* xd = lds[buf][0] + xpx * kRow + xc * 2;
        if (X8) {
            const float s = ck8_scale(sb);
            rows_u32x4 lo, hi;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned a, b;
                ck8_unpack4_bf16(qx[0][j], s, a, b);
                (j < 2 ? lo : hi)[2 * (j & 1)] = a;
                (j < 2 ? lo : hi)[2 * (j & 1) + 1] = b;
            }
            *(rows_u32x4*)xd = lo;
            *(rows_u32x4*)(xd + 16) = hi;
        } else {
            *(rows_u32x4*)xd = qx[0];
            *(rows_u32x4*)(xd + 16) = qx[1];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            *(rows_u32x4*)(lds[buf][1] + (zpx + 16 * j) * kRow + zc * 2) = qz[j];
            if (want_bias) {
                float f[8];
                RowVec<__bf16>::unpack(qz[j], f);
#pragma unroll
                for (int k = 0; k < 8; ++k) bias[k] += f[k];
            }
        }
    };

    // ---- operand roles: 16 lanes read 4 pixels x 16 channels; lanes 0..31 get pixels 0..7 of a k-step, 32..63 8..15
    const int g = lane >> 4, q = (lane >> 2) & 3, pq = lane & 3;
    const int at = (8 * (g >> 1) + q) * kRow + (16 * (g & 1) + 4 * pq) * 2;
    const int zat = at + (wave >> 1) * 128, xat = at + (wave & 1) * 128;
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    // tiles of the wave that hold outputs (a wave without one only stages)
    const int wco = __builtin_amdgcn_readfirstlane(co0 + (wave >> 1) * 64), wci = __builtin_amdgcn_readfirstlane(ci0 + (wave & 1) * 64);
    const int ni = p.cout - wco, nj = p.cin - wci;

    load(0);
    store(0);
    if (steps > 1) load(1);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const char *bx = lds[s & 1][0], *bz = lds[s & 1][1];
#pragma unroll
        for (int ks = 0; ks < kStep / 16; ++ks) {
            pw_bf16x8 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const char *az = bz + zat + ks * 16 * kRow + i * 64, *ax = bx + xat + ks * 16 * kRow + i * 64;
                if (32 * i < ni && nj > 0) a[i] = __builtin_shufflevector(read_tr(az), read_tr(az + 4 * kRow), 0, 1, 2, 3, 4, 5, 6, 7);
                if (32 * i < nj && ni > 0) b[i] = __builtin_shufflevector(read_tr(ax), read_tr(ax + 4 * kRow), 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (32 * i < ni && 32 * j < nj) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
        }
        // the other buffer's readers were done before the last barrier
        if (s + 1 < steps) store((s + 1) & 1);
        if (s + 2 < steps) load(s + 2);
        __syncthreads();
    }

    // register r of lane l: row (r & 3) + 8 (r >> 2) + 4 (l >> 5) (= co), column l & 31 (= ci)
    float* dw = p.dw + (size_t)run * p.cout * p.cin;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int ci = ci0 + (wave & 1) * 64 + j * 32 + (lane & 31);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int co = co0 + (wave >> 1) * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
                if (co < p.cout && ci < p.cin) dw[(size_t)co * p.cin + ci] = acc[i][j][r];
            }
        }
    if (want_bias) {   // (uniform over the work-group; the last barrier freed the buffers)
        float* sum = (float*)&lds[0][0][0];   // [16 pixel rows][128 channels]
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[zpx * kBlock + zc + k] = bias[k];
        __syncthreads();
        if (tid < kBlock && co0 + tid < p.cout) {
            float v = sum[tid];
#pragma unroll
            for (int k = 1; k < 16; ++k) v += sum[k * kBlock + tid];
            p.db[(size_t)run * p.cout + co0 + tid] = v;
        }
    }
}

// Adds the runs' partial sums: 64 elements to a block, 16 thread groups taking every 16th run, then theirs in order.
__global__ __launch_bounds__(1024) void wgrad1x1_sums_kernel(const float* __restrict__ pw, const float* __restrict__ pb, float* __restrict__ dw,
                                                             float* __restrict__ db, const int nw, const int nb, const int runs)
{
    __shared__ float red[16][64];
    const int col = threadIdx.x & 63, part = threadIdx.x >> 6;
    const int e = (int)blockIdx.x * 64 + col;
    const float* src = e < nw ? pw + e : pb + (e - nw);
    const int stride = e < nw ? nw : nb;
    float s = 0.0f;
    if (e < nw + nb)
#pragma unroll 8
        for (int k = part; k < runs; k += 16) s += src[(size_t)k * stride];
    red[part][col] = s;
    __syncthreads();
    if (part != 0 || e >= nw + nb) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][col];
    if (e < nw) dw[e] = s;
    else db[e - nw] = s;
}

struct PwPlan {
    int nci, blocks, runs;
    long long run;
};
PwPlan pw_plan(const long long npix, const int cin, const int cout)
{
    PwPlan q;
    q.nci = srhip_div_up(cin, kBlock);
    q.blocks = q.nci * srhip_div_up(cout, kBlock);
    const long long steps = (npix + kStep - 1) / kStep;
    // three work-groups to a CU hide the loads' latency (160 -> 112 channels, a million pixels: 109 us; two 125, four 150: the
    // registers hold three); a run of eight steps pays for its 64 KB of partial sums (65 k pixels: 21.5 us; sixteen 24.2)
    long long runs = 3ll * srhip_num_cus() / q.blocks;
    if (runs > steps / 8) runs = steps / 8;
    if (runs < 1) runs = 1;
    q.run = (steps + runs - 1) / runs * kStep;
    q.runs = (int)((npix + q.run - 1) / q.run);
    return q;
}

}  // namespace

extern "C" {

SRHIP_API size_t srhip_wgrad1x1_workspace_bytes(long long npix, int cin, int cout)
{
    if (npix < 1 || cin < 1 || cout < 1) return 0;
    const PwPlan q = pw_plan(npix, cin, cout);
    return q.runs > 1 ? (size_t)q.runs * ((size_t)cin + 1) * cout * sizeof(float) : 0;
}

SRHIP_API int srhip_wgrad1x1(const void* x, const void* x_scales, const void* dz, float* dw, float* db, void* workspace, long long npix, int cin,
                             int x_cstride, int cout, int dz_cstride, void* stream)
{
    SRHIP_REQUIRE(npix >= 1 && cin >= 1 && cout >= 1, "wgrad1x1: empty layer (%lld pixels, %d -> %d channels)", npix, cin, cout);
    SRHIP_REQUIRE(x && dz && dw, "wgrad1x1: null pointer");
    const int per = x_scales ? 16 : 8;
    SRHIP_REQUIRE(x_cstride >= cin && x_cstride % per == 0 && dz_cstride >= cout && dz_cstride % 8 == 0,
                  "wgrad1x1: %d and %d channels per pixel (at least the layer's %d and %d, multiples of %d and 8)", x_cstride, dz_cstride, cin, cout, per);
    SRHIP_REQUIRE((((size_t)x | (size_t)dz) & 15) == 0, "wgrad1x1: maps start at multiples of 16 bytes");
    // (a launch has fewer than 2^32 threads: the sums' has 1024 for 64 weights or biases)
    SRHIP_REQUIRE((long long)cout * (cin + 1ll) < (1ll << 28) - 64, "wgrad1x1: weight too large");
    const PwPlan q = pw_plan(npix, cin, cout);
    SRHIP_REQUIRE(q.runs == 1 || workspace, "wgrad1x1: null workspace");
    PwParams p;
    p.x = (const char*)x; p.scales = (const char*)x_scales; p.dz = (const char*)dz;
    float* pb = (float*)workspace + (size_t)q.runs * cout * cin;
    p.dw = q.runs > 1 ? (float*)workspace : dw;
    p.db = db == nullptr ? nullptr : q.runs > 1 ? pb : db;
    p.npix = npix; p.run = q.run;
    p.cin = cin; p.xs = x_cstride; p.xg = srhip_div_up(x_cstride, kCk8Group); p.cout = cout; p.zs = dz_cstride;
    p.nci = q.nci; p.blocks = q.blocks; p.runs = q.runs;
    const long long grid = (long long)srhip_div_up(q.runs, 8) * 8 * q.blocks;
    SRHIP_REQUIRE(grid < (1ll << 32) / kThreads, "wgrad1x1: layer too large");
    hipStream_t s = (hipStream_t)stream;
    if (x_scales) hipLaunchKernelGGL(wgrad1x1_kernel<true>, dim3((unsigned)grid), dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL(wgrad1x1_kernel<false>, dim3((unsigned)grid), dim3(kThreads), 0, s, p);
    const int rc = srhip_check_launch("wgrad1x1_kernel");
    if (rc != SRHIP_OK || q.runs == 1) return rc;
    const int nw = cout * cin, nb = db ? cout : 0;
    hipLaunchKernelGGL(wgrad1x1_sums_kernel, dim3((unsigned)srhip_div_up((long long)nw + nb, 64)), dim3(1024), 0, s, p.dw, pb, dw, db, nw, nb, q.runs);
    return srhip_check_launch("wgrad1x1_sums_kernel");
}

}  // extern "C"
