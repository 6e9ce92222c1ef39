// 8-bit activation checkpoints for gfx950: what a training step keeps of a map for its backward pass, at 33 bytes for 32
// channels instead of 64 (bf16) or 128 (fp32).  (The maps that autograd saves for loss.backward() at core/trainer.py:160:
// the inputs of every nn.Conv2d, core/models/model.py:12,26-28,112-114, and the outputs of its ReLUs.)
//
//   a = max |x| over the finite values of 32 channels = m 2^E, 1 <= m < 2
//   scale 2^e with e = max(E - 8 + [m > 1.75], -117): the smallest power of two that brings a to 448, the largest e4m3
//     value, or less -- the largest of a group uses the code's top binade or the one below it and no value saturates, but
//     one above 1.75 * 2^127, which is kept as that
//   code = x 2^-e rounded to the nearest e4m3 value, ties to even; x <> 0 never becomes 0 but the smallest code of its
//     sign, so that [code > 0] is the ReLU pattern of x.  Infinities and NaN become NaN, the rest of their group does not
//     change.
//
// A power of two as scale makes the decoded value exact in bf16 (4 significant bits), hence one definition for every reader
// (restore, weight gradient, norm backward), and encoding free of divisions.
//
// All kernels here stream: bound by HBM.
#include "rows_util.h"

namespace {

constexpr int kThreads = 256;

// ---- encode one chunk of 8 channels held by a lane; LANES lanes side by side (4: 32 channels) hold a group
struct Encoded {
    rows_u32x2 codes;
    unsigned scale;
};
template <int LANES>
__device__ __forceinline__ Encoded ck8_encode(float* f)
{
    float a = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = fmaxf(a, fabsf(f[j]));   // a NaN operand is passed over
    const float top = __uint_as_float(kCk8Largest);
    if (a > top) {                                              // rare: the largest FINITE value counts, infinities become NaN
        a = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (fabsf(f[j]) == INFINITY) f[j] = NAN;
            else if (fabsf(f[j]) > top) f[j] = copysignf(top, f[j]);
            a = fmaxf(a, fabsf(f[j]));
        }
    }
    a = lanes_max<LANES>(a);
    // a mantissa above 1.75 carries into the exponent field
    int e = (int)((__float_as_uint(a) + 0x1fffffu) >> 23) - 8;
    e = e < kCk8Lowest ? kCk8Lowest : e;
    const float inv = __uint_as_float((unsigned)(2 * kCk8Bias - e) << 23);
    Encoded r;
    r.scale = (unsigned)e;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float* g = f + 4 * j;
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(g[0] * inv, g[1] * inv, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(g[2] * inv, g[3] * inv, w, true);
        // bytes whose magnitude is 0 although the value is not: |1
        unsigned nz = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) nz |= (__float_as_uint(g[k]) << 1) != 0u ? 1u << (8 * k) : 0u;
        const unsigned zero = ~(((unsigned)w & 0x7f7f7f7fu) + 0x7f7f7f7fu) >> 7;   // bit 0 of a byte: its magnitude is 0
        r.codes[j] = (unsigned)w | (nz & zero);
    }
    return r;
}

// 8 channels of a row from c0 on (nv of them exist) as fp32
template <class T>
__device__ __forceinline__ void load8(const char* p, const int nv, float* f)
{
    constexpr int VEC = RowVec<T>::VEC;
#pragma unroll
    for (int j = 0; j < 8 / VEC; ++j) RowVec<T>::unpack(load_row16<T>(p + 16 * j, nv - VEC * j), f + VEC * j);
}
template <class T>
__device__ __forceinline__ void store8(char* p, const int nv, const float* f)
{
    constexpr int VEC = RowVec<T>::VEC;
#pragma unroll
    for (int j = 0; j < 8 / VEC; ++j) store_row16<T>(p + 16 * j, RowVec<T>::pack(f + VEC * j), nv - VEC * j);
}
__device__ __forceinline__ rows_u32x2 load_codes8(const unsigned char* p, const int nv)
{
    rows_u32x2 q = {0u, 0u};
    if (nv >= 8) __builtin_memcpy(&q, p, 8);
    else
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (j < nv) q[j >> 2] |= (unsigned)p[j] << (8 * (j & 3));
    return q;
}
__device__ __forceinline__ void store_codes8(unsigned char* p, const rows_u32x2 q, const int nv)
{
    if (nv >= 8) __builtin_memcpy(p, &q, 8);
    else
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (j < nv) p[j] = (unsigned char)(q[j >> 2] >> (8 * (j & 3)));
}

// Where a lane's chunk lies.  LANES lanes serve one (row, group of 32 channels) unit: four, or, of maps that have no more than
// 16 or 8 channels, two or one.
struct Chunk {
    long long at;      // first element in the map
    long long unit;    // place of the group's scale
    int nv;            // channels of the chunk that exist, <= 0: none
};
__device__ __forceinline__ Chunk chunk_of(const long long unit, const int q, const int c, const int groups)
{
    Chunk k;
    k.unit = unit;
    // units of one launch fit 32 bits (the host cuts larger maps into several launches)
    const unsigned row = (unsigned)unit / (unsigned)groups;
    const int c0 = ((int)((unsigned)unit - row * (unsigned)groups)) * kCk8Group + 8 * q;
    k.at = (long long)row * c + c0;
    k.nv = c - c0;
    return k;
}

template <class T, int LANES>
__global__ __launch_bounds__(kThreads) void checkpoint8_pack_kernel(const char* __restrict__ x, unsigned char* __restrict__ codes,
                                                                    unsigned char* __restrict__ scales, const long long units,
                                                                    const int c, const int groups)
{
    const int q = threadIdx.x % LANES;
    const long long unit = (long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    if (unit >= units) return;   // all lanes of a unit
    const Chunk k = chunk_of(unit, q, c, groups);
    float f[8];
    load8<T>(x + k.at * RowVec<T>::SIZE, k.nv, f);
    const Encoded r = ck8_encode<LANES>(f);
    store_codes8(codes + k.at, r.codes, k.nv);
    if (q == 0) scales[unit] = (unsigned char)r.scale;
}

// The same for an (n, h, w, 64) bf16 map, with its ReLU pattern in the layout that the convolution's sign-bit forms read
// (srhip_conv3x3_signbits_bytes): a wave takes 32 pixels of a row, lane = (x % 8) * 8 + channel / 8 is a word's place.
__global__ __launch_bounds__(kThreads) void checkpoint8_pack_signbits_kernel(const char* __restrict__ x, unsigned char* __restrict__ codes,
                                                                             unsigned char* __restrict__ scales, unsigned* __restrict__ bits,
                                                                             const long long nwords, const int w, const int wgroups)
{
    const long long wv = (long long)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (wv >= nwords) return;
    const int lane = threadIdx.x & 63;
    const long long row = wv / wgroups;
    const int x0 = (int)(wv - row * wgroups) * 32 + (lane >> 3);
    unsigned word = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int px = x0 + 8 * k;
        if (px < w) {   // a pixel's eight lanes together
            const long long chunk = (row * w + px) * 8 + (lane & 7);
            float f[8];
            RowVec<__bf16>::unpack(load16(x + chunk * 16), f);
#pragma unroll
            for (int j = 0; j < 8; ++j) word |= f[j] > 0.0f ? 1u << (8 * k + j) : 0u;
            const Encoded r = ck8_encode<4>(f);
            *(rows_u32x2*)(codes + chunk * 8) = r.codes;
            if ((lane & 3) == 0) scales[chunk >> 2] = (unsigned char)r.scale;
        }
    }
    bits[wv * 64 + lane] = word;
}

template <class T, int LANES>
__global__ __launch_bounds__(kThreads) void checkpoint8_restore_kernel(const unsigned char* __restrict__ codes,
                                                                       const unsigned char* __restrict__ scales, char* __restrict__ y,
                                                                       const long long units, const int c, const int groups)
{
    const int q = threadIdx.x % LANES;
    const long long unit = (long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    if (unit >= units) return;
    const Chunk k = chunk_of(unit, q, c, groups);
    const rows_u32x2 w = load_codes8(codes + k.at, k.nv);
    const float s = ck8_scale(scales[unit]);
    float f[8];
    ck8_unpack4(w[0], s, f);
    ck8_unpack4(w[1], s, f + 4);
    store8<T>(y + k.at * RowVec<T>::SIZE, k.nv, f);
}

// out = dy where the code is positive, else 0: codes lie like the map's elements, whatever its channels
__global__ __launch_bounds__(kThreads) void relu_mask_checkpoint8_kernel(const char* dy, const unsigned char* __restrict__ codes, char* out,
                                                                         const long long n)
{
    const long long i = ((long long)blockIdx.x * kThreads + threadIdx.x) * 8;
    if (i >= n) return;
    const int nv = n - i < 8 ? (int)(n - i) : 8;
    const rows_u32x2 w = load_codes8(codes + i, nv);
    rows_u32x4 d = load_row16<__bf16>(dy + 2 * i, nv);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned code = (w[j >> 2] >> (8 * (j & 3))) & 0xffu;
        if (code - 1u >= 0x7eu) d[j >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;   // 0x01 .. 0x7e are the positive numbers
    }
    store_row16<__bf16>(out + 2 * i, d, nv);
}

// A launch has fewer than 2^32 threads, and units (rows times groups) that fit 31 bits: the rows of one launch whose units take
// `lanes` lanes each.
constexpr long long kMaxBlocks = (1ll << 32) / kThreads - 1;
long long slab_rows(const int groups, const int lanes)
{
    const long long units = kMaxBlocks * (kThreads / lanes);
    return (units < (1ll << 31) ? units : (1ll << 31) - 1) / groups;
}

template <class T, int LANES>
int pack_slab(const char* x, unsigned char* codes, unsigned char* scales, const long long units, const int c, const int groups, hipStream_t s)
{
    hipLaunchKernelGGL((checkpoint8_pack_kernel<T, LANES>), dim3((unsigned)((units + kThreads / LANES - 1) / (kThreads / LANES))), dim3(kThreads), 0, s,
                       x, codes, scales, units, c, groups);
    return srhip_check_launch("checkpoint8_pack_kernel");
}
template <class T, int LANES>
int restore_slab(const unsigned char* codes, const unsigned char* scales, char* y, const long long units, const int c, const int groups, hipStream_t s)
{
    hipLaunchKernelGGL((checkpoint8_restore_kernel<T, LANES>), dim3((unsigned)((units + kThreads / LANES - 1) / (kThreads / LANES))), dim3(kThreads), 0, s,
                       codes, scales, y, units, c, groups);
    return srhip_check_launch("checkpoint8_restore_kernel");
}
// Calls f(first row, units, lanes of a unit) for each launch over `rows` rows of c channels.
// (Two 540 x 959 maps of ten fp32 channels: with four lanes to a row 17 us, with two 13.6.)
template <class F>
int by_slabs(const long long rows, const int c, const int groups, F&& f)
{
    const int lanes = c <= 8 ? 1 : c <= 16 ? 2 : 4;
    const long long most = slab_rows(groups, lanes);
    for (long long r = 0; r < rows; r += most) {
        const int rc = f(r, (rows - r < most ? rows - r : most) * groups, lanes);
        if (rc != SRHIP_OK) return rc;
    }
    return SRHIP_OK;
}
template <class T>
int pack_rows(const char* x, unsigned char* codes, unsigned char* scales, const long long rows, const int c, hipStream_t s)
{
    const int groups = srhip_div_up(c, kCk8Group);
    return by_slabs(rows, c, groups, [&](const long long r, const long long units, const int lanes) {
        return (lanes == 1 ? pack_slab<T, 1> : lanes == 2 ? pack_slab<T, 2> : pack_slab<T, 4>)(x + r * c * RowVec<T>::SIZE, codes + r * c, scales + r * groups, units, c, groups, s);
    });
}
template <class T>
int restore_rows(const unsigned char* codes, const unsigned char* scales, char* y, const long long rows, const int c, hipStream_t s)
{
    const int groups = srhip_div_up(c, kCk8Group);
    return by_slabs(rows, c, groups, [&](const long long r, const long long units, const int lanes) {
        return (lanes == 1 ? restore_slab<T, 1> : lanes == 2 ? restore_slab<T, 2> : restore_slab<T, 4>)(codes + r * c, scales + r * groups, y + r * c * RowVec<T>::SIZE, units, c, groups, s);
    });
}

}  // namespace

extern "C" {

SRHIP_API int srhip_checkpoint8_pack(const void* x, int dtype, void* codes, void* scales, long long rows, int c, void* stream)
{
    SRHIP_REQUIRE(rows >= 0 && c >= 1, "checkpoint8_pack: bad shape (%lld rows of %d channels)", rows, c);
    SRHIP_REQUIRE(dtype == SRHIP_DT_BF16 || dtype == SRHIP_DT_F32, "checkpoint8_pack: unknown type %d", dtype);
    if (rows == 0) return SRHIP_OK;
    SRHIP_REQUIRE(x && codes && scales, "checkpoint8_pack: null pointer");
    return (dtype == SRHIP_DT_BF16 ? pack_rows<__bf16> : pack_rows<float>)((const char*)x, (unsigned char*)codes, (unsigned char*)scales, rows, c,
                                                                            (hipStream_t)stream);
}

SRHIP_API int srhip_checkpoint8_pack_signbits(const void* x, void* codes, void* scales, void* signbits, int n, int h, int w, void* stream)
{
    SRHIP_REQUIRE(n >= 0 && h >= 0 && w >= 0, "checkpoint8_pack_signbits: bad shape");
    if (n == 0 || h == 0 || w == 0) return SRHIP_OK;
    SRHIP_REQUIRE(x && codes && scales && signbits, "checkpoint8_pack_signbits: null pointer");
    SRHIP_REQUIRE((((size_t)x) & 15) == 0 && (((size_t)codes) & 7) == 0 && (((size_t)signbits) & 3) == 0,
                  "checkpoint8_pack_signbits: maps of 64 channels start at multiples of 16 (x), 8 (codes) and 4 bytes (signbits)");
    const int wgroups = srhip_div_up(w, 32);
    const long long nwords = (long long)n * h * wgroups;
    const long long blocks = (nwords + kThreads / 64 - 1) / (kThreads / 64);
    SRHIP_REQUIRE(blocks <= kMaxBlocks, "checkpoint8_pack_signbits: map too large");   // (2^31 pixels of whole groups of 32: 256 GB)
    hipLaunchKernelGGL(checkpoint8_pack_signbits_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, (const char*)x,
                       (unsigned char*)codes, (unsigned char*)scales, (unsigned*)signbits, nwords, w, wgroups);
    return srhip_check_launch("checkpoint8_pack_signbits_kernel");
}

SRHIP_API int srhip_checkpoint8_restore(const void* codes, const void* scales, void* y, int dtype, long long rows, int c, void* stream)
{
    SRHIP_REQUIRE(rows >= 0 && c >= 1, "checkpoint8_restore: bad shape (%lld rows of %d channels)", rows, c);
    SRHIP_REQUIRE(dtype == SRHIP_DT_BF16 || dtype == SRHIP_DT_F32, "checkpoint8_restore: unknown type %d", dtype);
    if (rows == 0) return SRHIP_OK;
    SRHIP_REQUIRE(codes && scales && y, "checkpoint8_restore: null pointer");
    return (dtype == SRHIP_DT_BF16 ? restore_rows<__bf16> : restore_rows<float>)((const unsigned char*)codes, (const unsigned char*)scales, (char*)y,
                                                                                  rows, c, (hipStream_t)stream);
}

SRHIP_API int srhip_relu_mask_checkpoint8(const void* dy, const void* codes, void* out, size_t n, void* stream)
{
    if (n == 0) return SRHIP_OK;
    SRHIP_REQUIRE(dy && codes && out, "relu_mask_checkpoint8: null pointer");
    constexpr size_t kMost = (size_t)kMaxBlocks * 8 * kThreads;   // elements of a launch
    for (size_t i = 0; i < n; i += kMost) {
        const size_t m = n - i < kMost ? n - i : kMost;
        hipLaunchKernelGGL(relu_mask_checkpoint8_kernel, dim3((unsigned)((m + 8 * kThreads - 1) / (8 * kThreads))), dim3(kThreads), 0, (hipStream_t)stream,
                           (const char*)dy + 2 * i, (const unsigned char*)codes + i, (char*)out + 2 * i, (long long)m);
        const int rc = srhip_check_launch("relu_mask_checkpoint8_kernel");
        if (rc != SRHIP_OK) return rc;
    }
    return SRHIP_OK;
}

}  // extern "C"
