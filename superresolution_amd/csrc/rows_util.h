// Device helpers of the kernels that work on rows of channels (a pixel's channels, or any (rows, c) matrix): 16-byte vectors
// of either map type at any alignment, sums and maxima over a group of lanes, the 8-bit checkpoint's number format.
#pragma once
#include "srhip_common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) unsigned rows_u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned rows_u32x2;

// ---- one vector of 16 bytes = VEC elements.  Rows of odd channel counts start at any element: gfx950 reads and writes
// global memory at any alignment with one instruction, so the same 16-byte access serves every row.
__device__ __forceinline__ rows_u32x4 load16(const char* p)
{
    rows_u32x4 q;
    __builtin_memcpy(&q, p, 16);
    return q;
}
__device__ __forceinline__ void store16(char* p, const rows_u32x4 q) { __builtin_memcpy(p, &q, 16); }

template <class T>
struct RowVec;
template <>
struct RowVec<__bf16> {
    using T = __bf16;
    __device__ static __forceinline__ rows_u32x4 load(const char* p) { return load16(p); }
    __device__ static __forceinline__ void store(char* p, const rows_u32x4 q) { store16(p, q); }
    static constexpr int VEC = 8, SIZE = 2;
    __device__ static __forceinline__ void unpack(const rows_u32x4 q, float* f)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) { f[2 * j] = bf16_lo(q[j]); f[2 * j + 1] = bf16_hi(q[j]); }
    }
    __device__ static __forceinline__ rows_u32x4 pack(const float* f)
    {
        rows_u32x4 q;
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
        return q;
    }
};
template <>
struct RowVec<float> {
    using T = float;
    __device__ static __forceinline__ rows_u32x4 load(const char* p) { return load16(p); }
    __device__ static __forceinline__ void store(char* p, const rows_u32x4 q) { store16(p, q); }
    static constexpr int VEC = 4, SIZE = 4;
    __device__ static __forceinline__ void unpack(const rows_u32x4 q, float* f)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(q[j]);
    }
    __device__ static __forceinline__ rows_u32x4 pack(const float* f)
    {
        rows_u32x4 q;
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = __float_as_uint(f[j]);
        return q;
    }
};

// One element instead of a vector, for rows that are shorter than one.
template <class T_>
struct RowOne {
    using T = T_;
    static constexpr int VEC = 1, SIZE = RowVec<T>::SIZE;
    __device__ static __forceinline__ rows_u32x4 load(const char* p)
    {
        rows_u32x4 q = {0u, 0u, 0u, 0u};
        unsigned w = 0u;
        __builtin_memcpy(&w, p, SIZE);
        q[0] = w;
        return q;
    }
    __device__ static __forceinline__ void store(char* p, const rows_u32x4 q)
    {
        const unsigned w = q[0];
        __builtin_memcpy(p, &w, SIZE);
    }
    __device__ static __forceinline__ void unpack(const rows_u32x4 q, float* f) { f[0] = SIZE == 2 ? bf16_lo(q[0]) : __uint_as_float(q[0]); }
    __device__ static __forceinline__ rows_u32x4 pack(const float* f)
    {
        rows_u32x4 q = {0u, 0u, 0u, 0u};
        q[0] = SIZE == 2 ? f32_to_bf16_bits(f[0]) : __float_as_uint(f[0]);
        return q;
    }
};

// The first `nv` elements (of SIZE bytes) of a vector whose 16 bytes reach past the end of the row; the others are 0.
template <int SIZE>
__device__ __forceinline__ rows_u32x4 load_part(const char* p, const int nv)
{
    rows_u32x4 q = {0u, 0u, 0u, 0u};
    if constexpr (SIZE == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < nv) q[j] = ((const unsigned*)p)[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < nv) q[j >> 1] |= (unsigned)((const unsigned short*)p)[j] << (16 * (j & 1));
    }
    return q;
}
template <int SIZE>
__device__ __forceinline__ void store_part(char* p, const rows_u32x4 q, const int nv)
{
    if constexpr (SIZE == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < nv) ((unsigned*)p)[j] = q[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < nv) ((unsigned short*)p)[j] = (unsigned short)(q[j >> 1] >> (16 * (j & 1)));
    }
}
// nv = elements of the row at and behind p: whole vector, part of one, or nothing (the row has ended)
template <class T>
__device__ __forceinline__ rows_u32x4 load_row16(const char* p, const int nv)
{
    if (nv >= RowVec<T>::VEC) return load16(p);
    return load_part<RowVec<T>::SIZE>(p, nv);
}
template <class T>
__device__ __forceinline__ void store_row16(char* p, const rows_u32x4 q, const int nv)
{
    if (nv >= RowVec<T>::VEC) store16(p, q);
    else store_part<RowVec<T>::SIZE>(p, q, nv);
}

// ---- sums and maxima over an aligned group of W lanes (a power of two), every lane of which gets the result.  Steps of 1
// to 8 lanes are data-parallel-primitive moves, 16 and 32 the row swaps of gfx950: no LDS instruction and no address.
template <int CTRL>
__device__ __forceinline__ float dpp_move(const float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int W, class Op>
__device__ __forceinline__ float lanes_reduce(float v, Op op)
{
    if constexpr (W >= 2) v = op(v, dpp_move<0xB1>(v));     // lanes 1 0 3 2 of each quad
    if constexpr (W >= 4) v = op(v, dpp_move<0x4E>(v));     // lanes 2 3 0 1
    if constexpr (W >= 8) v = op(v, dpp_move<0x141>(v));    // half-row mirror: the other quad of eight
    if constexpr (W >= 16) v = op(v, dpp_move<0x140>(v));   // row mirror: the other eight of sixteen
    if constexpr (W >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    if constexpr (W >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    return v;
}
template <int W>
__device__ __forceinline__ float lanes_sum(const float v)
{
    return lanes_reduce<W>(v, [](float a, float b) { return a + b; });
}
// Sum over the lanes of a wave that have the same place in their group of W lanes; every lane gets it.
template <int W>
__device__ __forceinline__ float same_place_sum(float v)
{
    if constexpr (W <= 1) v += dpp_move<0xB1>(v);
    if constexpr (W <= 2) v += dpp_move<0x4E>(v);     // the other pair of each quad
    if constexpr (W <= 4) v += dpp_move<0x124>(v);    // rotate sixteen lanes by 4, then by 8: all four quads
    if constexpr (W <= 8) v += dpp_move<0x128>(v);
    if constexpr (W <= 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if constexpr (W <= 32) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return v;
}
template <int W>
__device__ __forceinline__ float lanes_max(const float v)
{
    return lanes_reduce<W>(v, [](float a, float b) { return fmaxf(a, b); });
}

// ---- 8-bit checkpoint: e4m3 codes (4 exponent bits, 3 of mantissa, largest value 448, no infinity) and, for every 32
// channels of a row, one byte s: the scale 2^(s - 127).
constexpr int kCk8Group = 32;
constexpr int kCk8Bias = 127;
// Lowest scale byte.  The smallest code times 2^(10 - 127) is 2^-9 * 2^-117 = 2^-126, the smallest normal fp32 and bf16
// number, and no value reaches 2^128: every value that a checkpoint stands for is exact in both types.
constexpr int kCk8Lowest = 10;
// The largest magnitude kept, 1.75 * 2^127 = 448 * 2^119: a larger one would round to 2^128 in a coarser scale.
constexpr unsigned kCk8Largest = 0x7f600000u;

__device__ __forceinline__ float ck8_scale(const unsigned s) { return __uint_as_float(s << 23); }
// values of the 4 codes in w (one instruction decodes and scales two: exact, the scale is a power of two)
__device__ __forceinline__ void ck8_unpack4(const unsigned w, const float scale, float* f)
{
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
    f[0] = lo[0]; f[1] = lo[1]; f[2] = hi[0]; f[3] = hi[1];
}
// ... as bf16 pairs, exact as well
__device__ __forceinline__ void ck8_unpack4_bf16(const unsigned w, const float scale, unsigned& lo, unsigned& hi)
{
    lo = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
    hi = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
}

}  // namespace
