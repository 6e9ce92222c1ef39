// What the forward and backward kernels of the fused block norm share: how a row of channels lies on a group of lanes, sums
// over a row, the gate.
#pragma once
#include "rows_util.h"

namespace {

// A group of TPR lanes (a power of two) holds a row: vector v of lane t starts at channel (v * TPR + t) * VEC.  Groups of up
// to 64 lanes lie in one wave, several rows to a wave; wider ones are some waves of a work-group or all of them.
template <class T_, int TPR_, int V_>
struct RowCfg {
    using T = T_;
    static constexpr int TPR = TPR_, V = V_, VEC = RowVec<T>::VEC;
    static constexpr int THREADS = TPR <= 256 ? 256 : TPR;
    static constexpr int RPB = THREADS / TPR;      // rows in flight per work-group
    static constexpr int E = V * VEC;              // elements of a row per lane
    static constexpr int CMAX = TPR * E;
};

// Sums over the TPR lanes of a row; `turn` alternates between two scratch areas, so that one barrier per sum is enough.
template <class C>
struct RowSum {
    float* scratch;   // row_sum_scratch() floats
    int turn;
    __device__ __forceinline__ void two(float& a, float& b)
    {
        if constexpr (C::TPR <= 64) {
            a = lanes_sum<C::TPR>(a);
            b = lanes_sum<C::TPR>(b);
        } else {
            constexpr int NW = C::TPR / 64;
            a = lanes_sum<64>(a);
            b = lanes_sum<64>(b);
            float* s = scratch + (turn * C::RPB + threadIdx.x / C::TPR) * 2 * NW;
            turn ^= 1;
            const int w = (threadIdx.x % C::TPR) >> 6;
            if ((threadIdx.x & 63) == 0) { s[w] = a; s[NW + w] = b; }
            __syncthreads();
            a = s[0]; b = s[NW];
#pragma unroll
            for (int k = 1; k < NW; ++k) { a += s[k]; b += s[NW + k]; }
        }
    }
    __device__ __forceinline__ float one(float a)
    {
        float b = 0.0f;
        if constexpr (C::TPR <= 64) return lanes_sum<C::TPR>(a);
        two(a, b);
        return a;
    }
};
template <class C>
constexpr int row_sum_scratch() { return C::TPR <= 64 ? 1 : 4 * C::RPB * (C::TPR / 64); }

// What a lane holds of channels behind the row's end becomes 0.  Lanes that lie inside the row skip it: one branch.
template <class C>
__device__ __forceinline__ void zero_absent(float* f, const int* nv)
{
#pragma unroll
    for (int v = 0; v < C::V; ++v)
        if (nv[v] < C::VEC)
#pragma unroll
            for (int k = 0; k < C::VEC; ++k)
                if (k >= nv[v]) f[v * C::VEC + k] = 0.0f;
}

// Rows held as f[E] (absent channels 0) become (f - mean) / sqrt(mean square of that + eps), without the mean for the rms
// form; returns the factor 1 / sqrt.  Two sums over registers: the squares are taken of differences from the mean, as the
// definition has it, so a mean that is large against the spread costs no digits.  Two rows at once share their sums' steps.
template <class C>
__device__ __forceinline__ void normalise(RowSum<C>& sum, const bool first, float* f, const bool second, float* g, const int* nv, const bool layer,
                                          const float inv_c, const float eps, float& rstd_f, float& rstd_g)
{
    float a = 0.0f, b = 0.0f;
    if (layer) {
        if (first)
#pragma unroll
            for (int j = 0; j < C::E; ++j) a += f[j];
        if (second)
#pragma unroll
            for (int j = 0; j < C::E; ++j) b += g[j];
        sum.two(a, b);
        a *= inv_c;
        b *= inv_c;
        if (first) {
#pragma unroll
            for (int j = 0; j < C::E; ++j) f[j] -= a;
            zero_absent<C>(f, nv);
        }
        if (second) {
#pragma unroll
            for (int j = 0; j < C::E; ++j) g[j] -= b;
            zero_absent<C>(g, nv);
        }
        a = b = 0.0f;
    }
    if (first)
#pragma unroll
        for (int j = 0; j < C::E; ++j) a += f[j] * f[j];
    if (second)
#pragma unroll
        for (int j = 0; j < C::E; ++j) b += g[j] * g[j];
    sum.two(a, b);
    rstd_f = 1.0f / sqrtf(a * inv_c + eps);
    rstd_g = 1.0f / sqrtf(b * inv_c + eps);
    if (first)
#pragma unroll
        for (int j = 0; j < C::E; ++j) f[j] *= rstd_f;
    if (second)
#pragma unroll
        for (int j = 0; j < C::E; ++j) g[j] *= rstd_g;
}
template <class C>
__device__ __forceinline__ float normalise(RowSum<C>& sum, float* f, const int* nv, const bool layer, const float inv_c, const float eps)
{
    float a = 0.0f;
    if (layer) {
#pragma unroll
        for (int j = 0; j < C::E; ++j) a += f[j];
        a = sum.one(a) * inv_c;
#pragma unroll
        for (int j = 0; j < C::E; ++j) f[j] -= a;
        zero_absent<C>(f, nv);
        a = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < C::E; ++j) a += f[j] * f[j];
    const float rstd = 1.0f / sqrtf(sum.one(a) * inv_c + eps);
#pragma unroll
    for (int j = 0; j < C::E; ++j) f[j] *= rstd;
    return rstd;
}

// A parameter vector's values of a lane's channels: `none` where there is no vector, 0 for absent channels.
template <class C>
__device__ __forceinline__ void load_params(const float* p, const int* c0, const int* nv, const float none, float* f)
{
#pragma unroll
    for (int v = 0; v < C::V; ++v)
#pragma unroll
        for (int j = 0; j < C::VEC; ++j) f[v * C::VEC + j] = j < nv[v] ? (p != nullptr ? p[c0[v] + j] : none) : 0.0f;
}
// A map's row, or part of it.  `whole`: no lane's vector reaches past the row's end (one test for the launch).
template <class C>
__device__ __forceinline__ void load_row(const char* p, const int* c0, const int* nv, const bool whole, rows_u32x4* q)
{
    using T = typename C::T;
    if (whole) {
#pragma unroll
        for (int v = 0; v < C::V; ++v) q[v] = load16(p + c0[v] * RowVec<T>::SIZE);
    } else {
#pragma unroll
        for (int v = 0; v < C::V; ++v) q[v] = load_row16<T>(p + c0[v] * RowVec<T>::SIZE, nv[v]);
    }
}
template <class C>
__device__ __forceinline__ void store_row(char* p, const int* c0, const int* nv, const bool whole, const float* f)
{
    using T = typename C::T;
    if (whole) {
#pragma unroll
        for (int v = 0; v < C::V; ++v) store16(p + c0[v] * RowVec<T>::SIZE, RowVec<T>::pack(f + v * C::VEC));
    } else {
#pragma unroll
        for (int v = 0; v < C::V; ++v) store_row16<T>(p + c0[v] * RowVec<T>::SIZE, RowVec<T>::pack(f + v * C::VEC), nv[v]);
    }
}
template <class C>
__device__ __forceinline__ void unpack_row(const rows_u32x4* q, float* f)
{
#pragma unroll
    for (int v = 0; v < C::V; ++v) RowVec<typename C::T>::unpack(q[v], f + v * C::VEC);
}
// the gate map's row where it is fp32 beside bf16 maps
template <class C>
__device__ __forceinline__ void load_gate_f32(const char* p, const int* c0, const int* nv, float* g)
{
    load_params<C>((const float*)p, c0, nv, 0.0f, g);
}

__device__ __forceinline__ float sigmoid_f32(const float x) { return 1.0f / (1.0f + expf(-x)); }

}  // namespace
