// What the forward and backward kernels of the fused block norm share: how a row of channels lies on a group of lanes, sums
// over a row, the gate.
#pragma once
#include "rows_util.h"

namespace {

// A group of TPR lanes (a power of two) holds a row: vector v of lane t starts at channel (v * TPR + t) * VEC.  Groups of up
// to 64 lanes lie in one wave, several rows to a wave; wider ones are some waves of a work-group or all of them.
// ODD: the channel count is no multiple of a vector.  The row's last vector then starts early enough to end with the row; its
// leading elements are the previous vector's as well: both lanes compute (and write) the same values of them, the sums leave
// the second lane's out.  So every access is a whole vector, at any channel count from one vector on.
template <class Vec_, int TPR_, int V_, bool ODD_>
struct RowCfg {
    using Vec = Vec_;
    static constexpr int TPR = TPR_, V = V_, VEC = Vec::VEC, SIZE = Vec::SIZE;
    static constexpr bool ODD = ODD_;
    static constexpr int THREADS = TPR <= 256 ? 256 : TPR;
    static constexpr int RPB = THREADS / TPR;      // rows in flight per work-group
    static constexpr int E = V * VEC;              // elements of a row per lane
    static constexpr int CMAX = TPR * E;
};

// A lane's part of a row.  Vectors behind the row's end read channel 0 on, which is there, and count for nothing.
template <class C>
struct Lane {
    int c0[C::V];                    // first channel of a vector
    bool in[C::V];                   // it is in the row
    unsigned e[C::V];                // first element of it, from the first row of the work-group's pass on
    int shared[C::ODD ? C::V : 1];   // ODD: the leading elements of a vector that do not count in sums (all, behind the row)
    int rg;                          // the lane's row of the pass
    bool whole;                      // every vector of every lane is in the row
    __device__ __forceinline__ Lane(const int c)
    {
        const int t = threadIdx.x % C::TPR;
        rg = threadIdx.x / C::TPR;
        whole = c == C::CMAX;
#pragma unroll
        for (int v = 0; v < C::V; ++v) {
            const int start = (v * C::TPR + t) * C::VEC;
            in[v] = start < c;
            c0[v] = !in[v] ? 0 : C::ODD && start + C::VEC > c ? c - C::VEC : start;
            e[v] = (unsigned)(rg * c + c0[v]);
            if constexpr (C::ODD) shared[v] = in[v] ? start - c0[v] : C::VEC;
        }
    }
    // whether element j is this lane's in the sums
    __device__ __forceinline__ bool mine(const int j) const { return C::ODD ? j % C::VEC >= shared[j / C::VEC] : in[j / C::VEC]; }
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

// Sum over the lane's channels of term(j).
template <class C, class F>
__device__ __forceinline__ float lane_sum(const Lane<C>& l, F&& term)
{
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < C::V; ++v) {
        float a = 0.0f;
#pragma unroll
        for (int j = v * C::VEC; j < (v + 1) * C::VEC; ++j) {
            if constexpr (C::ODD) a += l.mine(j) ? term(j) : 0.0f;   // (a choice, not a product: the term may be infinite)
            else a += term(j);
        }
        if (l.whole) s += a;
        else s += l.in[v] ? a : 0.0f;
    }
    return s;
}

// Rows held as f[E] (and g[E]) become (f - mean) / sqrt(mean square of that + eps), without the mean for the rms form; returns
// the factors 1 / sqrt.  Two sums over registers: the squares are taken of differences from the mean, as the definition has it,
// so a mean that is large against the spread costs no digits.  Two rows at once share the steps of their sums.
template <class C>
__device__ __forceinline__ void normalise(RowSum<C>& sum, const Lane<C>& l, const bool first, float* f, const bool second, float* g, const bool layer,
                                          const float inv_c, const float eps, float& rstd_f, float& rstd_g)
{
    float a = 0.0f, b = 0.0f;
    if (layer) {
        if (first) a = lane_sum<C>(l, [&](int j) { return f[j]; });
        if (second) b = lane_sum<C>(l, [&](int j) { return g[j]; });
        sum.two(a, b);
        a *= inv_c;
        b *= inv_c;
        if (first)
#pragma unroll
            for (int j = 0; j < C::E; ++j) f[j] -= a;
        if (second)
#pragma unroll
            for (int j = 0; j < C::E; ++j) g[j] -= b;
        a = b = 0.0f;
    }
    if (first) a = lane_sum<C>(l, [&](int j) { return f[j] * f[j]; });
    if (second) b = lane_sum<C>(l, [&](int j) { return g[j] * g[j]; });
    sum.two(a, b);
    rstd_f = rsqrtf(a * inv_c + eps);
    rstd_g = rsqrtf(b * inv_c + eps);
    if (first)
#pragma unroll
        for (int j = 0; j < C::E; ++j) f[j] *= rstd_f;
    if (second)
#pragma unroll
        for (int j = 0; j < C::E; ++j) g[j] *= rstd_g;
}
template <class C>
__device__ __forceinline__ float normalise(RowSum<C>& sum, const Lane<C>& l, float* f, const bool layer, const float inv_c, const float eps)
{
    float a = 0.0f;
    if (layer) {
        a = sum.one(lane_sum<C>(l, [&](int j) { return f[j]; })) * inv_c;
#pragma unroll
        for (int j = 0; j < C::E; ++j) f[j] -= a;
    }
    const float rstd = rsqrtf(sum.one(lane_sum<C>(l, [&](int j) { return f[j] * f[j]; })) * inv_c + eps);
#pragma unroll
    for (int j = 0; j < C::E; ++j) f[j] *= rstd;
    return rstd;
}

// A parameter vector's values of a lane's channels; `none` where there is no vector
template <class C>
__device__ __forceinline__ void load_params(const float* p, const Lane<C>& l, const float none, float* f)
{
#pragma unroll
    for (int j = 0; j < C::E; ++j) f[j] = p != nullptr ? p[l.c0[j / C::VEC] + j % C::VEC] : none;
}
// A lane's part of a map's row: `pass` is the (uniform) first row of the pass, `back` the elements by which lanes behind the last
// row step back to it.
template <class C>
__device__ __forceinline__ void load_row(const char* pass, const Lane<C>& l, const unsigned back, rows_u32x4* q)
{
#pragma unroll
    for (int v = 0; v < C::V; ++v) q[v] = C::Vec::load(pass + (size_t)((l.e[v] - back) * C::SIZE));
}
template <class C>
__device__ __forceinline__ void store_row(char* pass, const Lane<C>& l, const float* f)
{
#pragma unroll
    for (int v = 0; v < C::V; ++v)
        if (l.in[v]) C::Vec::store(pass + (size_t)(l.e[v] * C::SIZE), C::Vec::pack(f + v * C::VEC));
}
template <class C>
__device__ __forceinline__ void unpack_row(const rows_u32x4* q, float* f)
{
#pragma unroll
    for (int v = 0; v < C::V; ++v) C::Vec::unpack(q[v], f + v * C::VEC);
}
// the gate map's row where it is fp32 beside bf16 maps
template <class C>
__device__ __forceinline__ void load_gate_f32(const char* pass, const Lane<C>& l, const unsigned back, float* g)
{
#pragma unroll
    for (int j = 0; j < C::E; ++j) g[j] = ((const float*)pass)[l.e[j / C::VEC] - back + j % C::VEC];
}

// 1 / (1 + 2^(-x log2 e)) on the hardware's exponential and reciprocal, each good to one unit in the last place: the product's
// rounding costs |x| 2^-24 of the exponential, 2^-20 of a gate where it is still 10^-7 (library expf and an IEEE division are
// 25 instructions more an element: with a gate map, half of the backward pass)
__device__ __forceinline__ float sigmoid_f32(const float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }

}  // namespace
