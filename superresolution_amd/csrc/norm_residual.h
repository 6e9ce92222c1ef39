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

// mean (0 for the rms form) and 1 / sqrt(mean square of what is left + eps) of a row held as f[E]; elements from nv[v] on do
// not exist and are 0.  Two sums over registers: the squares are taken of differences from the mean, as the definition has
// it, so a mean that is large against the spread costs no digits.
template <class C>
__device__ __forceinline__ void row_statistics(RowSum<C>& sum, const float* f, const int* nv, const bool layer, const float inv_c, const float eps,
                                               float& mean, float& rstd)
{
    mean = 0.0f;
    if (layer) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < C::E; ++j) s += f[j];
        mean = sum.one(s) * inv_c;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < C::E; ++j) {
        const float d = f[j] - mean;
        q += j % C::VEC < nv[j / C::VEC] ? d * d : 0.0f;
    }
    rstd = 1.0f / sqrtf(sum.one(q) * inv_c + eps);
}

// `nv` floats of a parameter vector from channel c0 on; absent channels and an absent vector give `none`
template <class C>
__device__ __forceinline__ void load_params(const float* p, const int c0, const int nv, const float none, float* f)
{
#pragma unroll
    for (int j = 0; j < C::VEC; ++j) f[j] = p != nullptr && j < nv ? p[c0 + j] : none;
}

__device__ __forceinline__ float sigmoid_f32(const float x) { return 1.0f / (1.0f + expf(-x)); }

}  // namespace
