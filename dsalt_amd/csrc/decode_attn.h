// What the attention kernels over the paged caches share: operands, weights and the join of a split row.
#pragma once
#include "common.h"

namespace dsalt {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// number of bfloat16 parts of a query element (exact: 8, 11 and 24 bits) and of a weight over the 8-bit cache: 16 bits of it for
// 16-bit outputs, whose own rounding, half a step of 2^-8 or 2^-11 of a value, is far coarser, 24 for float32 (lists keep
// weights in float32)
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int q = 1, p = 2; };
template <> struct Parts<f16> { static constexpr int q = 2, p = 2; };
template <> struct Parts<float> { static constexpr int q = 3, p = 3; };

__device__ __forceinline__ uint32_t half_pair(uint32_t a, uint32_t b, bool hi) {  // halves of a and b side by side
    return __builtin_amdgcn_perm(b, a, hi ? 0x07060302u : 0x05040100u);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32: to 1 ulp, 0 below 2^-126

// eight elements of a 16-byte aligned row as floats
template <typename T>
__device__ __forceinline__ void load8(const T* x, float* f) {
    typedef T vec __attribute__((ext_vector_type(8), aligned(16)));
    const vec v = *(const vec*)x;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = to_float(v[e]);
}

// eight floats into PARTS bfloat16 operands that sum to them
template <int PARTS>
__device__ __forceinline__ void split8(const float* x, bf16x8* o) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float r = x[e];
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
            const bf16 h = (bf16)r;
            o[k][e] = h;
            r -= (float)h;
        }
    }
}

// The splits of a row and head joined: a block each, its waves over the splits, a lane D / 64 elements.
constexpr int kJoinWaves = 8;

template <typename T, int D, typename Params>
__global__ __launch_bounds__(64 * kJoinWaves) void cache_attn_join_kernel(Params p, int ns) {
    constexpr int E = D / 64;
    typedef float vec __attribute__((ext_vector_type(E)));
    __shared__ vec outs[kJoinWaves][64];
    __shared__ float sums[kJoinWaves];
    const int64_t th = blockIdx.x;
    const int t = (int)(th / p.n_heads), h = (int)(th - (int64_t)t * p.n_heads), lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const float2* ml = (const float2*)p.ws + th * ns;
    const float* acc = (const float*)p.ws + 2 * (int64_t)p.n_rows * p.n_heads * ns + th * ns * D + lane * E;
    float M = -INFINITY, L = 0.f;
    for (int k = lane; k < ns; k += 64) M = fmaxf(M, ml[k].x);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, wave_xor(M, o));
    const float mb = M == -INFINITY ? 0.f : M;
    vec o = {};
#pragma unroll 4
    for (int k = wv; k < ns; k += kJoinWaves) {
        const float2 v = ml[k];
        const vec x = *(const vec*)(acc + (int64_t)k * D);
        const float f = v.x == -INFINITY ? 1.f : exp2_(v.x - mb);
        L += v.y == 0.f ? 0.f : v.y * f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += v.y == 0.f ? 0.f : x[e] * f;  // (a split with sum 0 wrote no values)
    }
    outs[wv][lane] = o;
    if (lane == 0) sums[wv] = L;
    __syncthreads();
    if (wv == 0) {
        for (int k = 1; k < kJoinWaves; ++k) {
            o += outs[k][lane];
            L += sums[k];
        }
        T* y = (T*)p.out + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = from_float<T>(L == 0.f ? 0.f : o[e] / L);
        if (lane == 0) p.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    }
}

}  // namespace

}  // namespace dsalt
