// e4m3 numbers (3 mantissa bits, subnormal step 2^-9, largest 448, no infinities, NaN 0x7f) and the
// power-of-two scales of the 8-bit cache.
#pragma once
#include "common.h"

namespace dsalt {

typedef float floatx2 __attribute__((ext_vector_type(2)));

// four e4m3 codes as float32
__device__ __forceinline__ void e4m3_x4(uint32_t u, float* f) {
    const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false);
    const floatx2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
    f[0] = a[0];
    f[1] = a[1];
    f[2] = b[0];
    f[3] = b[1];
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// four float32 values rounded to e4m3 (ties to even, past 448 to 448, not finite to NaN)
__device__ __forceinline__ uint32_t to_e4m3_x4(float a, float b, float c, float d) {
    auto in = [](float x) { return finite(x) ? fminf(fmaxf(x, -448.f), 448.f) : 0.f; };
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(in(a), in(b), 0, false);
    u = __builtin_amdgcn_cvt_pk_fp8_f32(in(c), in(d), u, true);
    if (!finite(a)) u |= 0x7f;
    if (!finite(b)) u |= 0x7f << 8;
    if (!finite(c)) u |= 0x7f << 16;
    if (!finite(d)) u |= 0x7f << 24;
    return (uint32_t)u;
}

// the least power of two s in [2^-126, 2^119] with amax <= 448 s (448 = 1.75 2^8), amax finite and >= 0
__device__ __forceinline__ float scale_of(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float((uint32_t)(min(max(e, -126), 119) + 127) << 23);
}

}  // namespace dsalt
