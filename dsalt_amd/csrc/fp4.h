// e2m1 numbers (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign) and the power-of-two scales of the 4-bit cache, one for 32 of them,
// held as the exponent above -127 (255: NaN).  The conversions take that exponent from a float32 of it.
#pragma once
#include "common.h"

namespace dsalt {

typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float e8m0(uint32_t byte) { return __uint_as_float(byte << 23); }

// The exponent of 32 elements whose largest magnitude is amax (finite, >= 0): that of the least power of two s in
// [2^-126, 2^125] with amax <= 7 s.  (Elements past 6 s become 6 s, off by s at most, as those between 4 s and 6 s are; with
// all within 6 s half of the scales would be twice as large, and every smaller element's step with them.)
__device__ __forceinline__ uint32_t e8m0_of(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 2 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // 7 = 1.75 2^2
    return (uint32_t)min(max(e, 1), 252);
}

// eight elements over the scale 2^e, rounded to the nearest code, ties to the even one
__device__ __forceinline__ uint32_t to_e2m1_x8(const float* x, float scale) {
    uint32_t u = 0;
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[0], x[1], scale, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[2], x[3], scale, 1);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[6], x[7], scale, 3);
}

// eight codes as float32
__device__ __forceinline__ void e2m1_x8(uint32_t u, float scale, float* f) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 3);
    f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1], f[4] = c[0], f[5] = c[1], f[6] = d[0], f[7] = d[1];
}

// two codes (byte B of u) as bfloat16, exact
template <int B>
__device__ __forceinline__ uint32_t e2m1_bf16(uint32_t u, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, B));
}
// eight codes as a matrix operand
__device__ __forceinline__ bf16x8 e2m1_op(uint32_t u, float scale) {
    return __builtin_bit_cast(bf16x8, u32x4{e2m1_bf16<0>(u, scale), e2m1_bf16<1>(u, scale), e2m1_bf16<2>(u, scale),
                                            e2m1_bf16<3>(u, scale)});
}

}  // namespace dsalt
