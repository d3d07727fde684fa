// Whole weights of logits, round(2^42 2^t): sums of them do not depend on their order.
#pragma once
#include "common.h"

namespace dsalt {

namespace {

constexpr unsigned long long kUnit = 1ull << 42;  // sums over 2^20 tokens stay below 2^62

// 2^42 (2^f - 1) = f P(f) for f in [-1/2, 1/2], P the degree 9 polynomial through the ten Chebyshev nodes (relative
// error of 2^f below 2^-50)
__device__ constexpr double kPow2[10] = {0x1.62e42fefa39f7p41, 0x1.ebfbdff82c590p39, 0x1.c6b08d7044119p37, 0x1.3b2ab6fba385fp35,
                                         0x1.5d87fe908f88ap32, 0x1.4309130378460p29, 0x1.ffcb76789860fp25, 0x1.62bfe46117445p22,
                                         0x1.b6571de2f2351p18, 0x1.e5e9f548e5725p14};

// x f + c with c in scalar registers (from vector registers it would be copied before each sum)
__device__ __forceinline__ double fma_s(double x, double f, double c) {
    double y;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(y) : "v"(x), "v"(f), "s"(c));
    return y;
}

// round(2^42 2^t) for t in [-60, 0].  (Sums with 1.5 2^52 and 2^52 round to a whole number and leave it in the mantissa.)
__device__ __forceinline__ unsigned long long whole_weight(double t) {
    const double s = t + 6755399441055744.0;
    const double f = t - (s - 6755399441055744.0);
    double y = kPow2[9];
#pragma unroll
    for (int k = 8; k >= 0; --k) y = fma_s(y, f, kPow2[k]);
    y = fma_s(y, f, 0x1p42);
    y = __hiloint2double(__double2hiint(y) + (__double2loint(s) << 20), __double2loint(y)) + 4503599627370496.0;
    return (unsigned long long)__double_as_longlong(y) & 0xfffffffffffffull;
}

}  // namespace

}  // namespace dsalt
