// 2^x on the FMA pipe, for kernels whose special-function unit is busy.
#pragma once

#include "common.cuh"

namespace b200q {

// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of a pair on the FMA pipe, x < 128: x = n + f with n the nearest integer (Cody and Waite's reduction; the rounding constant
// 1.5 * 2^23 is raised by 127, so that the low bits of the sum are the biased exponent of 2^n), 2^f by the polynomial of degree 6
// with constant term 1 of the smallest largest relative error on [-1/2, 1/2] (2.0e-9, from a weighted least-squares exchange).  With
// the fp32 roundings of Horner's scheme: largest relative error 7.9e-8, root mean square 2.7e-8, mean 9e-10; ex2.approx over the same
// range [-20, 9]: 1.4e-7, 5.5e-8, -2.4e-8.  Below -126.5 the result is 0; NaN stays NaN.
__device__ __forceinline__ uint64_t ex2_poly2(uint64_t x) {
  constexpr float kRound = 12582912.0f + 127.0f;
  const auto both = [](float c) { return pack2(c, c); };
  const float2 a = unpack2(x);
  x = pack2(max_nan(a.x, -127.0f), max_nan(a.y, -127.0f));
  const uint64_t t = add2(x, both(kRound));
  const uint64_t f = add2(x, fma2(t, both(-1.0f), both(kRound)));
  uint64_t y = fma2(f, both(0x1.41fbbcp-13f), both(0x1.5f3e54p-10f));
  y = fma2(y, f, both(0x1.3b2d4cp-7f));
  y = fma2(y, f, both(0x1.c6aee8p-5f));
  y = fma2(y, f, both(0x1.ebfbdcp-3f));
  y = fma2(y, f, both(0x1.62e430p-1f));
  y = fma2(y, f, both(1.0f));
  const float2 n = unpack2(t);
  return mul2(y, pack2(__uint_as_float(__float_as_uint(n.x) << 23), __uint_as_float(__float_as_uint(n.y) << 23)));
}

}  // namespace b200q
