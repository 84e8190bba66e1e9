// Two f32 lanes in one instruction (f32x2 of sm_100), and the approximate exponential and reciprocal.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tropnn_b200 {

__device__ __forceinline__ uint64_t bits2(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 float2_of(uint64_t r) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ float2 mul2(float2 x, float2 y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(x)), "l"(bits2(y)));
  return float2_of(r);
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(x)), "l"(bits2(y)));
  return float2_of(r);
}
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(x)), "l"(bits2(y)), "l"(bits2(z)));
  return float2_of(r);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// 2^x to 2 ulp (a flushed result below 2^-126), 1 / x to 1 ulp.
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 2^x for x <= 0 on the FMA and integer pipes, to 2.2e-7 of it (0 below 2^-126.5): x = n + f with n whole
// and |f| <= 1/2, 2^f by the polynomial of degree 5 that is closest to it in relative error (7.5e-8,
// fitted by iteratively reweighted least squares on Chebyshev nodes), times 2^n put together from its
// bits. Adding 1.5 * 2^23 rounds x to n and leaves n in the sum's low bits.
__device__ __forceinline__ float2 exp2_poly2(float2 x) {
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x.x) : "f"(x.x), "f"(-127.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x.y) : "f"(x.y), "f"(-127.f));
  const float2 t = add2(x, both(12582912.f)), n = add2(t, both(-12582912.f)), f = fma2(n, both(-1.f), x);
  float2 p = fma2(f, both(0.001327647129073739f), both(0.009675540961325169f));
  p = fma2(p, f, both(0.05550713092088699f));
  p = fma2(p, f, both(0.24022120237350464f));
  p = fma2(p, f, both(0.6931469440460205f));
  p = fma2(p, f, both(1.0000001192092896f));
  const float2 scale = make_float2(__int_as_float(__float_as_int(t.x) * (1 << 23) + 0x3F800000),
                                   __int_as_float(__float_as_int(t.y) * (1 << 23) + 0x3F800000));
  return mul2(p, scale);
}

}  // namespace tropnn_b200
