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

}  // namespace tropnn_b200
