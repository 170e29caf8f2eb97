// The special-function unit's exponential and reciprocal (2^-22 and 2^-23 of the result), and the sigmoid made of them: a sixth of the instructions of expf and a division, for kernels
// that would else be bound by issuing them.
#pragma once

namespace dewb {
namespace special {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-LOG2E * x)); }

}  // namespace special
}  // namespace dewb
