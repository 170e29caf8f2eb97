// The special-function unit's exponential and reciprocal (2^-22 and 2^-23 of the result), and e^-x and the sigmoid made of them, for kernels that would else be bound by issuing expf and a
// division.
//
// A rounded product x log2 e costs |x| 2^-24 of 2^(x log2 e), so e^-x takes along what that product lost: with p = -x log2 e rounded, e^-x = 2^p (1 + r), r = -x - p ln 2, below 2^-16.
// Logits from -86 to 80, in units of 2^-24 of the result: sigmoid off by 5 at most, softplus (selective.cuh) by 7; with the rounded product alone by 64.  Results in bf16, whose half step is
// 2^16 such units, take that (`gate`): 8192 rows of 8192 values through the norm both ways 220 us, 242 with the remainder.
#pragma once

namespace dewb {
namespace special {

constexpr double LN2_EXACT = 0.69314718055994530942, LOG2E_EXACT = 1.4426950408889634074;
constexpr float LOG2E = static_cast<float>(LOG2E_EXACT), LOG2E_LOW = static_cast<float>(LOG2E_EXACT - LOG2E);
constexpr float LN2 = static_cast<float>(LN2_EXACT), LN2_LOW = static_cast<float>(LN2_EXACT - LN2);

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
__device__ __forceinline__ float times_log2e(float x) { return fmaf(x, LOG2E, x * LOG2E_LOW); }      // rounded once
// e^-x of a finite x
__device__ __forceinline__ float exp_minus(float x) {
  const float p = -LOG2E * x, t = ex2(p);
  return fmaf(t, fmaf(p, -LN2_LOW, fmaf(p, -LN2, -x)), t);
}
// (within a finite number of either end; what is no number stays none)
__device__ __forceinline__ float at_most(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float at_least(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float exp_minus_abs(float x) { return exp_minus(at_most(fabsf(x), 128.f)); }             // (0 from 88 on)
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + exp_minus(at_most(at_least(x, -88.7f), 128.f))); }      // (0 up to -88)
// ... of a gate whose results have type T
template <typename T>
__device__ __forceinline__ float gate(float x) { return sizeof(T) == 2 ? rcp(1.f + ex2(-LOG2E * x)) : sigmoid(x); }

}  // namespace special
}  // namespace dewb
