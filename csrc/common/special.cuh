// The special-function unit's exponential and reciprocal (2^-22 and 2^-23 of the result), and e^-|x| and the sigmoid made of them, for kernels that would else be bound by issuing expf and
// a division.
//
// A rounded product x log2 e costs |x| 2^-24 of 2^(x log2 e), so e^-|x| takes what that product and the constant lost along: 2^(hi + lo) = 2^hi (1 + lo ln 2), lo below 2^-17.  Logits from
// -86 to 80, in units of 2^-24 of the result: sigmoid and softplus (selective.cuh) off by MEASURED at most; with the rounded product alone by 64.  Below -87 e^-|x| is 0.
#pragma once

namespace dewb {
namespace special {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOG2E_LOW = static_cast<float>(1.4426950408889634074 - static_cast<double>(LOG2E));

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
__device__ __forceinline__ float exp_minus(float x) {        // e^-|x|
  float m = fabsf(x);
  m = m > 128.f ? 128.f : m;                                  // (an infinite product would lose an infinite rest; no number stays none)
  const float hi = -LOG2E * m, lo = fmaf(-LOG2E, m, -hi) - LOG2E_LOW * m, t = ex2(hi);
  return fmaf(t, LN2 * lo, t);
}
__device__ __forceinline__ float sigmoid(float x) {
  const float t = exp_minus(x), r = rcp(1.f + t);
  return x < 0.f ? t * r : r;
}

}  // namespace special
}  // namespace dewb
