// What the kernels of the selective state space scan share: their arguments, how a warp lies over channels and states, and how a tile of tokens comes in.
//
//   s = softplus(dt) (or dt);   h_t[n] = exp(s a[c, n]) h_{t-1}[n] + s x_t B_t[n];   y_t = (sum_n C_t[n] h_t[n] + D x_t) silu(z_t)
//
// A lane owns four channels and NS states of each; LN lanes share the states, 32 / LN groups of lanes the channels.  So a number of B or C serves four channels and a step NS states,
// and what is summed over states or over channels is added up in the lane before it crosses lanes.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "special.cuh"

// x, dt, z, b, c: row r, token t starts at r * row + t * token (elements).  Null where a call has none: z, d, initial, last, checkpoints, starts, sums, positions, lengths, row_ids.
// With `heads` > 0 a channel is one of heads * dim, and the decay (a, dt, dt_bias, d) is a head's.
extern "C" struct dewb_selective_args {
  const void *x, *dt, *z, *b, *c;
  long long x_row, x_token, dt_row, dt_token, z_row, z_token, b_row, b_token, c_row, c_token;
  const float *a, *dt_bias, *d;        // [C, N] or [heads]; [heads]; [C] or [heads]
  const float* initial;                // [rows, C, N]; with positions, [store rows, C, N], and `last` is the same tensor
  float* last;
  void* y;                             // [R, T, C]
  float* checkpoints;                  // [R, ceil(T / EVERY), groups * padded, padded N]: the state in front of every EVERY tokens
  float *starts, *sums;                // [R, segments, groups * padded, padded N], [R, segments, groups * padded]: see scan_kernel
  const int *positions, *lengths, *row_ids;
  int R, T, C, N, groups, heads, segments, segment, padded, states_each;      // `padded`: channels of a group in checkpoints, starts and sums, a multiple of 128 (with heads, of 256);
                                       // `states_each`:
                                       // states of a lane where there are up to 16 (1, 2 or 4); of token_kernel, rows of a block
  int softplus, log_a, dt_fp32, stored;      // `stored`: rows of the store, where row_ids or positions name them
  int* status;                         // told of a row outside the store, which then has no tokens
};
static_assert(sizeof(dewb_selective_args) == 280, "packed by ops/selective.py");

namespace dewb {
namespace selective {

using bf16 = __nv_bfloat16;
using Args = dewb_selective_args;

constexpr int THREADS = 128, WARPS = 4;
constexpr int OUTSIDE = 6;             // the status of a row that the store does not have
constexpr int EVERY = 16;              // tokens between two kept states
using special::ex2;
using special::exp_minus_abs;
using special::gate;
using special::LN2;
using special::rcp;
using special::sigmoid;
using special::times_log2e;

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <int LN, int NS>
struct Lay {
  static constexpr int CG = 32 / LN;             // groups of lanes: four channels each
  static constexpr int CW = 4 * CG;              // channels of a warp
  static constexpr int CB = WARPS * CW;          // ... of a block
  static constexpr int NP = LN * NS;             // states, padded
  static constexpr int TT = 16;                  // tokens of a tile
  static constexpr int PASSES = TT >= LN ? TT / LN : 1;      // a lane's pieces of four channels in a tile: token lane / CG + pass * LN
};

// ln(1 + e^x) = max(x, 0) + ln(1 + t), t = e^-|x|: with q = t / (2 + t) <= 1/3, ln(1 + t) = 2 artanh q = 2 (q + q^3 / 3 + ... + q^13 / 13), the next term below 2e-8 of the sum
__device__ __forceinline__ float softplus(float x) {
  const float t = exp_minus_abs(x), q = t * rcp(2.f + t), r = q * q;
  float p = fmaf(r, 1.f / 13.f, 1.f / 11.f);
  p = fmaf(p, r, 1.f / 9.f);
  p = fmaf(p, r, 1.f / 7.f);
  p = fmaf(p, r, 1.f / 5.f);
  p = fmaf(p, r, 1.f / 3.f);
  p = fmaf(p, r, 1.f);
  return fmaf(2.f * q, p, fmaxf(x, 0.f));
}

// Two fp32 numbers side by side, of two neighbouring channels: one instruction for both.
struct f2 {
  unsigned long long v;
  __device__ __forceinline__ f2() {}
  __device__ __forceinline__ f2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ float2 get() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
};
__device__ __forceinline__ f2 mul(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ f2 fma(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ f2 ex2(f2 x) {
  const float2 t = x.get();
  return f2(ex2(t.x), ex2(t.y));
}
// n pairs that lie together
template <int N>
__device__ __forceinline__ void pairs(const float2* p, f2 (&v)[N]) {
  if constexpr (N == 1) {
    v[0].v = *reinterpret_cast<const unsigned long long*>(p);
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(p + k);
      v[k].v = t.x; v[k + 1].v = t.y;
    }
  }
}
__device__ __forceinline__ void pair(const float* p, f2& a, f2& b) {         // four numbers, 16 bytes
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  a.v = v.x; b.v = v.y;
}

__device__ __forceinline__ float ld(const float* p) { return *p; }
__device__ __forceinline__ float ld(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st(float* p, float v) { *p = v; }
__device__ __forceinline__ void st(bf16* p, float v) { *p = __float2bfloat16(v); }

// Four neighbouring values as they lie in memory, on their way.
template <typename T> struct Raw;
template <> struct Raw<bf16> {
  uint2 v;
  __device__ __forceinline__ void get(float (&f)[4]) const {
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
  }
};
template <> struct Raw<float> {
  uint4 v;
  __device__ __forceinline__ void get(float (&f)[4]) const {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
// A number as it lies in memory, and as fp32.
__device__ __forceinline__ uint32_t word(const float* p) { return __float_as_uint(*p); }
__device__ __forceinline__ uint32_t word(const bf16* p) { return *reinterpret_cast<const unsigned short*>(p); }
template <typename T>
__device__ __forceinline__ float value(uint32_t w) { return __uint_as_float(sizeof(T) == 2 ? w << 16 : w); }
__device__ __forceinline__ uint32_t bits(const bf16* p) { return *reinterpret_cast<const unsigned short*>(p); }

// `whole`: a vector load; else `n` (0 to 4) of the values, zeros behind.
__device__ __forceinline__ Raw<bf16> fetch(const bf16* p, bool whole, int n) {
  Raw<bf16> r{make_uint2(0u, 0u)};
  if (whole) { r.v = *reinterpret_cast<const uint2*>(p); return r; }
  if (n > 0) r.v.x = bits(p);
  if (n > 1) r.v.x |= bits(p + 1) << 16;
  if (n > 2) r.v.y = bits(p + 2);
  if (n > 3) r.v.y |= bits(p + 3) << 16;
  return r;
}
__device__ __forceinline__ Raw<float> fetch(const float* p, bool whole, int n) {
  Raw<float> r{make_uint4(0u, 0u, 0u, 0u)};
  const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
  if (whole) { r.v = *reinterpret_cast<const uint4*>(p); return r; }
  if (n > 0) r.v.x = q[0];
  if (n > 1) r.v.y = q[1];
  if (n > 2) r.v.z = q[2];
  if (n > 3) r.v.w = q[3];
  return r;
}
__device__ __forceinline__ void put(float* p, const float (&f)[4], bool whole, int n) {
  if (whole) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); return; }
#pragma unroll
  for (int j = 0; j < 4; ++j) if (j < n) p[j] = f[j];
}
__device__ __forceinline__ void put(bf16* p, const float (&f)[4], bool whole, int n) {
  if (whole) {
    __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) if (j < n) p[j] = __float2bfloat16(f[j]);
}

// Four values, each twice.
template <typename T>
__device__ __forceinline__ void twice(float2* to, const Raw<T>& r) {
  float f[4];
  r.get(f);
  reinterpret_cast<float4*>(to)[0] = make_float4(f[0], f[0], f[1], f[1]);
  reinterpret_cast<float4*>(to)[1] = make_float4(f[2], f[2], f[3], f[3]);
}

// Whether four values at multiples of four columns can be read as one piece.
template <typename T>
__host__ __device__ __forceinline__ bool fours(const void* p, long long row, long long token) {
  return (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0 && ((row | token) & 3) == 0;
}

// Sums of four channels' numbers over the LN lanes that share their states: the lane's result is that of channel `own_channel(lane)` (lanes with sl >= 4 hold copies).
template <int LN>
__device__ __forceinline__ float over_states(const float (&y)[4], int sl) {
  const bool b0 = sl & 1, b1 = sl & 2;
  const float p0 = (b0 ? y[2] : y[0]) + __shfl_xor_sync(0xffffffffu, b0 ? y[0] : y[2], 1);
  const float p1 = (b0 ? y[3] : y[1]) + __shfl_xor_sync(0xffffffffu, b0 ? y[1] : y[3], 1);
  float q = (b1 ? p1 : p0) + __shfl_xor_sync(0xffffffffu, b1 ? p0 : p1, 2);
#pragma unroll
  for (int o = 4; o < LN; o <<= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
  return q;
}
__device__ __forceinline__ int own_channel(int sl) { return (sl & 1) * 2 + ((sl >> 1) & 1); }

// The sum of `n` pieces of four, `stride` apart, from the `first` on and round (so that neighbouring lanes read from different banks).
__device__ __forceinline__ float4 sum4(const float4* p, int n, int stride, int first) {
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const float4 v = p[((i + first) & (n - 1)) * stride];
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  return s;
}

template <int LN>
__device__ __forceinline__ int turn_of(int lane) { return LN == 4 ? lane % 8 >> 1 : lane & 7; }

// Which tokens of row `row` a call has, and where its state lies.
struct Row {
  int len;             // live tokens
  bool held;           // a state to begin with
  long long at;        // row of `initial` and `last`
};
__device__ __forceinline__ Row row_of(const Args& p, int row) {
  if (p.positions == nullptr) return {p.T, p.initial != nullptr, row};
  const int first = p.positions[static_cast<long long>(row) * p.T], at = p.row_ids == nullptr ? row : p.row_ids[row];
  const bool inside = p.initial == nullptr || (at >= 0 && at < p.stored);
  if (!inside && p.status != nullptr) atomicExch(p.status, OUTSIDE);
  return {first < 0 || !inside ? 0 : max(0, min(p.lengths[row] - first, p.T)), p.initial != nullptr && first > 0, at};
}

inline bool args_ok(const Args& p) {
  if (p.R < 1 || p.T < 1 || p.C < 1 || p.N < 1 || p.groups < 1 || p.segments < 1 || p.segment < 1) return false;
  if (p.heads > 0 ? p.C % p.heads || p.heads % p.groups : p.groups != 1) return false;
  if (p.x == nullptr || p.dt == nullptr || p.b == nullptr || p.c == nullptr || p.a == nullptr || p.y == nullptr) return false;
  if (p.padded % (p.heads > 0 ? 256 : 128) || p.padded < p.C / p.groups || p.segment % EVERY || static_cast<long long>(p.segments) * p.segment < p.T || (p.segments > 1 && (p.starts == nullptr || p.sums == nullptr))) return false;
  return p.positions == nullptr || (p.lengths != nullptr && p.initial == p.last);
}

// A rate of minus infinity (a state without memory; what e^A_log gives from 88.8 on) becomes one of -1e30: a step of 0 (a token behind the row's end) or a sum of none leaves a decay of one, where
// 0 times infinity is no number, and every other step nothing, as the definition has it.
__device__ __forceinline__ float finite_rate(float a) { return a < -1e30f ? -1e30f : a; }
__device__ __forceinline__ float rate_of(const Args& p, float a) { return finite_rate(p.log_a ? -expf(a) : a); }

// The rate of channel c's state n times log2 e, 0 outside.
template <bool HEADS>
__device__ __forceinline__ float rate(const Args& p, int c, int n, int dim) {
  if (c >= p.C || n >= p.N) return 0.f;
  return times_log2e(rate_of(p, p.a[HEADS ? c / dim : static_cast<long long>(c) * p.N + n]));
}

}  // namespace selective
}  // namespace dewb
