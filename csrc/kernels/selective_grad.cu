// Gradients of the selective state space scan, for sm_100a (the equations and the lanes' layout: selective.cuh).  With u = s x, w = dy silu(z) and a_t = exp(s_t A):
//
//   g_t = w_t C_t + a_{t+1} g_{t+1}  (from the gradient of the last state)         dC_t[n] = sum_c w h          dB_t[n] = sum_c u g
//   dx = s sum_n g B + D w       ds = x sum_n g B + sum_n A q,  q = g a h_{t-1}     dA = sum_t s q               dD = sum_t w x       dz = dy (sum_n C h + D x) silu'(z)
//
//   back_ends_kernel  with several segments: what each makes of a gradient of zeros at its end
//   grad_kernel       sixteen tokens at a time, from the last on: the states again from the one that the forward kept in front of them (they stand in shared memory, eight tokens'
//                     at a time), then the tokens backwards with g in registers.  Sums over channels leave a block as parts, so the result has one order whatever runs first
//   grad_sum_kernel   adds up the parts
//
// All in fp32; inputs and gradients are bf16 or fp32 (template T; the steps' logits either).  Compiled without fast math.
#include "../common/selective.cuh"

// `f`: what the forward was given (f.y is not read), with its checkpoints.  starts and sums are this pass's own.
extern "C" struct dewb_selective_grad_args {
  dewb_selective_args f;
  const void* dy;
  long long dy_row, dy_token;
  const float* dlast;                  // [R, C, N] or null
  void *dx, *ddt, *dz;                 // [R, T, C]; dz null where the call has no gate
  void *db, *dc;                       // [R, T, N]
  float *da, *dd, *dinitial;           // [C, N], [C], [R, C, N]; dd and dinitial may be null
  float *bc_parts, *a_parts, *d_parts; // [channel blocks, R * T, 2, padded N], [R * segments, padded C, padded N], [R * segments, padded C]
};

namespace dewb {
namespace selective {

using Grad = dewb_selective_grad_args;
constexpr int HALF = 8;                // tokens whose states stand in shared memory together

template <int LN>
struct Shared {
  using L = Lay<LN, 4>;
  float step[WARPS][TT][L::CW], w[WARPS][TT][L::CW], c[TT][L::NP];               // s, w, C: what back_ends_kernel has
  float in[WARPS][TT][L::CW], b[TT][L::NP];                                      // u, B
  float sums[WARPS][HALF][3][L::CW];                                             // sum g B, sum A q, sum C h
  float bc[WARPS][TT][2][L::NP];
  float4 h[WARPS][HALF][4][32];                                                  // h_{t-1}: token, channel of the lane's four, lane
};

// Where a lane loads and stores: four channels of token lt + pass * LN.
template <typename T, int LN>
struct Place {
  using L = Lay<LN, 4>;
  int lt, lc, left;
  bool x_whole, dt_whole, z_whole, dy_whole, y_whole;
  const T *x, *z, *dy;
  long long dt_row;
  __device__ __forceinline__ Place(const Grad& g, int row, int c0, int lane) {
    const Args& p = g.f;
    lt = lane / L::CG;
    lc = c0 + lane % L::CG * 4;
    left = max(0, min(4, p.C - lc));
    x = static_cast<const T*>(p.x) + row * p.x_row + lc;
    z = p.z == nullptr ? nullptr : static_cast<const T*>(p.z) + row * p.z_row + lc;
    dy = static_cast<const T*>(g.dy) + row * g.dy_row + lc;
    dt_row = row * p.dt_row + lc;
    const bool even = left == 4;
    x_whole = even && fours<T>(p.x, p.x_row, p.x_token);
    z_whole = even && fours<T>(p.z, p.z_row, p.z_token);
    dy_whole = even && fours<T>(g.dy, g.dy_row, g.dy_token);
    dt_whole = even && (p.dt_fp32 ? fours<float>(p.dt, p.dt_row, p.dt_token) : fours<bf16>(p.dt, p.dt_row, p.dt_token));
    y_whole = even && (p.C & 3) == 0;
  }
};

// Sixteen tokens from t0 on: s, u and w of the warp's channels, B and C of the block.
template <typename T, int LN, bool STATES>
__device__ __forceinline__ void stage(Shared<LN>& sm, const Grad& g, const Place<T, LN>& at, int row, int t0, int t_end, int warp, int lane, float (&total)[4]) {
  using L = Lay<LN, 4>;
  const Args& p = g.f;
#pragma unroll
  for (int i = 0; i < L::PASSES; ++i) {
    const int t = at.lt + i * LN;
    const bool on = t < TT && t0 + t < t_end;
    const int n = on ? at.left : 0;
    const long long tok = t0 + t;
    float x[4], s[4], w[4], z[4];
    if (STATES) fetch(at.x + tok * p.x_token, on && at.x_whole, n).get(x);
    fetch_step(p.dt, at.dt_row + tok * p.dt_token, p.dt_fp32, on && at.dt_whole, n).get(s, p.dt_fp32);
    fetch(at.dy + tok * g.dy_token, on && at.dy_whole, n).get(w);
    if (at.z != nullptr) fetch(at.z + tok * p.z_token, on && at.z_whole, n).get(z);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j] = j < n ? (p.softplus ? softplus(s[j]) : s[j]) : 0.f;
      if (at.z != nullptr) w[j] *= z[j] * sigmoid(z[j]);
      total[j] += s[j];
    }
    if (t < TT) {
      const int c = lane % L::CG * 4;
      *reinterpret_cast<float4*>(&sm.step[warp][t][c]) = make_float4(s[0], s[1], s[2], s[3]);
      *reinterpret_cast<float4*>(&sm.w[warp][t][c]) = make_float4(w[0], w[1], w[2], w[3]);
      if (STATES) *reinterpret_cast<float4*>(&sm.in[warp][t][c]) = make_float4(s[0] * x[0], s[1] * x[1], s[2] * x[2], s[3] * x[3]);
    }
  }
  const T *b = static_cast<const T*>(p.b) + row * p.b_row, *c = static_cast<const T*>(p.c) + row * p.c_row;
  for (int i = threadIdx.x; i < TT * L::NP; i += THREADS) {
    const int t = i / L::NP, n = i % L::NP;
    const bool on = t0 + t < t_end && n < p.N;
    if (STATES) sm.b[t][n] = on ? ld(b + (t0 + t) * p.b_token + n) : 0.f;
    sm.c[t][n] = on ? ld(c + (t0 + t) * p.c_token + n) : 0.f;
  }
}

template <int LN>
__device__ __forceinline__ void load_rates(const Args& p, int c, int n, float (&a)[4][4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) a[j][k] = rate<false>(p, c + j, n + k, 1);
}

__device__ __forceinline__ void load4x4(const float* p, int stride, float (&h)[4][4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 v = *reinterpret_cast<const float4*>(p + static_cast<long long>(j) * stride);
    h[j][0] = v.x; h[j][1] = v.y; h[j][2] = v.z; h[j][3] = v.w;
  }
}
__device__ __forceinline__ void store4x4(float* p, int stride, const float (&h)[4][4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(p + static_cast<long long>(j) * stride) = make_float4(h[j][0], h[j][1], h[j][2], h[j][3]);
}

// grid R * (segments - 1) * channel blocks, of segments 1, 2, ...: starts[r, j] is the gradient of the state in front of segment j that the segment itself makes (the last one: with dlast).
template <typename T, int LN>
__global__ void __launch_bounds__(THREADS)
back_ends_kernel(const Grad g) {
  using L = Lay<LN, 4>;
  __shared__ __align__(16) char raw[offsetof(Shared<LN>, in)];
  Shared<LN>& sm = *reinterpret_cast<Shared<LN>*>(raw);
  const Args& p = g.f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sl = lane % LN, cg = lane / LN;
  const int blocks = (p.C + L::CB - 1) / L::CB, padded = blocks * L::CB;
  const int cb = blockIdx.x % blocks, seg = 1 + blockIdx.x / blocks % (p.segments - 1), row = blockIdx.x / blocks / (p.segments - 1);
  const int c0 = cb * L::CB + warp * L::CW, t_begin = seg * p.segment, t_end = min(p.T, t_begin + p.segment);
  const Place<T, LN> at(g, row, c0, lane);
  float a[4][4], d[4][4], total[4] = {0.f, 0.f, 0.f, 0.f};
  load_rates<LN>(p, c0 + cg * 4, sl * 4, a);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = c0 + cg * 4 + j, n = sl * 4 + k;
      d[j][k] = seg == p.segments - 1 && g.dlast != nullptr && c < p.C && n < p.N ? g.dlast[(static_cast<long long>(row) * p.C + c) * p.N + n] : 0.f;
    }
  for (int t0 = t_begin + (t_end - t_begin - 1) / TT * TT; t0 >= t_begin; t0 -= TT) {
    __syncthreads();
    stage<T, LN, false>(sm, g, at, row, t0, t_end, warp, lane, total);
    __syncthreads();
#pragma unroll 4
    for (int t = min(TT, t_end - t0) - 1; t >= 0; --t) {
      const float4 s4 = *reinterpret_cast<const float4*>(&sm.step[warp][t][cg * 4]), w4 = *reinterpret_cast<const float4*>(&sm.w[warp][t][cg * 4]);
      const float4 c4 = *reinterpret_cast<const float4*>(&sm.c[t][sl * 4]);
      const float s[4] = {s4.x, s4.y, s4.z, s4.w}, w[4] = {w4.x, w4.y, w4.z, w4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) d[j][k] = ex2(s[j] * a[j][k]) * fmaf(w[j], c[k], d[j][k]);
    }
  }
  const long long out = (static_cast<long long>(row) * p.segments + seg) * padded + c0;
  store4x4(p.starts + (out + cg * 4) * L::NP + sl * 4, L::NP, d);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int o = L::CG; o < 32; o <<= 1) total[j] += __shfl_xor_sync(0xffffffffu, total[j], o);
    if (at.lt == 0) p.sums[out + lane % L::CG * 4 + j] = total[j];
  }
}

// Eight numbers of a lane (dB and dC of its four states) summed over the 32 / LN groups of lanes: lane keeps COUNT = 8 / groups of them, from `base` on.
template <int LN>
__device__ __forceinline__ int over_channels(float (&v)[8], int lane) {
  int base = 0;
#pragma unroll
  for (int o = LN, half = 4; o < 32; o <<= 1, half >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < half) {
        const float give = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    }
    base += upper ? half : 0;
  }
  return base;
}

template <typename T, int LN>
__global__ void __launch_bounds__(THREADS)
grad_kernel(const Grad g) {
  using L = Lay<LN, 4>;
  constexpr int CG = L::CG, NP = L::NP, COUNT = 8 / CG;
  extern __shared__ __align__(16) char raw[];
  Shared<LN>& sm = *reinterpret_cast<Shared<LN>*>(raw);
  const Args& p = g.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sl = lane % LN, cg = lane / LN;
  const int blocks = (p.C + L::CB - 1) / L::CB, padded = blocks * L::CB;
  const int cb = blockIdx.x % blocks, seg = blockIdx.x / blocks % p.segments, row = blockIdx.x / blocks / p.segments;
  const int c0 = cb * L::CB + warp * L::CW, t_begin = seg * p.segment, t_end = min(p.T, t_begin + p.segment);
  const Place<T, LN> at(g, row, c0, lane);
  const long long pad_row = static_cast<long long>(row) * p.segments * padded + c0 + cg * 4;
  float a[4][4], d[4][4], da[4][4];
  load_rates<LN>(p, c0 + cg * 4, sl * 4, a);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = c0 + cg * 4 + j, n = sl * 4 + k;
      da[j][k] = 0.f;
      d[j][k] = seg == p.segments - 1 && g.dlast != nullptr && c < p.C && n < p.N ? g.dlast[(static_cast<long long>(row) * p.C + c) * p.N + n] : 0.f;
    }
  for (int q = p.segments - 1; q > seg; --q) {    // what comes from behind the segment
    float e[4][4];
    load4x4(p.starts + (pad_row + static_cast<long long>(q) * padded) * NP + sl * 4, NP, e);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float sum = q < p.segments - 1 ? p.sums[pad_row + static_cast<long long>(q) * padded + j] : 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) d[j][k] = ex2(sum * a[j][k]) * d[j][k] + e[j][k];
    }
  }
  float skip[4], dd[4] = {0.f, 0.f, 0.f, 0.f}, unused[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) skip[j] = p.d != nullptr && j < at.left ? p.d[at.lc + j] : 0.f;
  const int kept = (p.T + EVERY - 1) / EVERY;
  const long long here = static_cast<long long>(row) * p.T * p.C + at.lc;
  for (int t0 = t_begin + (t_end - t_begin - 1) / TT * TT; t0 >= t_begin; t0 -= TT) {
    stage<T, LN, true>(sm, g, at, row, t0, t_end, warp, lane, unused);
    __syncthreads();
    const float* before = p.checkpoints + ((static_cast<long long>(row) * kept + t0 / EVERY) * padded + c0 + cg * 4) * NP + sl * 4;
    const int count = min(TT, t_end - t0);
    for (int half = count > HALF ? 1 : 0; half >= 0; --half) {
      const int from = half * HALF, n_here = min(HALF, count - from);
      float h[4][4];
      load4x4(before, NP, h);
      auto forth = [&](int t) {
        const float4 s4 = *reinterpret_cast<const float4*>(&sm.step[warp][t][cg * 4]), u4 = *reinterpret_cast<const float4*>(&sm.in[warp][t][cg * 4]);
        const float4 b4 = *reinterpret_cast<const float4*>(&sm.b[t][sl * 4]);
        const float s[4] = {s4.x, s4.y, s4.z, s4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) h[j][k] = fmaf(ex2(s[j] * a[j][k]), h[j][k], u[j] * b[k]);
      };
#pragma unroll 2
      for (int t = 0; t < from; ++t) forth(t);
#pragma unroll 2
      for (int t = 0; t < n_here; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sm.h[warp][t][j][lane] = make_float4(h[j][0], h[j][1], h[j][2], h[j][3]);
        if (t + 1 < n_here) forth(from + t);
      }
#pragma unroll 1
      for (int i = n_here - 1; i >= 0; --i) {
        const int t = from + i;
        const float4 s4 = *reinterpret_cast<const float4*>(&sm.step[warp][t][cg * 4]), u4 = *reinterpret_cast<const float4*>(&sm.in[warp][t][cg * 4]);
        const float4 w4 = *reinterpret_cast<const float4*>(&sm.w[warp][t][cg * 4]);
        const float4 b4 = *reinterpret_cast<const float4*>(&sm.b[t][sl * 4]), c4 = *reinterpret_cast<const float4*>(&sm.c[t][sl * 4]);
        const float s[4] = {s4.x, s4.y, s4.z, s4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w}, w[4] = {w4.x, w4.y, w4.z, w4.w};
        const float b[4] = {b4.x, b4.y, b4.z, b4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
        float bc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, s1[4], s2[4], s3[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 v = sm.h[warp][i][j][lane];
          const float hp[4] = {v.x, v.y, v.z, v.w};
          s1[j] = s2[j] = s3[j] = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float e = ex2(s[j] * a[j][k]), ah = e * hp[k], now = fmaf(u[j], b[k], ah);
            d[j][k] = fmaf(w[j], c[k], d[j][k]);
            bc[k] = fmaf(u[j], d[j][k], bc[k]);
            bc[4 + k] = fmaf(w[j], now, bc[4 + k]);
            s1[j] = fmaf(d[j][k], b[k], s1[j]);
            s3[j] = fmaf(now, c[k], s3[j]);
            const float q = d[j][k] * ah;
            s2[j] = fmaf(q, a[j][k], s2[j]);
            da[j][k] = fmaf(q, s[j], da[j][k]);
            d[j][k] *= e;
          }
        }
        const int own = cg * 4 + own_channel(sl);
        const float r1 = over_states<LN>(s1, sl), r2 = over_states<LN>(s2, sl), r3 = at.z != nullptr ? over_states<LN>(s3, sl) : 0.f;
        if (sl < 4) {
          sm.sums[warp][i][0][own] = r1;
          sm.sums[warp][i][1][own] = r2;
          sm.sums[warp][i][2][own] = r3;
        }
        const int base = over_channels<LN>(bc, lane);
#pragma unroll
        for (int q = 0; q < COUNT; ++q) sm.bc[warp][t][(base + q) / 4][sl * 4 + (base + q) % 4] = bc[q];
      }
      __syncwarp();
#pragma unroll
      for (int pass = 0; pass < (HALF + LN - 1) / LN; ++pass) {
        const int i = at.lt + pass * LN, t = from + i;
        if (i >= n_here) continue;
        const long long tok = t0 + t;
        float x[4], raw_step[4], dx[4], ds[4], dy[4], z[4];
        fetch(at.x + tok * p.x_token, at.x_whole, at.left).get(x);
        if (p.softplus) fetch_step(p.dt, at.dt_row + tok * p.dt_token, p.dt_fp32, at.dt_whole, at.left).get(raw_step, p.dt_fp32);
        const int c = lane % CG * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float r1 = sm.sums[warp][i][0][c + j], w = sm.w[warp][t][c + j];
          dx[j] = fmaf(sm.step[warp][t][c + j], r1, skip[j] * w);
          ds[j] = fmaf(x[j], r1, LN2 * sm.sums[warp][i][1][c + j]);
          if (p.softplus) ds[j] *= sigmoid(raw_step[j]);
          dd[j] = fmaf(w, x[j], dd[j]);
        }
        put(static_cast<T*>(g.dx) + here + tok * p.C, dx, at.y_whole, at.left);
        if (p.dt_fp32) put(static_cast<float*>(g.ddt) + here + tok * p.C, ds, at.y_whole, at.left);
        else put(static_cast<bf16*>(g.ddt) + here + tok * p.C, ds, at.y_whole, at.left);
        if (at.z != nullptr) {
          fetch(at.dy + tok * g.dy_token, at.dy_whole, at.left).get(dy);
          fetch(at.z + tok * p.z_token, at.z_whole, at.left).get(z);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float sig = sigmoid(z[j]);
            z[j] = dy[j] * fmaf(skip[j], x[j], sm.sums[warp][i][2][c + j]) * sig * fmaf(z[j], 1.f - sig, 1.f);
          }
          put(static_cast<T*>(g.dz) + here + tok * p.C, z, at.y_whole, at.left);
        }
      }
      __syncwarp();                               // (the sums and states have been read)
    }
    __syncthreads();
    for (int i = tid; i < count * 2 * NP; i += THREADS) {
      const int t = i / (2 * NP), q = i % (2 * NP);
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) v += sm.bc[k][t][q / NP][q % NP];
      g.bc_parts[((static_cast<long long>(cb) * p.R + row) * p.T + t0 + t) * (2 * NP) + q] = v;
    }
  }
  const long long part = (static_cast<long long>(row) * p.segments + seg) * padded + c0;
  store4x4(g.a_parts + (part + cg * 4) * NP + sl * 4, NP, da);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int o = CG; o < 32; o <<= 1) dd[j] += __shfl_xor_sync(0xffffffffu, dd[j], o);
    if (at.lt == 0) g.d_parts[part + lane % CG * 4 + j] = dd[j];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = c0 + cg * 4 + j, n = sl * 4 + k;
      if (seg == 0 && g.dinitial != nullptr && c < p.C && n < p.N) g.dinitial[(static_cast<long long>(row) * p.C + c) * p.N + n] = d[j][k];
    }
  }
}

// A thread a number: dB and dC, then dA, then dD.
template <typename T>
__global__ void __launch_bounds__(256)
grad_sum_kernel(const Grad g, int blocks, int padded, int np) {
  const Args& p = g.f;
  const long long tokens = static_cast<long long>(p.R) * p.T, nbc = tokens * 2 * p.N, na = static_cast<long long>(p.C) * p.N;
  long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i < nbc) {
    const long long tok = i / (2 * p.N);
    const int q = static_cast<int>(i - tok * 2 * p.N), which = q / p.N, n = q % p.N;
    const float* v = g.bc_parts + tok * 2 * np + which * np + n;
    float s = 0.f;
    for (int k = 0; k < blocks; ++k) s += v[k * tokens * 2 * np];
    st(static_cast<T*>(which ? g.dc : g.db) + tok * p.N + n, s);
    return;
  }
  i -= nbc;
  const int parts = p.R * p.segments;
  if (i < na) {
    const long long c = i / p.N;
    const float* v = g.a_parts + c * np + i % p.N;
    float s = 0.f;
    for (int k = 0; k < parts; ++k) s += v[static_cast<long long>(k) * padded * np];
    g.da[i] = s;
    return;
  }
  i -= na;
  if (i < p.C && g.dd != nullptr) {
    float s = 0.f;
    for (int k = 0; k < parts; ++k) s += g.d_parts[static_cast<long long>(k) * padded + i];
    g.dd[i] = s;
  }
}

template <typename T, int LN>
int grad_go(const Grad& g, cudaStream_t stream) {
  using L = Lay<LN, 4>;
  const Args& p = g.f;
  const long long blocks = (p.C + L::CB - 1) / L::CB;
  const long long sums = (static_cast<long long>(p.R) * p.T * 2 * p.N + static_cast<long long>(p.C) * (p.N + 1) + 255) / 256;
  if (blocks * p.segments * p.R > 0x7fffffffLL || sums > 0x7fffffffLL) return -3;
  constexpr int smem = static_cast<int>(sizeof(Shared<LN>));
  cudaError_t e = cudaFuncSetAttribute(grad_kernel<T, LN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (p.segments > 1) back_ends_kernel<T, LN><<<static_cast<unsigned>(blocks * (p.segments - 1) * p.R), THREADS, 0, stream>>>(g);
  grad_kernel<T, LN><<<static_cast<unsigned>(blocks * p.segments * p.R), THREADS, smem, stream>>>(g);
  grad_sum_kernel<T><<<static_cast<unsigned>(sums), 256, 0, stream>>>(g, static_cast<int>(blocks), static_cast<int>(blocks) * L::CB, L::NP);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int grad_any(const Grad& g, cudaStream_t stream) {
  if (g.f.N <= 16) return grad_go<T, 4>(g, stream);
  if (g.f.N <= 32) return grad_go<T, 8>(g, stream);
  if (g.f.N <= 64) return grad_go<T, 16>(g, stream);
  if (g.f.N <= 128) return grad_go<T, 32>(g, stream);
  return -3;
}

}  // namespace selective
}  // namespace dewb

using namespace dewb::selective;

extern "C" int dewb_selective_grad(const dewb_selective_grad_args* a, int fp32, void* stream_ptr) {
  if (a == nullptr) return -3;
  const Args& p = a->f;
  if (p.R < 1 || p.T < 1 || p.C < 1 || p.N < 1 || p.heads > 0 || p.groups != 1 || p.positions != nullptr || p.checkpoints == nullptr || p.segments < 1 || p.segment < 1 || p.segment % EVERY)
    return -3;
  // every segment has a token, and every token a segment
  if (static_cast<long long>(p.segments) * p.segment < p.T || static_cast<long long>(p.segments - 1) * p.segment >= p.T) return -3;
  if (p.segments > 1 && (p.starts == nullptr || p.sums == nullptr)) return -3;
  if (a->dy == nullptr || a->dx == nullptr || a->ddt == nullptr || a->db == nullptr || a->dc == nullptr || a->da == nullptr || a->bc_parts == nullptr || a->a_parts == nullptr || a->d_parts == nullptr)
    return -3;
  if ((p.z != nullptr) != (a->dz != nullptr)) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  return fp32 ? grad_any<float>(*a, stream) : grad_any<bf16>(*a, stream);
}
