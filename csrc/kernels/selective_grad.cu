// Gradients of the selective state space scan, for sm_100a (the equations and the lanes' layout: selective.cuh).  With u = s x, w = dy silu(z) and a_t = exp(s_t A):
//
//   g_t = w_t C_t + a_{t+1} g_{t+1}  (from the gradient of the last state)         dC_t[n] = sum_c w h          dB_t[n] = sum_c u g
//   dx = s sum_n g B + D w       ds = x sum_n g B + sum_n A q,  q = g a h_{t-1}     dA = sum_t s q               dD = sum_t w x       dz = dy (sum_n C h + D x) silu'(z)
//
//   back_ends_kernel  with several segments: what each makes of a gradient of zeros at its end
//   grad_kernel       sixteen tokens at a time, from the last on: the states in front of every four of them, from the one that the forward kept; then four tokens forwards, with their
//                     decays and decayed states kept in registers, and the same four backwards.  Sums over channels leave a block as parts, so the result has one order whatever
//                     runs first
//   grad_sum_kernel   adds up the parts
//
// All in fp32; inputs and gradients are bf16 or fp32 (template T; the steps' logits either).  Compiled without fast math.
//
// 4 rows of 2048 tokens of 4096 channels of 16 states: 826 us in eight segments, their ends 182, the parts' sums 15; bytes 83 us, exponentials (1.75 a state) 280.  A token of a warp's 32
// channels takes 366 instructions (320 cycles of the multiply-add pipe, 290 of the special-function unit, 100 wavefronts of shared memory) in 830 cycles: two blocks of four warps an
// SM (255 registers, 108 KB), each waiting 1.3 of 4.2 cycles for the instruction before.  Kept for it: decays and decayed states of four tokens in registers (all eight states in front of
// a token in shared memory and the exponentials anew: 929); sums over lanes through shared memory, where a lane leaves its shares and the lanes that form the gradients add them up
// (shuffles: 1000 and more); two states a lane, which leave room for 12 warps, only where there are few channels (large calls: 938).
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
  float *bc_parts, *a_parts, *d_parts; // [channel blocks, R * T, 2, padded N], [R * segments, padded, padded N], [R * segments, padded]
};
static_assert(sizeof(dewb_selective_grad_args) == 280 + 120, "packed by ops/selective.py");

namespace dewb {
namespace selective {

using Grad = dewb_selective_grad_args;
constexpr int TT = Lay<4, 4>::TT;
constexpr int FOUR = 4;                // tokens whose decays and states a lane has in registers

template <int LN, int NS>
struct Shared {
  using L = Lay<LN, NS>;
  float step[WARPS][TT][L::CW], w[WARPS][TT][L::CW];      // s, w
  float2 c[TT][L::NP];                                    // C, each number twice; up to here, what back_ends_kernel has
  float in[WARPS][TT][L::CW];                             // u
  float2 b[TT][L::NP];
  float bc[WARPS][TT][2][L::NP];                          // dB and dC of the warp's channels
  float4 h[WARPS][TT / FOUR][NS][32];                     // a lane's states in front of every four tokens, in pairs of channels as they are
  float4 shares[WARPS][FOUR][3][32];                      // a lane's shares of sum g B, sum A q and sum C h, four channels each
  float4 both[WARPS][FOUR][NS / 2][32];                   // ... and of dB and dC, NS states each
};

// Where a lane loads and stores: four channels of token lt + pass * LN; and what it has of a tile's tokens.
template <typename T, typename TD, int LN, int NS, bool STATES>
struct Place {
  using L = Lay<LN, NS>;
  int lt, lq, lc, left;
  bool whole;                          // ... all over the block, in pieces of four
  const T *x, *z, *dy;
  const TD* dt;
  Raw<T> rx[L::PASSES], rz[L::PASSES], ry[L::PASSES];
  Raw<TD> rd[L::PASSES];
  __device__ __forceinline__ Place(const Grad& g, int row, int c_block, int c0, int lane) {
    const Args& p = g.f;
    lt = lane / L::CG;
    lq = lane % L::CG * 4;
    lc = c0 + lq;
    left = max(0, min(4, p.C - lc));
    x = static_cast<const T*>(p.x) + row * p.x_row + lc;
    z = p.z == nullptr ? nullptr : static_cast<const T*>(p.z) + row * p.z_row + lc;
    dy = static_cast<const T*>(g.dy) + row * g.dy_row + lc;
    dt = static_cast<const TD*>(p.dt) + row * p.dt_row + lc;
    whole = c_block + L::CB <= p.C && (p.C & 3) == 0 && fours<T>(p.x, p.x_row, p.x_token) && fours<TD>(p.dt, p.dt_row, p.dt_token) && fours<T>(g.dy, g.dy_row, g.dy_token) &&
            (z == nullptr || fours<T>(p.z, p.z_row, p.z_token));
  }
  // ahead of their turn, as far as L2
  __device__ __forceinline__ void call(const Grad& g, int t0, int t_end) const {
#pragma unroll
    for (int i = 0; i < L::PASSES; ++i) {
      const int t = t0 + lt + i * LN;
      if (lt < TT && t < t_end && left > 0 && t >= 0) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(x + t * g.f.x_token));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(dt + t * g.f.dt_token));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(dy + t * g.dy_token));
        if (z != nullptr) asm volatile("prefetch.global.L2 [%0];" ::"l"(z + t * g.f.z_token));
      }
    }
  }
  template <bool FAST>
  __device__ __forceinline__ void bring(const Grad& g, int i, int t0, int t_end) {
    const int t = t0 + lt + i * LN, n = lt < TT && t < t_end ? left : 0;
    if (!FAST || LN <= TT || lt < TT) {
      if (STATES) rx[i] = fetch(x + t * g.f.x_token, FAST, n);
      rd[i] = fetch(dt + t * g.f.dt_token, FAST, n);
      ry[i] = fetch(dy + t * g.dy_token, FAST, n);
      if (z != nullptr) rz[i] = fetch(z + t * g.f.z_token, FAST, n);
    }
  }
  __device__ __forceinline__ void bring(const Grad& g, int t0, int t_end) {
    if (whole && t0 + TT <= t_end) {
#pragma unroll
      for (int i = 0; i < L::PASSES; ++i) bring<true>(g, i, t0, t_end);
    } else {
#pragma unroll
      for (int i = 0; i < L::PASSES; ++i) bring<false>(g, i, t0, t_end);
    }
  }
};

// What a block has of a tile's B and C, four states of a token a piece.
template <typename T, int LN, int NS, bool STATES>
struct Narrow {
  using L = Lay<LN, NS>;
  static constexpr int ALL = TT * L::NP / 4, EACH = (ALL + THREADS - 1) / THREADS;
  Raw<T> b[STATES ? EACH : 1], c[EACH];
  const T *pb, *pc;
  bool b_whole, c_whole;
  __device__ __forceinline__ Narrow(const Args& p, int row) {
    pb = static_cast<const T*>(p.b) + row * p.b_row;
    pc = static_cast<const T*>(p.c) + row * p.c_row;
    b_whole = fours<T>(pb, p.b_row, p.b_token);
    c_whole = fours<T>(pc, p.c_row, p.c_token);
  }
  __device__ __forceinline__ void bring(const Args& p, int i, int t0, int t_end) {
    const int at = threadIdx.x + i * THREADS, t = t0 + at / (L::NP / 4), n = at % (L::NP / 4) * 4;
    const int there = at < ALL && t < t_end ? max(0, min(4, p.N - n)) : 0;
    if (STATES) b[i] = fetch(pb + t * p.b_token + n, b_whole && there == 4, there);
    c[i] = fetch(pc + t * p.c_token + n, c_whole && there == 4, there);
  }
  __device__ __forceinline__ void put(Shared<LN, NS>& sm, int i) const {
    const int at = threadIdx.x + i * THREADS, t = at / (L::NP / 4), n = at % (L::NP / 4) * 4;
    if (ALL % THREADS == 0 || at < ALL) {
      if (STATES) twice(&sm.b[t][n], b[i]);
      twice(&sm.c[t][n], c[i]);
    }
  }
  __device__ __forceinline__ void bring(const Args& p, int t0, int t_end) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) bring(p, i, t0, t_end);
  }
  __device__ __forceinline__ void put(Shared<LN, NS>& sm) const {
#pragma unroll
    for (int i = 0; i < EACH; ++i) put(sm, i);
  }
};

// s, u and w of the warp's channels from what the lanes have brought, pass i; behind t_end and the last channel, zeros.
template <typename T, typename TD, int LN, int NS, bool STATES>
__device__ __forceinline__ void stage(Shared<LN, NS>& sm, const Place<T, TD, LN, NS, STATES>& at, bool steps, int i, int t0, int t_end, int warp, float (&total)[4]) {
  const bool all = t0 + TT <= t_end && at.left == 4;
  const int t = at.lt + i * LN;
  if (LN > TT && t >= TT) return;
  float x[4], s[4], w[4], z[4];
  if (STATES) at.rx[i].get(x);
  at.rd[i].get(s);
  at.ry[i].get(w);
  if (at.z != nullptr) at.rz[i].get(z);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (steps) s[j] = softplus(s[j]);
    if (at.z != nullptr) w[j] *= z[j] * gate<T>(z[j]);
    if (!all && (j >= at.left || t0 + t >= t_end)) s[j] = w[j] = 0.f;
    if (STATES) x[j] = !all && (j >= at.left || t0 + t >= t_end) ? 0.f : s[j] * x[j];
    total[j] += s[j];
  }
  *reinterpret_cast<float4*>(&sm.step[warp][t][at.lq]) = make_float4(s[0], s[1], s[2], s[3]);
  *reinterpret_cast<float4*>(&sm.w[warp][t][at.lq]) = make_float4(w[0], w[1], w[2], w[3]);
  if (STATES) *reinterpret_cast<float4*>(&sm.in[warp][t][at.lq]) = make_float4(x[0], x[1], x[2], x[3]);
}

// Numbers of four channels and NS states, channels in pairs.
template <int NS>
struct Block {
  f2 v[2][NS];
  template <typename F>
  __device__ __forceinline__ static Block make(F f) {
    Block r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NS; ++k) r.v[i][k] = f2(f(2 * i, k), f(2 * i + 1, k));
    return r;
  }
  // `channels` of them (0 to 4), zeros in place of the others
  __device__ __forceinline__ static Block load(const float* p, int stride, int channels = 4) {
    float2 e[4][NS / 2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < NS / 2; ++k) e[j][k] = j < channels ? *reinterpret_cast<const float2*>(p + j * stride + 2 * k) : make_float2(0.f, 0.f);
    Block r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NS / 2; ++k) {
        r.v[i][2 * k] = f2(e[2 * i][k].x, e[2 * i + 1][k].x);
        r.v[i][2 * k + 1] = f2(e[2 * i][k].y, e[2 * i + 1][k].y);
      }
    return r;
  }
  __device__ __forceinline__ void store(float* p, int stride) const {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NS; k += 2) {
        const float2 e0 = v[i][k].get(), e1 = v[i][k + 1].get();
        *reinterpret_cast<float2*>(p + 2 * i * stride + k) = make_float2(e0.x, e1.x);
        *reinterpret_cast<float2*>(p + (2 * i + 1) * stride + k) = make_float2(e0.y, e1.y);
      }
  }
};

template <int NS>
__device__ __forceinline__ Block<NS> last_of(const Grad& g, int row, int c, int n, bool there) {
  const Args& p = g.f;
  return Block<NS>::make([&](int j, int k) { return there && g.dlast != nullptr && c + j < p.C && n + k < p.N ? g.dlast[(static_cast<long long>(row) * p.C + c + j) * p.N + n + k] : 0.f; });
}

// grid R * (segments - 1) * channel blocks, of segments 1, 2, ...: starts[r, j] is the gradient of the state in front of segment j that the segment itself makes (the last one: with dlast).
template <typename T, typename TD, int LN, int NS>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 2 : 4)
back_ends_kernel(const Grad g) {
  using L = Lay<LN, NS>;
  using S = Shared<LN, NS>;
  __shared__ __align__(16) char raw[offsetof(S, in)];
  S& sm = *reinterpret_cast<S*>(raw);
  const Args& p = g.f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sl = lane % LN, cg = lane / LN;
  const int blocks = (p.C + L::CB - 1) / L::CB, padded = p.padded;
  const int cb = blockIdx.x % blocks, seg = 1 + blockIdx.x / blocks % (p.segments - 1), row = blockIdx.x / blocks / (p.segments - 1);
  const int c0 = cb * L::CB + warp * L::CW, t_begin = seg * p.segment, t_end = min(p.T, t_begin + p.segment);
  Place<T, TD, LN, NS, false> at(g, row, cb * L::CB, c0, lane);
  Narrow<T, LN, NS, false> narrow(p, row);
  float total[4] = {0.f, 0.f, 0.f, 0.f};
  const Block<NS> a = Block<NS>::make([&](int j, int k) { return rate<false>(p, c0 + cg * 4 + j, sl * NS + k, 1); });
  Block<NS> d = last_of<NS>(g, row, c0 + cg * 4, sl * NS, seg == p.segments - 1);
  int t0 = t_begin + (t_end - t_begin - 1) / TT * TT;
  at.bring(g, t0, t_end);
  narrow.bring(p, t0, t_end);
  for (; t0 >= t_begin; t0 -= TT) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < L::PASSES; ++i) stage<T, TD, LN, NS, false>(sm, at, p.softplus, i, t0, t_end, warp, total);
    narrow.put(sm);
    __syncthreads();
    if (t0 > t_begin) {
      at.bring(g, t0 - TT, t_end);
      narrow.bring(p, t0 - TT, t_end);
    }
    const int count = min(TT, t_end - t0);
#pragma unroll 4
    for (int t = (count + 3) / 4 * 4 - 1; t >= 0; --t) {
      f2 s[2], w[2], c[NS];
      pair(&sm.step[warp][t][cg * 4], s[0], s[1]);
      pair(&sm.w[warp][t][cg * 4], w[0], w[1]);
      pairs(&sm.c[t][sl * NS], c);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < NS; ++k) d.v[i][k] = mul(ex2(mul(s[i], a.v[i][k])), fma(w[i], c[k], d.v[i][k]));
    }
  }
  const long long out = (static_cast<long long>(row) * p.segments + seg) * padded + c0;
  d.store(p.starts + (out + cg * 4) * L::NP + sl * NS, L::NP);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int o = L::CG; o < 32; o <<= 1) total[j] += __shfl_xor_sync(0xffffffffu, total[j], o);
    if (at.lt == 0) p.sums[out + at.lq + j] = total[j];
  }
}

template <typename T, typename TD, int LN, int NS>
__global__ void __launch_bounds__(THREADS, NS == 2 ? 3 : 2)
grad_kernel(const Grad g) {
  using L = Lay<LN, NS>;
  constexpr int CG = L::CG, NP = L::NP;
  extern __shared__ __align__(16) char raw[];
  Shared<LN, NS>& sm = *reinterpret_cast<Shared<LN, NS>*>(raw);
  const Args& p = g.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sl = lane % LN, cg = lane / LN;
  const int blocks = (p.C + L::CB - 1) / L::CB, padded = p.padded;
  const int cb = blockIdx.x % blocks, seg = blockIdx.x / blocks % p.segments, row = blockIdx.x / blocks / p.segments;
  const int c0 = cb * L::CB + warp * L::CW, t_begin = seg * p.segment, t_end = min(p.T, t_begin + p.segment);
  Place<T, TD, LN, NS, true> at(g, row, cb * L::CB, c0, lane);
  int t0 = t_begin + (t_end - t_begin - 1) / TT * TT;
  const long long pad_row = static_cast<long long>(row) * p.segments * padded + c0 + cg * 4;
  const Block<NS> a = Block<NS>::make([&](int j, int k) { return rate<false>(p, c0 + cg * 4 + j, sl * NS + k, 1); });
  Block<NS> d = last_of<NS>(g, row, c0 + cg * 4, sl * NS, seg == p.segments - 1), da = Block<NS>::make([](int, int) { return 0.f; });
#pragma unroll 2
  for (int q = p.segments - 1; q > seg; --q) {    // what comes from behind the segment
    const long long there = pad_row + static_cast<long long>(q) * padded;
    const Block<NS> e = Block<NS>::load(p.starts + there * NP + sl * NS, NP);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f2 sum = q < p.segments - 1 ? f2(p.sums[there + 2 * i], p.sums[there + 2 * i + 1]) : f2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < NS; ++k) d.v[i][k] = fma(ex2(mul(sum, a.v[i][k])), d.v[i][k], e.v[i][k]);
    }
  }
  float skip[4], dd[4] = {0.f, 0.f, 0.f, 0.f}, unused[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) skip[j] = p.d != nullptr && j < at.left ? p.d[at.lc + j] : 0.f;
  const int kept = (p.T + EVERY - 1) / EVERY;
  const long long here = static_cast<long long>(row) * p.T * p.C + at.lc;
  const bool y_whole = at.left == 4 && (p.C & 3) == 0;
  auto piece = [&](const float4* q, f2& x, f2& y) { pair(&q->x, x, y); };
  auto leave = [](float4* q, f2 x, f2 y) { *reinterpret_cast<ulonglong2*>(q) = make_ulonglong2(x.v, y.v); };
  for (; t0 >= t_begin; t0 -= TT) {
    if (t0 > t_begin) at.call(g, t0 - TT, t_end);
    Narrow<T, LN, NS, true> narrow(p, row);
    if constexpr (sizeof(T) == 2) {               // all loads of the tile on their way together
      at.bring(g, t0, t_end);
      narrow.bring(p, t0, t_end);
#pragma unroll
      for (int i = 0; i < L::PASSES; ++i) stage<T, TD, LN, NS, true>(sm, at, p.softplus, i, t0, t_end, warp, unused);
      narrow.put(sm);
    } else {                                      // one after another: fp32 takes twice the registers
#pragma unroll
      for (int i = 0; i < L::PASSES; ++i) {
        if (at.whole && t0 + TT <= t_end) at.template bring<true>(g, i, t0, t_end);
        else at.template bring<false>(g, i, t0, t_end);
        stage<T, TD, LN, NS, true>(sm, at, p.softplus, i, t0, t_end, warp, unused);
        asm volatile("" ::: "memory");
      }
#pragma unroll
      for (int i = 0; i < narrow.EACH; ++i) {
        narrow.bring(p, i, t0, t_end);
        narrow.put(sm, i);
        asm volatile("" ::: "memory");
      }
    }
    // (channels behind the last one have no kept states: the forward's blocks may be narrower)
    const float* before = p.checkpoints + ((static_cast<long long>(row) * kept + t0 / EVERY) * padded + c0 + cg * 4) * NP + sl * NS;
    Block<NS> h = Block<NS>::load(before, NP, p.C - c0 - cg * 4);
    if (t0 > t_begin && c0 + cg * 4 < p.C) asm volatile("prefetch.global.L2 [%0];" ::"l"(before - static_cast<long long>(padded) * NP));
    __syncthreads();
    const int count = min(TT, t_end - t0), groups = (count + FOUR - 1) / FOUR;
    // (behind the last token steps, u and w are zero: decays of one, and nothing added to any sum)
#pragma unroll 1
    for (int q = 0; q < groups; ++q) {
#pragma unroll
      for (int i = 0; i < NS; ++i) leave(&sm.h[warp][q][i][lane], h.v[i / (NS / 2)][i % (NS / 2) * 2], h.v[i / (NS / 2)][i % (NS / 2) * 2 + 1]);
      if (q + 1 < groups) {
#pragma unroll
        for (int i = 0; i < FOUR; ++i) {
          const int t = q * FOUR + i;
          f2 s[2], u[2], b[NS];
          pair(&sm.step[warp][t][cg * 4], s[0], s[1]);
          pair(&sm.in[warp][t][cg * 4], u[0], u[1]);
          pairs(&sm.b[t][sl * NS], b);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < NS; ++k) h.v[j][k] = fma(ex2(mul(s[j], a.v[j][k])), h.v[j][k], mul(u[j], b[k]));
        }
      }
    }
#pragma unroll 1
    for (int q = groups - 1; q >= 0; --q) {
      const int from = q * FOUR, mine = from + at.lt;
      const long long tok = t0 + mine;
      const bool ends = at.lt < FOUR && mine < count;          // this lane forms gradients of four channels of a token
      const int n = ends ? at.left : 0;
      const bool fast = at.whole && ends;
      const Raw<T> rx = fetch(at.x + tok * p.x_token, fast, n), ry = fetch(at.dy + tok * g.dy_token, fast, n);
      const Raw<TD> rd = fetch(at.dt + tok * p.dt_token, fast, n);
      Raw<T> rz;
      if (at.z != nullptr) rz = fetch(at.z + tok * p.z_token, fast, n);
#pragma unroll
      for (int i = 0; i < NS; ++i) piece(&sm.h[warp][q][i][lane], h.v[i / (NS / 2)][i % (NS / 2) * 2], h.v[i / (NS / 2)][i % (NS / 2) * 2 + 1]);
      Block<NS> e[FOUR], ah[FOUR];
#pragma unroll
      for (int i = 0; i < FOUR; ++i) {
        const int t = from + i;
        f2 s[2], u[2], b[NS];
        pair(&sm.step[warp][t][cg * 4], s[0], s[1]);
        pair(&sm.in[warp][t][cg * 4], u[0], u[1]);
        pairs(&sm.b[t][sl * NS], b);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < NS; ++k) {
            e[i].v[j][k] = ex2(mul(s[j], a.v[j][k]));
            ah[i].v[j][k] = mul(e[i].v[j][k], h.v[j][k]);
            if (i + 1 < FOUR) h.v[j][k] = fma(u[j], b[k], ah[i].v[j][k]);
          }
      }
#pragma unroll
      for (int i = FOUR - 1; i >= 0; --i) {
        const int t = from + i;
        f2 s[2], u[2], w[2], b[NS], c[NS], db[NS], dc[NS], s1[2], s2[2], s3[2];
        pair(&sm.step[warp][t][cg * 4], s[0], s[1]);
        pair(&sm.in[warp][t][cg * 4], u[0], u[1]);
        pair(&sm.w[warp][t][cg * 4], w[0], w[1]);
        pairs(&sm.b[t][sl * NS], b);
        pairs(&sm.c[t][sl * NS], c);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < NS; ++k) {
            const f2 now = fma(u[j], b[k], ah[i].v[j][k]), gt = fma(w[j], c[k], d.v[j][k]), through = mul(gt, ah[i].v[j][k]);
            db[k] = j == 0 ? mul(u[j], gt) : fma(u[j], gt, db[k]);
            dc[k] = j == 0 ? mul(w[j], now) : fma(w[j], now, dc[k]);
            s1[j] = k == 0 ? mul(gt, b[k]) : fma(gt, b[k], s1[j]);
            s2[j] = k == 0 ? mul(through, a.v[j][k]) : fma(through, a.v[j][k], s2[j]);
            s3[j] = k == 0 ? mul(now, c[k]) : fma(now, c[k], s3[j]);
            da.v[j][k] = fma(through, s[j], da.v[j][k]);
            d.v[j][k] = mul(gt, e[i].v[j][k]);
          }
        float v[2 * NS];
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          const float2 x = db[k].get(), y = dc[k].get();
          v[k] = x.x + x.y;
          v[NS + k] = y.x + y.y;
        }
        leave(&sm.shares[warp][i][0][lane], s1[0], s1[1]);
        leave(&sm.shares[warp][i][1][lane], s2[0], s2[1]);
        leave(&sm.shares[warp][i][2][lane], s3[0], s3[1]);
#pragma unroll
        for (int k = 0; k < NS / 2; ++k) sm.both[warp][i][k][lane] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
      }
      __syncwarp();
      // dB and dC of the warp's channels: a lane takes four of a token's numbers
#pragma unroll
      for (int o = lane; o < FOUR * NS / 2 * LN; o += 32) {
        const int state = o % LN, k = o / LN % (NS / 2), i = o / LN / (NS / 2);
        const float4 v = sum4(&sm.both[warp][i][k][state], CG, LN, k);
        if constexpr (NS == 4) {
          *reinterpret_cast<float4*>(&sm.bc[warp][from + i][k][state * 4]) = v;
        } else {
          *reinterpret_cast<float2*>(&sm.bc[warp][from + i][0][state * 2]) = make_float2(v.x, v.y);
          *reinterpret_cast<float2*>(&sm.bc[warp][from + i][1][state * 2]) = make_float2(v.z, v.w);
        }
      }
      if (ends) {
        const int turn = turn_of<LN>(lane), first = lane % CG * LN;
        const float4 v1 = sum4(&sm.shares[warp][at.lt][0][first], LN, 1, turn), v2 = sum4(&sm.shares[warp][at.lt][1][first], LN, 1, turn);
        const float4 s4 = *reinterpret_cast<const float4*>(&sm.step[warp][mine][at.lq]), w4 = *reinterpret_cast<const float4*>(&sm.w[warp][mine][at.lq]);
        const float r1[4] = {v1.x, v1.y, v1.z, v1.w}, r2[4] = {v2.x, v2.y, v2.z, v2.w}, s[4] = {s4.x, s4.y, s4.z, s4.w}, w[4] = {w4.x, w4.y, w4.z, w4.w};
        float x[4], raw_step[4], dx[4], ds[4];
        rx.get(x);
        rd.get(raw_step);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          dx[j] = fmaf(s[j], r1[j], skip[j] * w[j]);
          ds[j] = fmaf(x[j], r1[j], LN2 * r2[j]);
          if (p.softplus) ds[j] *= gate<TD>(raw_step[j]);
          dd[j] = fmaf(w[j], x[j], dd[j]);
        }
        put(static_cast<T*>(g.dx) + here + tok * p.C, dx, y_whole, at.left);
        put(static_cast<TD*>(g.ddt) + here + tok * p.C, ds, y_whole, at.left);
        if (at.z != nullptr) {
          const float4 v3 = sum4(&sm.shares[warp][at.lt][2][first], LN, 1, turn);
          const float r3[4] = {v3.x, v3.y, v3.z, v3.w};
          float dy[4], z[4];
          ry.get(dy);
          rz.get(z);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float sig = gate<T>(z[j]);
            z[j] = dy[j] * fmaf(skip[j], x[j], r3[j]) * sig * fmaf(z[j], 1.f - sig, 1.f);
          }
          put(static_cast<T*>(g.dz) + here + tok * p.C, z, y_whole, at.left);
        }
      }
      __syncwarp();                               // (the shares have been read)
    }
    __syncthreads();
    for (int o = tid; o < count * NP / 2; o += THREADS)
      *reinterpret_cast<float4*>(g.bc_parts + ((static_cast<long long>(cb) * p.R + row) * p.T + t0) * (2 * NP) + o * 4) =
          sum4(reinterpret_cast<const float4*>(&sm.bc[0][0][0][0]) + o, WARPS, TT * NP / 2, 0);
  }
  const long long part = (static_cast<long long>(row) * p.segments + seg) * padded + c0;
  da.store(g.a_parts + (part + cg * 4) * NP + sl * NS, NP);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int o = CG; o < 32; o <<= 1) dd[j] += __shfl_xor_sync(0xffffffffu, dd[j], o);
    if (at.lt == 0) g.d_parts[part + at.lq + j] = dd[j];
  }
  if (seg == 0 && g.dinitial != nullptr) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const int c = c0 + cg * 4 + 2 * i, n = sl * NS + k;
        const float2 v = d.v[i][k].get();
        if (c < p.C && n < p.N) g.dinitial[(static_cast<long long>(row) * p.C + c) * p.N + n] = v.x;
        if (c + 1 < p.C && n < p.N) g.dinitial[(static_cast<long long>(row) * p.C + c + 1) * p.N + n] = v.y;
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
#pragma unroll 8
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
#pragma unroll 8
    for (int k = 0; k < parts; ++k) s += v[static_cast<long long>(k) * padded * np];
    g.da[i] = s;
    return;
  }
  i -= na;
  if (i < p.C && g.dd != nullptr) {
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < parts; ++k) s += g.d_parts[static_cast<long long>(k) * padded + i];
    g.dd[i] = s;
  }
}

template <typename T, typename TD, int LN, int NS = 4>
int grad_go(const Grad& g, cudaStream_t stream) {
  using L = Lay<LN, NS>;
  const Args& p = g.f;
  const long long blocks = (p.C + L::CB - 1) / L::CB;
  const long long sums = (static_cast<long long>(p.R) * p.T * 2 * p.N + static_cast<long long>(p.C) * (p.N + 1) + 255) / 256;
  if (blocks * p.segments * p.R > 0x7fffffffLL || sums > 0x7fffffffLL) return -3;
  constexpr int smem = static_cast<int>(sizeof(Shared<LN, NS>));
  cudaError_t e = cudaFuncSetAttribute(grad_kernel<T, TD, LN, NS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (p.segments > 1) back_ends_kernel<T, TD, LN, NS><<<static_cast<unsigned>(blocks * (p.segments - 1) * p.R), THREADS, 0, stream>>>(g);
  grad_kernel<T, TD, LN, NS><<<static_cast<unsigned>(blocks * p.segments * p.R), THREADS, smem, stream>>>(g);
  grad_sum_kernel<T><<<static_cast<unsigned>(sums), 256, 0, stream>>>(g, static_cast<int>(blocks), p.padded, L::NP);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, typename TD>
int grad_any(const Grad& g, cudaStream_t stream) {
  if (g.f.N <= 16) {
    if (g.f.states_each == 2) return grad_go<T, TD, 8, 2>(g, stream);
    if constexpr (sizeof(T) == 2) return grad_go<T, TD, 4>(g, stream);
    return -3;                                    // (four states a lane: more registers than there are)
  }
  if (g.f.N <= 32) return grad_go<T, TD, 8>(g, stream);
  if (g.f.N <= 64) return grad_go<T, TD, 16>(g, stream);
  if (g.f.N <= 128) return grad_go<T, TD, 32>(g, stream);
  return -3;
}

}  // namespace selective
}  // namespace dewb

using namespace dewb::selective;

extern "C" int dewb_selective_grad(const dewb_selective_grad_args* a, int fp32, void* stream_ptr) {
  if (a == nullptr) return -3;
  const Args& p = a->f;
  if (p.R < 1 || p.T < 1 || p.C < 1 || p.N < 1 || p.heads > 0 || p.groups != 1 || p.positions != nullptr || p.checkpoints == nullptr || p.segments < 1 || p.segment < 1 || p.segment % EVERY ||
      p.padded % 128 || p.padded < p.C)
    return -3;
  // every segment has a token, and every token a segment
  if (static_cast<long long>(p.segments) * p.segment < p.T || static_cast<long long>(p.segments - 1) * p.segment >= p.T) return -3;
  if (p.segments > 1 && (p.starts == nullptr || p.sums == nullptr)) return -3;
  if (a->dy == nullptr || a->dx == nullptr || a->ddt == nullptr || a->db == nullptr || a->dc == nullptr || a->da == nullptr || a->bc_parts == nullptr || a->a_parts == nullptr || a->d_parts == nullptr)
    return -3;
  if ((p.z != nullptr) != (a->dz != nullptr)) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (fp32) return p.dt_fp32 ? grad_any<float, float>(*a, stream) : -3;
  return p.dt_fp32 ? grad_any<bf16, float>(*a, stream) : grad_any<bf16, bf16>(*a, stream);
}
