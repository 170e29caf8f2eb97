// The selective state space scan forward, for sm_100a (the equations and the lanes' layout: selective.cuh), over whole rows or over a call's rows with the states that a store keeps.
//
//   scan_kernel       tokens one after another with the states in registers, in fp32.  The row may be cut into segments that run side by side; the first launch (ENDS) then
//                     forms what each segment makes of a state of zeros and the sum of its steps, and the second one composes what stands in front of a segment from those
//   token_kernel      one token per row, a rate per channel and state: the state is read and written once
//   head_token_kernel one token per row, a decay per head
//
// A call row whose first position is 0 starts from zero; positions below 0 are padding at a row's end: they change no state and give zeros.
// Inputs and outputs are bf16 or fp32 (template T; the steps' logits either), everything else fp32.  Compiled without fast math.
#include "../common/selective.cuh"

namespace dewb {
namespace selective {

template <int LN, int NS, bool ENDS>
struct Tile {
  using L = Lay<LN, NS>;
  float step[WARPS][L::TT][L::CW], in[WARPS][L::TT][L::CW];                  // s (heads: the decay), s x
  float2 b[L::TT][L::NP], c[ENDS ? 1 : L::TT][L::NP];                        // each number twice: beside two channels
  float4 out[ENDS ? 1 : WARPS][ENDS ? 1 : L::TT][32];                        // a lane's share of sum C h, four channels
};

// grid R * segments * channel blocks.  With heads, a channel block lies within one group (that shares B and C).
//   starts[r, 0]       the state that row r begins with          starts[r, j]   what segment j - 1 ends with: from there on for j = 1, from zeros for the others
//   sums[r, j]         the sum of segment j's steps, per channel
// A tile's x and steps come a tile ahead, in registers; what the end of a tile needs (x again, z) is asked for at its beginning (L2) and read then.  The sums over states are formed at
// the end of a tile from what every lane leaves in shared memory: with shuffles after every token (or two, or four) a warp alone took 620 cycles a token, so: DEWB_ALONE.
template <typename T, typename TD, int LN, int NS, bool HEADS, bool ENDS>
__global__ void __launch_bounds__(THREADS, NS > 4 ? 2 : 4)
scan_kernel(const Args p) {
  using L = Lay<LN, NS>;
  constexpr int CG = L::CG, CW = L::CW, CB = L::CB, NP = L::NP, TT = L::TT, PASSES = L::PASSES, BC = (TT * NP + THREADS - 1) / THREADS;
  extern __shared__ __align__(16) char raw[];
  Tile<LN, NS, ENDS>& sm = *reinterpret_cast<Tile<LN, NS, ENDS>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sl = lane % LN, cg = lane / LN;
  const int per = p.C / p.groups, blocks = (per + CB - 1) / CB * p.groups, padded = blocks * CB;
  const int segments = ENDS ? p.segments - 1 : p.segments;
  const int cb = blockIdx.x % blocks, seg = blockIdx.x / blocks % segments, row = blockIdx.x / blocks / segments;
  const int group = cb / (blocks / p.groups), c_end = (group + 1) * per;                      // channels of this block's group end there
  const int c_block = group * per + cb % (blocks / p.groups) * CB, c0 = c_block + warp * CW;
  const int dim = HEADS ? p.C / p.heads : 1;
  const Row r = row_of(p, row);
  const int t_begin = seg * p.segment, t_end = min(r.len, t_begin + p.segment), t_stop = min(p.T, t_begin + p.segment);
  // where this lane loads and stores: four channels of token lane / CG + pass * LN
  const int lt = lane / CG, lq = lane % CG * 4, lc = c0 + lq, left = max(0, min(4, c_end - lc));
  T* y = static_cast<T*>(p.y) + static_cast<long long>(row) * p.T * p.C + lc;
  const bool y_whole = left == 4 && ((c_block | p.C) & 3) == 0;
  const int last_seg = r.len > 0 ? (r.len - 1) / p.segment : -1;
  if (!ENDS) {
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t = max(t_begin, t_end) + lt; t < t_stop; t += LN) put(y + static_cast<long long>(t) * p.C, none, y_whole, left);
  }
  if (seg > last_seg) return;

  f2 a[2][NS], h[2][NS];                          // of channels 2 i and 2 i + 1
  const long long pad_row = (static_cast<long long>(row) * p.segments) * padded + static_cast<long long>(cb) * CB + warp * CW + cg * 4;      // of segment 0, this lane's first channel
  auto held = [&](int c, int n) { return (ENDS || p.segments == 1) && seg == 0 && r.held && c < c_end && n < p.N ? p.initial[(r.at * p.C + c) * p.N + n] : 0.f; };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = c0 + cg * 4 + 2 * i;
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int n = sl * NS + k;
      a[i][k] = HEADS && ENDS ? f2(0.f, 0.f) : f2(rate<HEADS>(p, c < c_end ? c : p.C, n, dim), rate<HEADS>(p, c + 1 < c_end ? c + 1 : p.C, n, dim));
      h[i][k] = f2(held(c, n), held(c + 1, n));
    }
  }
  // the states of this lane's channels at `to`, rows of NP
  auto keep = [&](float* to) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NS; k += 4) {
        const float2 e0 = h[i][k].get(), e1 = h[i][k + 1].get(), e2 = h[i][k + 2].get(), e3 = h[i][k + 3].get();
        *reinterpret_cast<float4*>(to + 2 * i * NP + k) = make_float4(e0.x, e1.x, e2.x, e3.x);
        *reinterpret_cast<float4*>(to + (2 * i + 1) * NP + k) = make_float4(e0.y, e1.y, e2.y, e3.y);
      }
  };
  if (ENDS && seg == 0) keep(p.starts + pad_row * NP + sl * NS);
  if (!ENDS && p.segments > 1) {                  // what stands in front of the segment
    for (int q = min(seg, 1); q <= seg; ++q) {
      const long long at = pad_row + static_cast<long long>(q) * padded;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f2 sum = q > 1 ? f2(p.sums[at - padded + 2 * i], p.sums[at - padded + 2 * i + 1]) : f2(0.f, 0.f);
        const float* e = p.starts + (at + 2 * i) * NP + sl * NS;
#pragma unroll
        for (int k = 0; k < NS; ++k) h[i][k] = fma(ex2(mul(sum, a[i][k])), h[i][k], f2(e[k], e[NP + k]));
      }
    }
  }

  // what a lane needs of its four channels where it loads
  float rate_of[4], bias[4], skip[4], total[4] = {0.f, 0.f, 0.f, 0.f};
  int head[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = min(lc + j, p.C - 1);
    head[j] = HEADS ? c / dim : 0;
    rate_of[j] = HEADS ? rate<true>(p, c, 0, dim) : 0.f;
    bias[j] = HEADS && p.dt_bias != nullptr ? p.dt_bias[head[j]] : 0.f;
    skip[j] = p.d != nullptr && !ENDS ? p.d[HEADS ? head[j] : c] : 0.f;
  }
  const T* x = static_cast<const T*>(p.x) + row * p.x_row + lc;
  const TD* dt = static_cast<const TD*>(p.dt) + row * p.dt_row + (HEADS ? 0 : lc);
  const T* z = p.z == nullptr || ENDS ? nullptr : static_cast<const T*>(p.z) + row * p.z_row + lc;
  const T* b = static_cast<const T*>(p.b) + row * p.b_row + group * p.N;
  const T* cc = static_cast<const T*>(p.c) + row * p.c_row + group * p.N;
  // whole pieces of four wherever the block loads and stores
  const bool whole = c_block + CB <= c_end && ((c_block | p.C) & 3) == 0 && fours<T>(p.x, p.x_row, p.x_token) && (z == nullptr || fours<T>(p.z, p.z_row, p.z_token)) &&
                     (HEADS || fours<TD>(p.dt, p.dt_row, p.dt_token));

  Raw<T> rx[PASSES];
  Raw<TD> rd[PASSES];
  uint32_t rh[HEADS ? PASSES : 1][4], rb[BC], rc[ENDS ? 1 : BC];
  auto bring = [&](int t0, auto fast) {
    constexpr bool FAST = decltype(fast)::value;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int t = t0 + lt + i * LN;
      const bool on = FAST ? LN <= TT || lt < TT : lt < TT && t < t_end;
      const int n = on ? left : 0;
      if (FAST) { if (on) rx[i] = fetch(x + t * p.x_token, true, 4); }
      else rx[i] = fetch(x + t * p.x_token, false, n);
      if (HEADS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) rh[i][j] = j < n ? word(dt + t * p.dt_token + head[j]) : 0u;
      } else {
        if (FAST) { if (on) rd[i] = fetch(dt + t * p.dt_token, true, 4); }
        else rd[i] = fetch(dt + t * p.dt_token, false, n);
      }
      if (z != nullptr && n > 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(z + t * p.z_token));
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) {
      const int at = tid + i * THREADS, t = t0 + at / NP, n = at % NP;
      const bool on = at < TT * NP && t < t_end && n < p.N;
      rb[i] = on ? word(b + t * p.b_token + n) : 0u;
      if (!ENDS) rc[i] = on ? word(cc + t * p.c_token + n) : 0u;
    }
  };
  auto next = [&](int t0) {
    if (whole && t0 + TT <= t_end) bring(t0, Yes());
    else bring(t0, No());
  };
  next(t_begin);
  for (int t0 = t_begin; t0 < t_end; t0 += TT) {
    __syncthreads();                              // (the tile before has been read)
    auto stage = [&](auto fast) {
      constexpr bool FAST = decltype(fast)::value;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int t = lt + i * LN;
        float xs[4], s[4];
        rx[i].get(xs);
        if (HEADS) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[j] = value<TD>(rh[i][j]);
        } else {
          rd[i].get(s);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[j] = p.softplus ? softplus(s[j] + bias[j]) : s[j] + bias[j];
          if (!FAST && (j >= left || t0 + t >= t_end)) s[j] = xs[j] = 0.f;
          if (ENDS && (LN <= TT || t < TT)) total[j] += s[j];
          xs[j] *= s[j];
          if (HEADS) s[j] = ex2(s[j] * rate_of[j]);
        }
        if (LN <= TT || t < TT) {
          *reinterpret_cast<float4*>(&sm.step[warp][t][lq]) = make_float4(s[0], s[1], s[2], s[3]);
          *reinterpret_cast<float4*>(&sm.in[warp][t][lq]) = make_float4(xs[0], xs[1], xs[2], xs[3]);
        }
      }
    };
    if (t0 + TT <= t_end && c_block + CB <= c_end) stage(Yes());
    else stage(No());
#pragma unroll
    for (int i = 0; i < BC; ++i) {
      const int at = tid + i * THREADS;
      if (TT * NP % THREADS == 0 || at < TT * NP) {
        const float bf = value<T>(rb[i]);
        sm.b[at / NP][at % NP] = make_float2(bf, bf);
        if (!ENDS) {
          const float cf = value<T>(rc[i]);
          sm.c[at / NP][at % NP] = make_float2(cf, cf);
        }
      }
    }
    __syncthreads();
    if (t0 + TT < t_end) next(t0 + TT);
    if (!ENDS && p.checkpoints != nullptr) {
      static_assert(EVERY == TT || NS > 4, "a kept state a tile");
      keep(p.checkpoints + ((static_cast<long long>(row) * ((p.T + EVERY - 1) / EVERY) + t0 / EVERY) * padded + static_cast<long long>(cb) * CB + warp * CW + cg * 4) * NP + sl * NS);
    }
    const int count = min(TT, t_end - t0);        // (four at a time; behind the last one steps and inputs are zero and change nothing)
#pragma unroll 1
    for (int f = 0; f < count; f += 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = f + i;
        f2 step[2], in[2], bb[NS], cv[NS], out[2];
        pair(&sm.step[warp][t][cg * 4], step[0], step[1]);
        pair(&sm.in[warp][t][cg * 4], in[0], in[1]);
#pragma unroll
        for (int k = 0; k < NS; k += 2) {
          pair(&sm.b[t][sl * NS + k].x, bb[k], bb[k + 1]);
          if (!ENDS) pair(&sm.c[t][sl * NS + k].x, cv[k], cv[k + 1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < NS; ++k) {
            h[j][k] = fma(HEADS ? step[j] : ex2(mul(step[j], a[j][k])), h[j][k], mul(in[j], bb[k]));
            if (!ENDS) out[j] = k == 0 ? mul(h[j][k], cv[k]) : fma(h[j][k], cv[k], out[j]);
          }
        if (!ENDS) *reinterpret_cast<ulonglong2*>(&sm.out[warp][t][lane]) = make_ulonglong2(out[0].v, out[1].v);
      }
    }
    if (!ENDS) {
      __syncwarp();
      auto finish = [&](auto fast) {
        constexpr bool FAST = decltype(fast)::value;
        Raw<T> ex[PASSES], ez[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int t = t0 + lt + i * LN;
          const int n = lt < TT && t < t_end ? left : 0;
          ex[i] = fetch(x + t * p.x_token, FAST && n > 0, n);
          if (z != nullptr) ez[i] = fetch(z + t * p.z_token, FAST && n > 0, n);
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int t = lt + i * LN;
          if (t >= TT || t0 + t >= t_end) continue;
          const float4 o4 = sum4(&sm.out[warp][t][lane % CG * LN], LN, 1, LN == 4 ? lane % CG >> 1 : 0);
          float o[4] = {o4.x, o4.y, o4.z, o4.w}, xs[4], g[4];
          ex[i].get(xs);
          if (z != nullptr) ez[i].get(g);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            o[j] = fmaf(skip[j], xs[j], o[j]);
            if (z != nullptr) o[j] *= g[j] * sigmoid(g[j]);
          }
          put(y + static_cast<long long>(t0 + t) * p.C, o, FAST || y_whole, left);
        }
      };
      if (whole) finish(Yes());
      else finish(No());
      __syncwarp();                               // (read before the next tile writes them)
    }
  }
  if (ENDS) {
    keep(p.starts + (pad_row + static_cast<long long>(seg + 1) * padded) * NP + sl * NS);
#pragma unroll
    for (int j = 0; j < 4; ++j) {                 // over the tokens' lanes
#pragma unroll
      for (int o = CG; o < 32; o <<= 1) total[j] += __shfl_xor_sync(0xffffffffu, total[j], o);
      if (lt == 0) p.sums[(static_cast<long long>(row) * p.segments + seg) * padded + static_cast<long long>(cb) * CB + warp * CW + lq + j] = total[j];
    }
  } else if (p.last != nullptr && seg == last_seg) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = c0 + cg * 4 + 2 * i;
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const int n = sl * NS + k;
        const float2 v = h[i][k].get();
        if (c < c_end && n < p.N) p.last[(r.at * p.C + c) * p.N + n] = v.x;
        if (c + 1 < c_end && n < p.N) p.last[(r.at * p.C + c + 1) * p.N + n] = v.y;
      }
    }
  }
}

// One token per row; a warp owns 32 channels of `rows_each` rows.  A lane forms the step, gate and output of channel 4 (lane / 4) + own_channel(lane % 4), and holds four states of each of
// its group's four channels; more than 16 states go by in sixteens.  grid (ceil(C / 128), ceil(R / rows_each)).
template <typename T, bool ONE>
__global__ void __launch_bounds__(THREADS)
token_kernel(const Args p, int rows_each) {
  const int lane = threadIdx.x & 31, sl = lane & 3, c4 = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * 32 + (lane >> 2) * 4, c = c4 + own_channel(sl);
  const bool on = c < p.C, fours_n = (p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.initial) & 15) == 0;
  if (c4 - (lane >> 2) * 4 >= p.C) return;
  const float skip = p.d != nullptr && on ? p.d[c] : 0.f;
  float a[4][4];
  auto rates = [&](int n0) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) a[j][k] = rate<false>(p, c4 + j, n0 + sl * 4 + k, 1);
  };
  if (ONE) rates(0);
  const int r1 = min(p.R, (static_cast<int>(blockIdx.y) + 1) * rows_each);
  for (int row = blockIdx.y * rows_each; row < r1; ++row) {
    T* y = static_cast<T*>(p.y) + static_cast<long long>(row) * p.C + c;
    const int pos = p.positions[row];
    const Row r = row_of(p, row);
    if (r.len == 0) {
      if (on) st(y, 0.f);
      continue;
    }
    const long long at = r.at;
    float* state = p.last + (at * p.C + c4) * p.N;
    const T *b = static_cast<const T*>(p.b) + row * p.b_row, *cc = static_cast<const T*>(p.c) + row * p.c_row;
    float x = 0.f, s = 0.f, g = 0.f;
    if (on) {
      x = ld(static_cast<const T*>(p.x) + row * p.x_row + c);
      s = p.dt_fp32 ? static_cast<const float*>(p.dt)[row * p.dt_row + c] : ld(static_cast<const bf16*>(p.dt) + row * p.dt_row + c);
      if (p.z != nullptr) g = ld(static_cast<const T*>(p.z) + row * p.z_row + c);
      s = p.softplus ? softplus(s) : s;
    }
    float out[4] = {0.f, 0.f, 0.f, 0.f};
    for (int n0 = 0; n0 < p.N; n0 += 16) {
      const int n = n0 + sl * 4;
      if (!ONE) rates(n0);
      float h[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        Raw<float> v = fetch(state + static_cast<long long>(j) * p.N + n, fours_n && n < p.N && c4 + j < p.C && pos > 0, 0);
        v.get(h[j]);
        if (!fours_n && pos > 0 && c4 + j < p.C) fetch(state + static_cast<long long>(j) * p.N + n, false, min(4, p.N - n)).get(h[j]);
      }
      float bb[4], cv[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) { bb[k] = n + k < p.N ? ld(b + n + k) : 0.f; cv[k] = n + k < p.N ? ld(cc + n + k) : 0.f; }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int from = (lane & ~3) + (j >> 1) + (j & 1) * 2;                     // the lane whose own channel j is
        const float sj = __shfl_sync(0xffffffffu, s, from), uj = sj * __shfl_sync(0xffffffffu, x, from);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[j][k] = fmaf(ex2(sj * a[j][k]), h[j][k], uj * bb[k]);
          out[j] = fmaf(h[j][k], cv[k], out[j]);
        }
        if (c4 + j < p.C) put(state + static_cast<long long>(j) * p.N + n, h[j], fours_n && n < p.N, p.N - n);
      }
    }
    float o = over_states<4>(out, sl) + skip * x;
    if (p.z != nullptr) o *= g * sigmoid(g);
    if (on) st(y, o);
  }
}

// One token per row, a decay per head.  A warp takes `ROWS` rows p of a head's [dim, N] state at a time, LN lanes a row.  grid (heads, parts, R).
template <typename T, int LN, int NS>
__global__ void __launch_bounds__(THREADS)
head_token_kernel(const Args p) {
  constexpr int CG = 32 / LN;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sl = lane % LN, cg = lane / LN;
  const int head = blockIdx.x, row = blockIdx.z, dim = p.C / p.heads, pos = p.positions[row];
  T* y = static_cast<T*>(p.y) + static_cast<long long>(row) * p.C + head * dim;
  const int first = (blockIdx.y * WARPS + warp) * 4 * CG, stride = gridDim.y * WARPS * 4 * CG;
  const Row r = row_of(p, row);
  if (r.len == 0) {
    for (int q = first; q < dim; q += stride)
      if (lane < 4 * CG && q + lane < dim) st(y + q + lane, 0.f);
    return;
  }
  const int group = head / (p.heads / p.groups);
  const long long at = r.at;
  float* state = p.last + (at * p.C + static_cast<long long>(head) * dim) * p.N;
  const bool fours_n = (p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.last) & 15) == 0;
  const T *x = static_cast<const T*>(p.x) + row * p.x_row + head * dim, *b = static_cast<const T*>(p.b) + row * p.b_row + group * p.N,
          *cc = static_cast<const T*>(p.c) + row * p.c_row + group * p.N;
  float s = p.dt_fp32 ? static_cast<const float*>(p.dt)[row * p.dt_row + head] : ld(static_cast<const bf16*>(p.dt) + row * p.dt_row + head);
  s += p.dt_bias == nullptr ? 0.f : p.dt_bias[head];
  s = p.softplus ? softplus(s) : s;
  const float decay = ex2(s * rate<true>(p, head * dim, 0, dim)), skip = p.d == nullptr ? 0.f : p.d[head];
  float bb[NS], cv[NS];
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    const int n = (k / 4 * LN + sl) * 4 + k % 4;
    bb[k] = n < p.N ? s * ld(b + n) : 0.f;
    cv[k] = n < p.N ? ld(cc + n) : 0.f;
  }
  for (int q = first + cg * 4; q - cg * 4 < dim; q += stride) {
    float h[4][NS], out[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < NS; k += 4) {
        const int n = (k / 4 * LN + sl) * 4;
        const bool on = q + j < dim && pos > 0;
        float f[4];
        if (fours_n) fetch(state + static_cast<long long>(q + j) * p.N + n, on && n < p.N, 0).get(f);
        else fetch(state + static_cast<long long>(q + j) * p.N + n, false, on ? p.N - n : 0).get(f);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[j][k + i] = f[i];
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float xj = q + j < dim ? ld(x + q + j) : 0.f;
#pragma unroll
      for (int k = 0; k < NS; k += 4) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[i] = fmaf(decay, h[j][k + i], xj * bb[k + i]);
          out[j] = fmaf(f[i], cv[k + i], out[j]);
        }
        const int n = (k / 4 * LN + sl) * 4;
        if (q + j < dim) put(state + static_cast<long long>(q + j) * p.N + n, f, fours_n && n < p.N, p.N - n);
      }
    }
    const float sum = over_states<LN>(out, sl);
    const int own = q + own_channel(sl);
    if (sl < 4 && own < dim) st(y + own, sum + skip * ld(x + own));
  }
}

template <typename T, typename TD, int LN, int NS, bool HEADS>
int scan_go(const Args& p, cudaStream_t stream) {
  using L = Lay<LN, NS>;
  const long long blocks = static_cast<long long>((p.C / p.groups + L::CB - 1) / L::CB) * p.groups;
  if (blocks * p.segments * p.R > 0x7fffffffLL) return -3;
  constexpr int ends = static_cast<int>(sizeof(Tile<LN, NS, true>)), whole = static_cast<int>(sizeof(Tile<LN, NS, false>));
  static_assert(ends <= 48 * 1024, "within what a launch has without asking");
  cudaError_t e = cudaFuncSetAttribute(scan_kernel<T, TD, LN, NS, HEADS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, whole);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (p.segments > 1) scan_kernel<T, TD, LN, NS, HEADS, true><<<static_cast<unsigned>(blocks * (p.segments - 1) * p.R), THREADS, ends, stream>>>(p);
  scan_kernel<T, TD, LN, NS, HEADS, false><<<static_cast<unsigned>(blocks * p.segments * p.R), THREADS, whole, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, typename TD>
int scan_any(const Args& p, cudaStream_t stream) {
  if (p.heads > 0) {
    if (p.N <= 16) return scan_go<T, TD, 4, 4, true>(p, stream);
    if (p.N <= 32) return scan_go<T, TD, 8, 4, true>(p, stream);
    if (p.N <= 64) return scan_go<T, TD, 16, 4, true>(p, stream);
    if (p.N <= 128) return scan_go<T, TD, 32, 4, true>(p, stream);
    if (p.N <= 256) return scan_go<T, TD, 32, 8, true>(p, stream);
    return -3;
  }
  if (p.N <= 16) return scan_go<T, TD, 4, 4, false>(p, stream);
  if (p.N <= 32) return scan_go<T, TD, 8, 4, false>(p, stream);
  if (p.N <= 64) return scan_go<T, TD, 16, 4, false>(p, stream);
  if (p.N <= 128) return scan_go<T, TD, 32, 4, false>(p, stream);
  return -3;
}

template <typename T>
int token_any(const Args& p, cudaStream_t stream) {
  if (p.heads > 0) {
    const dim3 grid(p.heads, 1, p.R);
    if (p.R > 65535) return -3;
    if (p.N <= 16) head_token_kernel<T, 4, 4><<<grid, THREADS, 0, stream>>>(p);
    else if (p.N <= 32) head_token_kernel<T, 8, 4><<<grid, THREADS, 0, stream>>>(p);
    else if (p.N <= 64) head_token_kernel<T, 16, 4><<<grid, THREADS, 0, stream>>>(p);
    else if (p.N <= 128) head_token_kernel<T, 32, 4><<<grid, THREADS, 0, stream>>>(p);
    else if (p.N <= 256) head_token_kernel<T, 32, 8><<<grid, THREADS, 0, stream>>>(p);
    else return -3;
    return static_cast<int>(cudaGetLastError());
  }
  const int rows_each = 1;
  const dim3 grid((p.C + THREADS - 1) / THREADS, (p.R + rows_each - 1) / rows_each);
  if (grid.y > 65535) return -3;
  if (p.N <= 16) token_kernel<T, true><<<grid, THREADS, 0, stream>>>(p, rows_each);
  else token_kernel<T, false><<<grid, THREADS, 0, stream>>>(p, rows_each);
  return static_cast<int>(cudaGetLastError());
}

inline bool args_ok(const Args& p) {
  if (p.R < 1 || p.T < 1 || p.C < 1 || p.N < 1 || p.groups < 1 || p.segments < 1 || p.segment < 1) return false;
  if (p.heads > 0 ? p.C % p.heads || p.heads % p.groups : p.groups != 1) return false;
  if (p.x == nullptr || p.dt == nullptr || p.b == nullptr || p.c == nullptr || p.a == nullptr || p.y == nullptr) return false;
  if (p.segment % EVERY || static_cast<long long>(p.segments) * p.segment < p.T || (p.segments > 1 && (p.starts == nullptr || p.sums == nullptr))) return false;
  return p.positions == nullptr || (p.lengths != nullptr && p.initial == p.last);
}

}  // namespace selective
}  // namespace dewb

using namespace dewb::selective;

// Channels and states as the workspaces pad them: checkpoints, starts [.., padded C, padded N], sums [.., padded C].
extern "C" int dewb_selective_padding(int C, int N, int groups, int* padded) {
  if (C < 1 || N < 1 || groups < 1 || C % groups) return -3;
  const int ln = N <= 16 ? 4 : N <= 32 ? 8 : N <= 64 ? 16 : 32, np = N <= 128 ? ln * 4 : 256, cb = WARPS * 4 * (32 / ln);
  padded[0] = (C / groups + cb - 1) / cb * cb * groups;
  padded[1] = np;
  return N <= 256 ? 0 : -3;
}

extern "C" int dewb_selective_scan(const dewb_selective_args* a, int fp32, void* stream_ptr) {
  if (a == nullptr || !args_ok(*a)) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (fp32) return a->dt_fp32 ? scan_any<float, float>(*a, stream) : -3;
  return a->dt_fp32 ? scan_any<bf16, float>(*a, stream) : scan_any<bf16, bf16>(*a, stream);
}

// One token per row, with positions and a state.
extern "C" int dewb_selective_token(const dewb_selective_args* a, int fp32, void* stream_ptr) {
  if (a == nullptr || !args_ok(*a) || a->T != 1 || a->positions == nullptr || a->last == nullptr) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  return fp32 ? token_any<float>(*a, stream) : token_any<bf16>(*a, stream);
}
