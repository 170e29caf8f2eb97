// The selective state space scan forward, for sm_100a (the equations and the lanes' layout: selective.cuh), over whole rows or over a call's rows with the states that a store keeps.
//
//   scan_kernel       tokens one after another with the states in registers, in fp32.  The row may be cut into segments that run side by side; the first launch (ENDS) then
//                     forms what each segment makes of a state of zeros and the sum of its steps, and the second one composes what stands in front of a segment from those
//   token_kernel      one token per row: the state is read and written once
//
// A call row whose first position is 0 starts from zero; positions below 0 are padding at a row's end: they change no state and give zeros.
// Inputs and outputs are bf16 or fp32 (template T; the steps' logits either), everything else fp32.  Compiled without fast math.
//
// What bounds scan_kernel is the exponential of every token, channel and state: the special-function unit takes eight cycles for a warp's, so 4 rows of 2048 tokens of 4096 channels of 16
// states cannot take less than 119 us (149 with those of steps and gates; the bytes, 41).  The ENDS pass comes to 75 % of that rate; the other reaches 56 to 70 %, where a SM has 16
// warps: 247 us in eight segments and 162 for their ends, or 396 for whole rows with two states a lane and 7 warps an SM, whose chains are then what takes the time (a warp waits 1.8
// of 5 cycles for the instruction before, 1.1 for an exponential or shared memory).  token_kernel is bound by memory: 128 rows of 8192 channels 27 us, 4.9 TB/s (32 where
// every load asks whether its channel and states are there: 450 instructions a row of 32 channels; states three rows ahead in shared memory instead of one in registers: 27).
#include "../common/selective.cuh"

namespace dewb {
namespace selective {

template <int LN, int NS, bool ENDS>
struct Tile {
  using L = Lay<LN, NS>;
  float step[WARPS][L::TT][L::CW], in[WARPS][L::TT][L::CW];                  // s, s x
  float2 b[L::TT][L::NP], c[ENDS ? 1 : L::TT][L::NP];                        // each number twice: beside two channels
  float4 out[ENDS ? 1 : WARPS][ENDS ? 1 : L::TT][32];                        // a lane's share of sum C h, four channels
};

// grid R * segments * channel blocks.
//   starts[r, 0]       the state that row r begins with          starts[r, j]   what segment j - 1 ends with: from there on for j = 1, from zeros for the others
//   sums[r, j]         the sum of segment j's steps, per channel
// A tile's x and steps come a tile ahead, in registers as they lie in memory (converted on arrival, every tile waited for them: 10 to 25 % of the time); what the end of a tile needs (x
// again, z) is asked for at its beginning (L2) and read then.  Channels go in pairs, two to an instruction: no more of them a second, but half as many to issue (one at a time: 3 %
// slower here, 13 % in the gradients).  The sums over states are formed at the end of a tile from what every lane leaves in shared memory: 4 whole rows of 2048 tokens of 4096 channels take
// 539 us with four states a lane and 396 with two, which have twice the sums to cross lanes (four states a lane with shuffles after every two tokens 665, after every four 528).  NS 4, 2, 1:
// what _split in ops/selective.py says of each.
template <typename T, typename TD, int LN, int NS, bool ENDS>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 3 : 4)
scan_kernel(const Args p) {
  using L = Lay<LN, NS>;
  constexpr int CG = L::CG, CW = L::CW, CB = L::CB, NP = L::NP, TT = L::TT, PASSES = L::PASSES, BC = (TT * NP / 4 + THREADS - 1) / THREADS;
  extern __shared__ __align__(16) char raw[];
  Tile<LN, NS, ENDS>& sm = *reinterpret_cast<Tile<LN, NS, ENDS>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sl = lane % LN, cg = lane / LN;
  const int blocks = (p.C + CB - 1) / CB, padded = p.padded;
  const int segments = ENDS ? p.segments - 1 : p.segments;
  const int cb = blockIdx.x % blocks, seg = blockIdx.x / blocks % segments, row = blockIdx.x / blocks / segments;
  const int c_block = cb * CB, c0 = c_block + warp * CW;
  const Row r = row_of(p, row);
  const int t_begin = seg * p.segment, t_end = min(r.len, t_begin + p.segment), t_stop = min(p.T, t_begin + p.segment);
  // where this lane loads and stores: four channels of token lane / CG + pass * LN
  const int lt = lane / CG, lq = lane % CG * 4, lc = c0 + lq, left = max(0, min(4, p.C - lc));
  T* y = static_cast<T*>(p.y) + static_cast<long long>(row) * p.T * p.C + lc;
  const bool y_whole = left == 4 && (p.C & 3) == 0;
  const int last_seg = r.len > 0 ? (r.len - 1) / p.segment : -1;
  if (!ENDS) {
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t = max(t_begin, t_end) + lt; t < t_stop; t += LN) put(y + static_cast<long long>(t) * p.C, none, y_whole, left);
  }
  if (seg > last_seg) return;

  f2 a[2][NS], h[2][NS];                          // of channels 2 i and 2 i + 1
  const long long pad_row = static_cast<long long>(row) * p.segments * padded + c0 + cg * 4;   // of segment 0, this lane's first channel
  auto held = [&](int c, int n) { return (ENDS || p.segments == 1) && seg == 0 && r.held && c < p.C && n < p.N ? p.initial[(r.at * p.C + c) * p.N + n] : 0.f; };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = c0 + cg * 4 + 2 * i;
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int n = sl * NS + k;
      a[i][k] = f2(rate<false>(p, c, n, 1), rate<false>(p, c + 1, n, 1));
      h[i][k] = f2(held(c, n), held(c + 1, n));
    }
  }
  // the states of this lane's channels at `to`, rows of NP
  auto keep = [&](float* to) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float e[2][NS];
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const float2 v = h[i][k].get();
        e[0][k] = v.x; e[1][k] = v.y;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* q = to + (2 * i + j) * NP;
        if constexpr (NS == 1) *q = e[j][0];
        else if constexpr (NS == 2) *reinterpret_cast<float2*>(q) = make_float2(e[j][0], e[j][1]);
        else
#pragma unroll
          for (int k = 0; k < NS; k += 4) *reinterpret_cast<float4*>(q + k) = make_float4(e[j][k], e[j][k + 1], e[j][k + 2], e[j][k + 3]);
      }
    }
  };
  if (ENDS && seg == 0) keep(p.starts + pad_row * NP + sl * NS);
  if (!ENDS && p.segments > 1) {                  // what stands in front of the segment
#pragma unroll 2
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
  float skip[4], total[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) skip[j] = p.d != nullptr && !ENDS ? p.d[min(lc + j, p.C - 1)] : 0.f;
  const T* x = static_cast<const T*>(p.x) + row * p.x_row + lc;
  const TD* dt = static_cast<const TD*>(p.dt) + row * p.dt_row + lc;
  const T* z = p.z == nullptr || ENDS ? nullptr : static_cast<const T*>(p.z) + row * p.z_row + lc;
  const T* b = static_cast<const T*>(p.b) + row * p.b_row;
  const T* cc = static_cast<const T*>(p.c) + row * p.c_row;
  // whole pieces of four wherever the block loads and stores
  const bool whole = c_block + CB <= p.C && (p.C & 3) == 0 && fours<T>(p.x, p.x_row, p.x_token) && (z == nullptr || fours<T>(p.z, p.z_row, p.z_token)) &&
                     fours<TD>(p.dt, p.dt_row, p.dt_token);

  Raw<T> rx[PASSES];
  Raw<TD> rd[PASSES];
  Raw<T> rb[BC], rc[ENDS ? 1 : BC];
  const bool b_whole = fours<T>(b, p.b_row, p.b_token), c_whole = fours<T>(cc, p.c_row, p.c_token);
  auto bring = [&](int t0, auto fast) {
    constexpr bool FAST = decltype(fast)::value;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int t = t0 + lt + i * LN;
      const bool on = FAST ? LN <= TT || lt < TT : lt < TT && t < t_end;
      const int n = on ? left : 0;
      if (FAST) { if (on) rx[i] = fetch(x + t * p.x_token, true, 4); }
      else rx[i] = fetch(x + t * p.x_token, false, n);
      if (FAST) { if (on) rd[i] = fetch(dt + t * p.dt_token, true, 4); }
      else rd[i] = fetch(dt + t * p.dt_token, false, n);
      if (z != nullptr && n > 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(z + t * p.z_token));
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) {                // four states of a token
      const int at = tid + i * THREADS, t = t0 + at / (NP / 4), n = at % (NP / 4) * 4;
      const int there = at < TT * NP / 4 && t < t_end ? max(0, min(4, p.N - n)) : 0;
      rb[i] = fetch(b + t * p.b_token + n, b_whole && there == 4, there);
      if (!ENDS) rc[i] = fetch(cc + t * p.c_token + n, c_whole && there == 4, there);
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
        rd[i].get(s);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (p.softplus) s[j] = softplus(s[j]);
          if (!FAST && (j >= left || t0 + t >= t_end)) s[j] = xs[j] = 0.f;
          if (ENDS && (LN <= TT || t < TT)) total[j] += s[j];
          xs[j] *= s[j];
        }
        if (LN <= TT || t < TT) {
          *reinterpret_cast<float4*>(&sm.step[warp][t][lq]) = make_float4(s[0], s[1], s[2], s[3]);
          *reinterpret_cast<float4*>(&sm.in[warp][t][lq]) = make_float4(xs[0], xs[1], xs[2], xs[3]);
        }
      }
    };
    if (t0 + TT <= t_end && c_block + CB <= p.C) stage(Yes());
    else stage(No());
#pragma unroll
    for (int i = 0; i < BC; ++i) {
      const int at = tid + i * THREADS, t = at / (NP / 4), n = at % (NP / 4) * 4;
      if (TT * NP / 4 % THREADS == 0 || at < TT * NP / 4) {
        twice(&sm.b[t][n], rb[i]);
        if (!ENDS) twice(&sm.c[t][n], rc[i]);
      }
    }
    __syncthreads();
    if (t0 + TT < t_end) next(t0 + TT);
    if (!ENDS && p.checkpoints != nullptr) {
      static_assert(EVERY == TT, "a kept state a tile");
      keep(p.checkpoints + ((static_cast<long long>(row) * ((p.T + EVERY - 1) / EVERY) + t0 / EVERY) * padded + c0 + cg * 4) * NP + sl * NS);
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
        pairs(&sm.b[t][sl * NS], bb);
        if (!ENDS) pairs(&sm.c[t][sl * NS], cv);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < NS; ++k) {
            h[j][k] = fma(ex2(mul(step[j], a[j][k])), h[j][k], mul(in[j], bb[k]));
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
          const float4 o4 = sum4(&sm.out[warp][t][lane % CG * LN], LN, 1, turn_of<LN>(lane));
          float o[4] = {o4.x, o4.y, o4.z, o4.w}, xs[4], g[4];
          ex[i].get(xs);
          if (z != nullptr) ez[i].get(g);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            o[j] = fmaf(skip[j], xs[j], o[j]);
            if (z != nullptr) o[j] *= g[j] * gate<T>(g[j]);
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
      if (lt == 0) p.sums[(static_cast<long long>(row) * p.segments + seg) * padded + c0 + lq + j] = total[j];
    }
  } else if (p.last != nullptr && seg == last_seg) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = c0 + cg * 4 + 2 * i;
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const int n = sl * NS + k;
        const float2 v = h[i][k].get();
        if (c < p.C && n < p.N) p.last[(r.at * p.C + c) * p.N + n] = v.x;
        if (c + 1 < p.C && n < p.N) p.last[(r.at * p.C + c + 1) * p.N + n] = v.y;
      }
    }
  }
}

// One token per row; a warp owns 32 channels of `rows_each` rows, whose rates it reads once.  A lane holds four states of
// each of channels lane / 4 + 8 j (so that a load of all lanes is 512 bytes in a row), and forms the step, gate and output of that of j = own_channel(lane % 4); more than 16 states go by
// in sixteens.  ALL: a warp's channels and a lane's states are all there, from boundaries of four.  The next row's states are on their way while one is worked on.
// grid (ceil(C / 128), ceil(R / rows_each)).
template <typename T, bool ONE, bool ALL>
__global__ void __launch_bounds__(THREADS)
token_kernel(const Args p, int rows_each) {
  const int lane = threadIdx.x & 31, sl = lane & 3, c4 = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * 32 + (lane >> 2), c = c4 + 8 * own_channel(sl);
  const bool on = ALL || c < p.C, whole = ALL || ((p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.initial) & 15) == 0);
  if (c4 - (lane >> 2) >= p.C) return;
  const float skip = p.d != nullptr && on ? p.d[c] : 0.f;
  float a[4][4];
  auto rates = [&](int n0) {
    const int n = n0 + sl * 4;
    const bool all = ALL || ((p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.a) & 15) == 0 && n < p.N);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int there = ALL ? 4 : c4 + 8 * j < p.C ? max(0, min(4, p.N - n)) : 0;
      fetch(p.a + static_cast<long long>(c4 + 8 * j) * p.N + n, all && there == 4, there).get(a[j]);
#pragma unroll
      for (int k = 0; k < 4; ++k) a[j][k] = k < there ? times_log2e(rate_of(p, a[j][k])) : 0.f;
    }
  };
  const bool b_whole = ALL || ((p.N & 3) == 0 && fours<T>(p.b, p.b_row, 0)), c_whole = ALL || ((p.N & 3) == 0 && fours<T>(p.c, p.c_row, 0));
  const int first = blockIdx.y * rows_each, rows = min(rows_each, p.R - first);
  // the rows' places, a lane each: what a row's loads begin with is there before its turn
  const Row mine = lane < rows ? row_of(p, first + lane) : Row{0, false, 0};
  struct Item {
    int len;
    bool held;
    float* state;
    Raw<float> h[4];
    Raw<T> b, c;
    float x, s, g;
  };
  auto states = [&](Item& it, int n0) {
    const int n = n0 + sl * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int there = it.held && (ALL || c4 + 8 * j < p.C) ? ALL ? 4 : max(0, min(4, p.N - n)) : 0;
      it.h[j] = fetch(it.state + static_cast<long long>(8 * j) * p.N + n, whole && there == 4, ALL ? 0 : there);
    }
  };
  auto narrow = [&](Item& it, int row, int n0) {
    const int n = n0 + sl * 4, there = ALL ? 4 : max(0, min(4, p.N - n));
    it.b = fetch(static_cast<const T*>(p.b) + row * p.b_row + n, b_whole && there == 4, there);
    it.c = fetch(static_cast<const T*>(p.c) + row * p.c_row + n, c_whole && there == 4, there);
  };
  auto bring = [&](Item& it, int i) {
    const int row = first + i;
    it.len = __shfl_sync(0xffffffffu, mine.len, i);
    it.held = __shfl_sync(0xffffffffu, mine.held, i) && it.len > 0;
    it.state = p.last + (static_cast<long long>(__shfl_sync(0xffffffffu, static_cast<int>(mine.at), i)) * p.C + c4) * p.N;
    it.x = it.s = it.g = 0.f;
    if (it.len > 0 && on) {
      it.x = ld(static_cast<const T*>(p.x) + row * p.x_row + c);
      it.s = p.dt_fp32 ? static_cast<const float*>(p.dt)[row * p.dt_row + c] : ld(static_cast<const bf16*>(p.dt) + row * p.dt_row + c);
      if (p.z != nullptr) it.g = ld(static_cast<const T*>(p.z) + row * p.z_row + c);
    }
    states(it, 0);
    if (ONE) narrow(it, row, 0);
  };
  auto work = [&](Item& it, int row) {
    T* y = static_cast<T*>(p.y) + static_cast<long long>(row) * p.C + c;
    if (it.len == 0) {
      if (on) st(y, 0.f);
      return;
    }
    const float s = p.softplus ? softplus(it.s) : it.s, u = s * it.x;
    float out[4] = {0.f, 0.f, 0.f, 0.f};
    for (int n0 = 0; n0 < p.N; n0 += 16) {
      const int n = n0 + sl * 4;
      if (!ONE) {
        rates(n0);
        if (n0 > 0) states(it, n0);
        narrow(it, row, n0);
      }
      float b[4], cv[4];
      it.b.get(b);
      it.c.get(cv);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int from = (lane & ~3) + (j >> 1) + (j & 1) * 2;                     // the lane whose own channel j is
        const float sj = __shfl_sync(0xffffffffu, s, from), uj = __shfl_sync(0xffffffffu, u, from);
        float h[4];
        it.h[j].get(h);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[k] = fmaf(ex2(sj * a[j][k]), h[k], uj * b[k]);
          out[j] = fmaf(h[k], cv[k], out[j]);
        }
        if (ALL || c4 + 8 * j < p.C) put(it.state + static_cast<long long>(8 * j) * p.N + n, h, ALL || (whole && n < p.N), p.N - n);
      }
      if (ONE) break;
    }
    float o = over_states<4>(out, sl) + skip * it.x;
    if (p.z != nullptr) o *= it.g * gate<T>(it.g);
    if (on) st(y, o);
  };
  Item now, next;
  bring(next, 0);
  if (ONE) rates(0);
  for (int i = 0; i < rows; ++i) {
    now = next;
    if (i + 1 < rows) bring(next, i + 1);
    work(now, first + i);
  }
}

template <typename T, typename TD, int LN, int NS>
int scan_go(const Args& p, cudaStream_t stream) {
  using L = Lay<LN, NS>;
  const long long blocks = (p.C + L::CB - 1) / L::CB;
  if (blocks * p.segments * p.R > 0x7fffffffLL) return -3;
  constexpr int ends = static_cast<int>(sizeof(Tile<LN, NS, true>)), whole = static_cast<int>(sizeof(Tile<LN, NS, false>));
  static_assert(ends <= 48 * 1024, "within what a launch has without asking");
  cudaError_t e = cudaFuncSetAttribute(scan_kernel<T, TD, LN, NS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, whole);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (p.segments > 1) scan_kernel<T, TD, LN, NS, true><<<static_cast<unsigned>(blocks * (p.segments - 1) * p.R), THREADS, ends, stream>>>(p);
  scan_kernel<T, TD, LN, NS, false><<<static_cast<unsigned>(blocks * p.segments * p.R), THREADS, whole, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, typename TD>
int scan_any(const Args& p, cudaStream_t stream) {
  if (p.N <= 16) {
    if (p.states_each == 1) return scan_go<T, TD, 16, 1>(p, stream);
    if (p.states_each == 2) return scan_go<T, TD, 8, 2>(p, stream);
    return scan_go<T, TD, 4, 4>(p, stream);
  }
  if (p.N <= 32) return scan_go<T, TD, 8, 4>(p, stream);
  if (p.N <= 64) return scan_go<T, TD, 16, 4>(p, stream);
  if (p.N <= 128) return scan_go<T, TD, 32, 4>(p, stream);
  return -3;
}

template <typename T>
int token_any(const Args& p, cudaStream_t stream) {
  const int across = (p.C + THREADS - 1) / THREADS, rows_each = p.states_each;
  const dim3 grid(across, (p.R + rows_each - 1) / rows_each);
  if (grid.y > 65535) return -3;
  const bool all = (p.N & 15) == 0 && (p.C & 31) == 0 && ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.last)) & 15) == 0 && fours<T>(p.b, p.b_row, 0) &&
                   fours<T>(p.c, p.c_row, 0);
  if (p.N <= 16) {
    if (all) token_kernel<T, true, true><<<grid, THREADS, 0, stream>>>(p, rows_each);
    else token_kernel<T, true, false><<<grid, THREADS, 0, stream>>>(p, rows_each);
  } else if (all) {
    token_kernel<T, false, true><<<grid, THREADS, 0, stream>>>(p, rows_each);
  } else {
    token_kernel<T, false, false><<<grid, THREADS, 0, stream>>>(p, rows_each);
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace selective
}  // namespace dewb

using namespace dewb::selective;

extern "C" int dewb_selective_scan(const dewb_selective_args* a, int fp32, void* stream_ptr) {
  if (a == nullptr || a->heads != 0 || !args_ok(*a)) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (fp32) return a->dt_fp32 ? scan_any<float, float>(*a, stream) : -3;
  return a->dt_fp32 ? scan_any<bf16, float>(*a, stream) : scan_any<bf16, bf16>(*a, stream);
}

// One token per row, with positions and a state.
extern "C" int dewb_selective_token(const dewb_selective_args* a, int fp32, void* stream_ptr) {
  if (a == nullptr || a->heads != 0 || !args_ok(*a) || a->T != 1 || a->positions == nullptr || a->last == nullptr || a->states_each < 1 || a->states_each > 32) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  return fp32 ? token_any<float>(*a, stream) : token_any<bf16>(*a, stream);
}
