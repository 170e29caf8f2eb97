// The state space scan with a decay per head, for sm_100a (selective.cuh: arguments, rows, segments):  h[p, n] = e^{s A} h[p, n] + s x_p B_n,  y_p = sum_n C_n h[p, n] + D x_p.
//
//   head_scan_kernel   tokens one after another with the states in registers, in fp32; segments of a row side by side as in selective_scan.cu
//   head_token_kernel  one token per row: the state is read and written once
//   head_steps_kernel  what the scan in chunks on the tensor cores (ssd_sm100.cu) wants of a call's rows: their steps, rates and places
//
// A lane owns eight channels (rows p of the state) and NS states of each, in pairs; LN lanes share the states.  A decay is one exponential a head, so what counts are three
// multiply-adds a state, and how often a number is fetched for them: B and C serve eight channels, a step all states (four channels a lane in pairs of channels, B and C twice in shared
// memory: 104 us for 5 rows of up to 300 tokens, 24 heads of 48 over 80 states, fp32; so, and in segments, 60).  head_token_kernel: 128 rows of 64 heads of 64 x 128 85 us, 6.1 TB/s.
// Compiled without fast math.
#include "../common/selective.cuh"

namespace dewb {
namespace selective {

constexpr int EIGHT = 8;               // channels of a lane
constexpr int MOST_Z = 65535;          // blocks along a grid's third axis

template <int LN, int NS>
struct HeadLay {
  static constexpr int CG = 32 / LN, CW = EIGHT * CG, CB = WARPS * CW, NP = LN * NS, TT = 16;
  static constexpr int PIECES = CW / 4, STEP = 32 / PIECES, PASSES = TT / STEP;      // pieces of four channels of a token; tokens that a warp loads at once
};

template <int LN, int NS>
struct HeadTile {
  using L = HeadLay<LN, NS>;
  float2 step[WARPS][L::TT][L::CW], in[WARPS][L::TT][L::CW];                         // the decay and s x, each twice: beside two states
  float b[L::TT][L::NP], c[L::TT][L::NP];
  float out[WARPS][L::TT][L::CW];
};

// Sums of eight channels' numbers over LN lanes: lane keeps 8 / min(8, LN) of them, from the returned channel on.
template <int LN>
__device__ __forceinline__ int eight_over_states(float (&v)[EIGHT], int sl) {
  int base = 0;
#pragma unroll
  for (int o = 1, half = 4; o < LN; o <<= 1, half >>= 1) {
    if (half > 0) {
      const bool upper = sl & o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < half) v[i] = (upper ? v[i + half] : v[i]) + __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + half], o);
      base += upper ? half : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return base;
}

// grid R * segments * channel blocks; a channel block lies within one group (that shares B and C).  starts and sums as in selective_scan.cu.
template <typename T, typename TD, int LN, int NS, bool ENDS>
__global__ void __launch_bounds__(THREADS, NS > 4 || LN <= 8 ? 2 : sizeof(T) == 4 ? 3 : 4)
head_scan_kernel(const Args p) {
  using L = HeadLay<LN, NS>;
  constexpr int CW = L::CW, CB = L::CB, NP = L::NP, TT = L::TT, PASSES = L::PASSES, BC = (TT * NP / 4 + THREADS - 1) / THREADS, KEPT = LN >= 8 ? 1 : 8 / LN;
  extern __shared__ __align__(16) char raw[];
  HeadTile<LN, NS>& sm = *reinterpret_cast<HeadTile<LN, NS>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sl = lane % LN, cg = lane / LN;
  const int per = p.C / p.groups, in_group = (per + CB - 1) / CB, blocks = in_group * p.groups, padded = p.padded * p.groups;
  const int segments = ENDS ? p.segments - 1 : p.segments;
  const int cb = blockIdx.x % blocks, seg = blockIdx.x / blocks % segments, row = blockIdx.x / blocks / segments;
  const int group = cb / in_group, c_end = (group + 1) * per, c_block = group * per + cb % in_group * CB, c0 = c_block + warp * CW, dim = p.C / p.heads;
  const Row r = row_of(p, row);
  const int t_begin = seg * p.segment, t_end = min(r.len, t_begin + p.segment), t_stop = min(p.T, t_begin + p.segment);
  // where this lane loads and stores: four channels of token lt + pass * STEP
  const int lt = lane / L::PIECES, lq = lane % L::PIECES * 4, lc = c0 + lq, left = max(0, min(4, c_end - lc));
  T* y = static_cast<T*>(p.y) + static_cast<long long>(row) * p.T * p.C + lc;
  const bool y_whole = left == 4 && ((c_block | p.C) & 3) == 0;
  const int last_seg = r.len > 0 ? (r.len - 1) / p.segment : -1;
  if (!ENDS) {
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t = max(t_begin, t_end) + lt; t < t_stop; t += L::STEP) put(y + static_cast<long long>(t) * p.C, none, y_whole, left);
  }
  if (seg > last_seg) return;

  f2 h[EIGHT][NS / 2];
  const int mine = c0 + cg * EIGHT, pad_c = group * p.padded + mine - group * per;          // this lane's first channel, and where the workspaces have it
  const long long pad_row = static_cast<long long>(row) * p.segments * padded + pad_c;       // of segment 0
  auto held = [&](int c, int n) { return (ENDS || p.segments == 1) && seg == 0 && r.held && c < c_end && n < p.N ? p.initial[(r.at * p.C + c) * p.N + n] : 0.f; };
#pragma unroll
  for (int j = 0; j < EIGHT; ++j)
#pragma unroll
    for (int k = 0; k < NS / 2; ++k) h[j][k] = f2(held(mine + j, sl * NS + 2 * k), held(mine + j, sl * NS + 2 * k + 1));
  auto keep = [&](float* to) {
#pragma unroll
    for (int j = 0; j < EIGHT; ++j)
#pragma unroll
      for (int k = 0; k < NS / 2; k += 2) *reinterpret_cast<ulonglong2*>(to + j * NP + 2 * k) = make_ulonglong2(h[j][k].v, h[j][k + 1].v);
  };
  if (ENDS && seg == 0) keep(p.starts + pad_row * NP + sl * NS);
  if (!ENDS && p.segments > 1) {                  // what stands in front of the segment
#pragma unroll 2
    for (int q = min(seg, 1); q <= seg; ++q) {
      const long long at = pad_row + static_cast<long long>(q) * padded;
#pragma unroll
      for (int j = 0; j < EIGHT; ++j) {
        const float decay = q > 1 ? ex2(p.sums[at - padded + j] * rate<true>(p, min(mine + j, p.C - 1), 0, dim)) : 1.f;
        f2 e[NS / 2];
        pairs(reinterpret_cast<const float2*>(p.starts + (at + j) * NP + sl * NS), e);
#pragma unroll
        for (int k = 0; k < NS / 2; ++k) h[j][k] = fma(f2(decay, decay), h[j][k], e[k]);
      }
    }
  }

  float rates[4], bias[4], skip[4], total[4] = {0.f, 0.f, 0.f, 0.f};
  int head[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = min(lc + j, p.C - 1);
    head[j] = c / dim;
    rates[j] = rate<true>(p, c, 0, dim);
    bias[j] = p.dt_bias != nullptr ? p.dt_bias[head[j]] : 0.f;
    skip[j] = p.d != nullptr && !ENDS ? p.d[head[j]] : 0.f;
  }
  const T* x = static_cast<const T*>(p.x) + row * p.x_row + lc;
  const TD* dt = static_cast<const TD*>(p.dt) + row * p.dt_row;
  const T* b = static_cast<const T*>(p.b) + row * p.b_row + group * p.N;
  const T* cc = static_cast<const T*>(p.c) + row * p.c_row + group * p.N;
  const bool x_whole = left == 4 && (c_block & 3) == 0 && fours<T>(p.x, p.x_row, p.x_token), b_whole = fours<T>(b, p.b_row, p.b_token), c_whole = fours<T>(cc, p.c_row, p.c_token);
  Raw<T> rx[PASSES], rb[BC], rc[ENDS ? 1 : BC];
  uint32_t rd[PASSES][4];
  auto bring = [&](int t0) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int t = t0 + lt + i * L::STEP, n = t < t_end ? left : 0;
      rx[i] = fetch(x + t * p.x_token, x_whole && n == 4, n);
#pragma unroll
      for (int j = 0; j < 4; ++j) rd[i][j] = j < n ? word(dt + t * p.dt_token + head[j]) : 0u;
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) {                // four states of a token
      const int at = tid + i * THREADS, t = t0 + at / (NP / 4), n = at % (NP / 4) * 4;
      const int there = at < TT * NP / 4 && t < t_end ? max(0, min(4, p.N - n)) : 0;
      rb[i] = fetch(b + t * p.b_token + n, b_whole && there == 4, there);
      if (!ENDS) rc[i] = fetch(cc + t * p.c_token + n, c_whole && there == 4, there);
    }
  };
  bring(t_begin);
  for (int t0 = t_begin; t0 < t_end; t0 += TT) {
    float xs[PASSES][4];
    __syncthreads();                              // (the tile before has been read)
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int t = lt + i * L::STEP, n = t0 + t < t_end ? left : 0;
      float u[4], e[4];
      rx[i].get(xs[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = value<TD>(rd[i][j]) + bias[j], step = j < n ? (p.softplus ? softplus(s) : s) : 0.f;
        u[j] = j < n ? step * xs[i][j] : 0.f;
        if (ENDS) total[j] += step;
        e[j] = ex2(step * rates[j]);
      }
      reinterpret_cast<float4*>(&sm.step[warp][t][lq])[0] = make_float4(e[0], e[0], e[1], e[1]);
      reinterpret_cast<float4*>(&sm.step[warp][t][lq])[1] = make_float4(e[2], e[2], e[3], e[3]);
      reinterpret_cast<float4*>(&sm.in[warp][t][lq])[0] = make_float4(u[0], u[0], u[1], u[1]);
      reinterpret_cast<float4*>(&sm.in[warp][t][lq])[1] = make_float4(u[2], u[2], u[3], u[3]);
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) {
      const int at = tid + i * THREADS, t = at / (NP / 4), n = at % (NP / 4) * 4;
      if (TT * NP / 4 % THREADS == 0 || at < TT * NP / 4) {
        float f[4];
        rb[i].get(f);
        *reinterpret_cast<float4*>(&sm.b[t][n]) = make_float4(f[0], f[1], f[2], f[3]);
        if (!ENDS) {
          rc[i].get(f);
          *reinterpret_cast<float4*>(&sm.c[t][n]) = make_float4(f[0], f[1], f[2], f[3]);
        }
      }
    }
    __syncthreads();
    if (t0 + TT < t_end) bring(t0 + TT);
    const int count = min(TT, t_end - t0);
#pragma unroll 2
    for (int t = 0; t < count; ++t) {
      f2 step[EIGHT], in[EIGHT], bb[NS / 2], cv[NS / 2];
      pairs(&sm.step[warp][t][cg * EIGHT], step);
      pairs(&sm.in[warp][t][cg * EIGHT], in);
      pairs(reinterpret_cast<const float2*>(&sm.b[t][sl * NS]), bb);
      if (!ENDS) pairs(reinterpret_cast<const float2*>(&sm.c[t][sl * NS]), cv);
      float o[EIGHT];
#pragma unroll
      for (int j = 0; j < EIGHT; ++j) {
        f2 sum;
#pragma unroll
        for (int k = 0; k < NS / 2; ++k) {
          h[j][k] = fma(step[j], h[j][k], mul(in[j], bb[k]));
          if (!ENDS) sum = k == 0 ? mul(h[j][k], cv[k]) : fma(h[j][k], cv[k], sum);
        }
        if (!ENDS) {
          const float2 v = sum.get();
          o[j] = v.x + v.y;
        }
      }
      if (!ENDS) {
        const int own = cg * EIGHT + eight_over_states<LN>(o, sl);
        if (LN <= 8 || sl < 8) {
#pragma unroll
          for (int i = 0; i < KEPT; ++i) sm.out[warp][t][own + i] = o[i];
        }
      }
    }
    if (!ENDS) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int t = lt + i * L::STEP;
        if (t0 + t >= t_end) continue;
        const float4 v = *reinterpret_cast<const float4*>(&sm.out[warp][t][lq]);
        const float o[4] = {fmaf(skip[0], xs[i][0], v.x), fmaf(skip[1], xs[i][1], v.y), fmaf(skip[2], xs[i][2], v.z), fmaf(skip[3], xs[i][3], v.w)};
        put(y + static_cast<long long>(t0 + t) * p.C, o, y_whole, left);
      }
      __syncwarp();                               // (read before the next tile writes them)
    }
  }
  if (ENDS) {
    keep(p.starts + (pad_row + static_cast<long long>(seg + 1) * padded) * NP + sl * NS);
#pragma unroll
    for (int j = 0; j < 4; ++j) {                 // over the tokens' lanes
#pragma unroll
      for (int o = L::PIECES; o < 32; o <<= 1) total[j] += __shfl_xor_sync(0xffffffffu, total[j], o);
      if (lt == 0) p.sums[(static_cast<long long>(row) * p.segments + seg) * padded + group * p.padded + c0 - group * per + lq + j] = total[j];
    }
  } else if (p.last != nullptr && seg == last_seg) {
#pragma unroll
    for (int j = 0; j < EIGHT; ++j)
#pragma unroll
      for (int k = 0; k < NS / 2; ++k) {
        const int c = mine + j, n = sl * NS + 2 * k;
        const float2 v = h[j][k].get();
        if (c < c_end && n < p.N) p.last[(r.at * p.C + c) * p.N + n] = v.x;
        if (c < c_end && n + 1 < p.N) p.last[(r.at * p.C + c) * p.N + n + 1] = v.y;
      }
  }
}

// One token per row, a decay per head.  A warp takes `ROWS` rows p of a head's [dim, N] state at a time, LN lanes a row.  grid (heads, parts, rows from `row0` on).
template <typename T, int LN, int NS>
__global__ void __launch_bounds__(THREADS)
head_token_kernel(const Args p, int row0) {
  constexpr int CG = 32 / LN;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sl = lane % LN, cg = lane / LN;
  const int head = blockIdx.x, row = row0 + blockIdx.z, dim = p.C / p.heads, pos = p.positions[row];
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

// steps [R, T, heads], rates [heads] (negative), places [3, R]: tokens that count, the store's row that a row begins with (-1: with zeros) and the one that it ends in (-1: none).
template <typename TD>
__global__ void __launch_bounds__(256)
head_steps_kernel(const Args p, float* __restrict__ steps, float* __restrict__ rates, int* __restrict__ places) {
  const int row = blockIdx.y;
  const Row r = row_of(p, row);
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) {
      places[row] = r.len;
      places[p.R + row] = r.len > 0 && r.held ? static_cast<int>(r.at) : -1;
      places[2 * p.R + row] = r.len > 0 && p.last != nullptr ? static_cast<int>(r.at) : -1;
    }
    if (row == 0)
      for (int h = threadIdx.x; h < p.heads; h += 256) rates[h] = rate_of(p, p.a[h]);
  }
  const long long all = static_cast<long long>(p.T) * p.heads;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const int t = static_cast<int>(i / p.heads), h = static_cast<int>(i - static_cast<long long>(t) * p.heads);
    float s = 0.f;
    if (t < r.len) {
      s = ld(static_cast<const TD*>(p.dt) + row * p.dt_row + t * p.dt_token + h) + (p.dt_bias == nullptr ? 0.f : p.dt_bias[h]);
      s = p.softplus ? softplus(s) : s;
    }
    steps[row * all + i] = s;
  }
}

template <typename T, typename TD, int LN, int NS>
int head_go(const Args& p, cudaStream_t stream) {
  using L = HeadLay<LN, NS>;
  const long long blocks = static_cast<long long>((p.C / p.groups + L::CB - 1) / L::CB) * p.groups;
  if (blocks * p.segments * p.R > 0x7fffffffLL) return -3;
  constexpr int smem = static_cast<int>(sizeof(HeadTile<LN, NS>));
  if (p.segments > 1) {
    const cudaError_t e = cudaFuncSetAttribute(head_scan_kernel<T, TD, LN, NS, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    head_scan_kernel<T, TD, LN, NS, true><<<static_cast<unsigned>(blocks * (p.segments - 1) * p.R), THREADS, smem, stream>>>(p);
  }
  const cudaError_t e = cudaFuncSetAttribute(head_scan_kernel<T, TD, LN, NS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  head_scan_kernel<T, TD, LN, NS, false><<<static_cast<unsigned>(blocks * p.segments * p.R), THREADS, smem, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, typename TD>
int heads_any(const Args& p, cudaStream_t stream) {
  if (p.N <= 16) return head_go<T, TD, 4, 4>(p, stream);
  if (p.N <= 32) return head_go<T, TD, 8, 4>(p, stream);
  if (p.N <= 64) return head_go<T, TD, 16, 4>(p, stream);
  if (p.N <= 128) return head_go<T, TD, 32, 4>(p, stream);
  if (p.N <= 256) return head_go<T, TD, 32, 8>(p, stream);
  return -3;
}

template <typename T>
int head_token_any(const Args& p, cudaStream_t stream) {
  for (long long from = 0; from < p.R; from += MOST_Z) {
    const int row0 = static_cast<int>(from);
    const dim3 grid(p.heads, 1, p.R - row0 < MOST_Z ? p.R - row0 : MOST_Z);
    if (p.N <= 16) head_token_kernel<T, 4, 4><<<grid, THREADS, 0, stream>>>(p, row0);
    else if (p.N <= 32) head_token_kernel<T, 8, 4><<<grid, THREADS, 0, stream>>>(p, row0);
    else if (p.N <= 64) head_token_kernel<T, 16, 4><<<grid, THREADS, 0, stream>>>(p, row0);
    else if (p.N <= 128) head_token_kernel<T, 32, 4><<<grid, THREADS, 0, stream>>>(p, row0);
    else if (p.N <= 256) head_token_kernel<T, 32, 8><<<grid, THREADS, 0, stream>>>(p, row0);
    else return -3;
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace selective
}  // namespace dewb

using namespace dewb::selective;

// A call's rows, or one token per row (with positions and a state).
extern "C" int dewb_head_scan(const dewb_selective_args* a, int fp32, int token, void* stream_ptr) {
  if (a == nullptr || a->heads < 1 || !args_ok(*a) || (fp32 && !a->dt_fp32)) return -3;
  if (token && (a->T != 1 || a->positions == nullptr || a->last == nullptr)) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (token) return fp32 ? head_token_any<float>(*a, stream) : head_token_any<bf16>(*a, stream);
  if (fp32) return heads_any<float, float>(*a, stream);
  return a->dt_fp32 ? heads_any<bf16, float>(*a, stream) : heads_any<bf16, bf16>(*a, stream);
}

extern "C" int dewb_head_steps(const dewb_selective_args* a, float* steps, float* rates, int* places, void* stream_ptr) {
  if (a == nullptr || a->heads < 1 || a->R > 65535 || !args_ok(*a) || steps == nullptr || rates == nullptr || places == nullptr) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  const long long all = static_cast<long long>(a->T) * a->heads, blocks = (all + 255) / 256;
  const dim3 grid(static_cast<unsigned>(blocks < 512 ? blocks : 512), a->R);
  if (a->dt_fp32) head_steps_kernel<float><<<grid, 256, 0, stream>>>(*a, steps, rates, places);
  else head_steps_kernel<bf16><<<grid, 256, 0, stream>>>(*a, steps, rates, places);
  return static_cast<int>(cudaGetLastError());
}
