// Low-rank adapters of many requests beside one projection:  y_t += s_i B_i (A_i x_t),  i the adapter of token t (below 0: none).
//
// Two kernels: shares of A_i x in fp32 (the width is split over CTAs), then B_i times their sum, added to y.  An adapter's tokens are worked on together, up to 16 (steps of
// generation) or 64 (prompts) of them as the rows of products on the tensor cores, so that its A and B come from memory once for all of them.
//
//   rows of a tile   up to 512 tokens: each CTA looks through the ids itself.  CTA t goes on if token t is the first, 17th, 33rd ... of its adapter.  More tokens: a kernel of one
//                    CTA counts them and writes the tiles down (8192 tokens: 5 us, where looking through them all in each CTA would take longer than the products).
//   operands         go from memory to registers as the products take them.  A lane of m16n8k16 holds two pairs of neighbouring elements of a row; which elements of the
//                    sum they are does not matter as long as both operands agree.  So a lane takes eight in a row (16 bytes), four lanes 32, and calls them two products' worth.
//   results          the columns of four n8 blocks are dealt so that a lane's eight are neighbours: y is read and written 16 bytes at a time.
//
// Bound by memory: A and B once an adapter in a step of generation; x and twice y for prompts.  The values between the two are rounded to bf16 for the second product, after their
// sum and scale in fp32: what an adapter adds is off by at most half a step of each rank's share.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../common/mma_bf16.cuh"
#include "../common/ptx.cuh"

namespace dewb {
namespace adapters {

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16(x); }

struct Args {
  const void *x, *a, *b;
  const float* scale;
  const int* ids;
  float* low;                    // [splits, tokens, rank]
  void* y;
  long long x_stride;
  int tokens, adapters, rank, width, out, splits;
  int* err;
};

// fp32, and sizes the tensor cores' kernels are not for: a CTA a (token, part of the width), a CTA a (token, 128 columns).
template <typename T>
__global__ void __launch_bounds__(128) shrink_kernel(const __grid_constant__ Args a) {
  const int t = blockIdx.x, split = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int id = a.ids[t];
  if (id < 0) return;
  if (id >= a.adapters) { if (threadIdx.x == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG)); return; }
  const int per = (a.width + a.splits - 1) / a.splits, from = split * per, to = min(a.width, from + per);
  const T* x = static_cast<const T*>(a.x) + t * a.x_stride;
  for (int r = warp; r < a.rank; r += 4) {
    const T* row = static_cast<const T*>(a.a) + (static_cast<long long>(id) * a.rank + r) * a.width;
    float s = 0.f;
    for (int k = from + lane; k < to; k += 32) s = fmaf(as_float(x[k]), as_float(row[k]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) a.low[(static_cast<long long>(split) * a.tokens + t) * a.rank + r] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(128) expand_kernel(const __grid_constant__ Args a) {
  extern __shared__ float low[];
  const int t = blockIdx.x, n = blockIdx.y * 128 + threadIdx.x;
  const int id = a.ids[t];
  if (id < 0 || id >= a.adapters) return;
  const float by = a.scale[id];
  for (int r = threadIdx.x; r < a.rank; r += 128) {
    float s = 0.f;
    for (int i = 0; i < a.splits; ++i) s += a.low[(static_cast<long long>(i) * a.tokens + t) * a.rank + r];
    low[r] = s * by;
  }
  __syncthreads();
  if (n >= a.out) return;
  const T* row = static_cast<const T*>(a.b) + (static_cast<long long>(id) * a.out + n) * a.rank;
  float s = 0.f;
  for (int r = 0; r < a.rank; ++r) s = fmaf(low[r], as_float(row[r]), s);
  T* y = static_cast<T*>(a.y) + static_cast<long long>(t) * a.out + n;
  put(y, as_float(*y) + s);
}

// ---------------------------------------------------------------------------------------------------------- bf16
using bf16 = __nv_bfloat16;
constexpr int SCANNED = 512;     // tokens whose ids each CTA looks through
constexpr int RB = 64;           // rank's values a CTA makes
constexpr int COLS = 256;        // y's columns a CTA adds to
constexpr int MOST_ADAPTERS = 4096;

struct Tile { int adapter, begin, count, pad; };

struct Mma {
  const bf16 *x, *a, *b;
  const float* scale;
  const int* ids;
  const int *order, *tiles_n;    // the tokens by adapter, and (behind) their tiles; null: look through the ids
  const Tile* tiles;
  float* low;                    // [splits, tokens, rank]
  bf16* y;
  long long x_stride;
  int tokens, adapters, rank, width, out, splits;
  bool wide_x, wide_b, wide_y;   // whether rows of x and a, of b, of y can be taken 16 bytes at a time
  int* err;
};

// Eight elements of a row, the first `n` of which exist.
__device__ __forceinline__ uint4 load8(const bf16* p, int n, bool wide) {
  if (n <= 0) return make_uint4(0, 0, 0, 0);
  if (wide) return __ldg(reinterpret_cast<const uint4*>(p));         // (n is 8: sizes are multiples of 8 then)
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = 2 * i < n ? __bfloat16_as_ushort(p[2 * i]) : 0u, hi = 2 * i + 1 < n ? __bfloat16_as_ushort(p[2 * i + 1]) : 0u;
    w[i] = lo | hi << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The CTA's tile: its adapter, and its tokens in rows[0, MT) (-1 behind the last).  False: nothing to do.  All threads.
template <int MT>
__device__ __forceinline__ bool find_tile(const Mma& m, int* rows, int& adapter) {
  __shared__ int found;
  const int lane = threadIdx.x & 31;
  if (m.order != nullptr) {
    if (static_cast<int>(blockIdx.x) >= *m.tiles_n) return false;
    const Tile t = m.tiles[blockIdx.x];
    for (int i = threadIdx.x; i < MT; i += blockDim.x) rows[i] = i < t.count ? m.order[t.begin + i] : -1;
    adapter = t.adapter;
    __syncthreads();
    return true;
  }
  if (threadIdx.x < 32) {
    const int t0 = blockIdx.x, mine = m.ids[t0];
    bool go = mine >= 0 && mine < m.adapters;
    if (mine >= m.adapters && lane == 0) atomicCAS(m.err, 0, static_cast<int>(ERR_BAD_ARG));
    int before = 0, n = 0;
    if (go) {
#pragma unroll 4
      for (int i0 = 0; i0 < m.tokens; i0 += 32) {
        const int i = i0 + lane;
        const unsigned same = __ballot_sync(0xffffffffu, i < m.tokens && m.ids[i] == mine);
        const unsigned earlier = t0 >= i0 + 32 ? 0xffffffffu : t0 <= i0 ? 0u : (1u << (t0 - i0)) - 1;
        before += __popc(same & earlier);
        const unsigned mine_on = same & ~earlier;
        const int at = n + __popc(mine_on & ((1u << lane) - 1));
        if ((mine_on >> lane & 1) && at < MT) rows[at] = i;
        n += __popc(mine_on);
      }
      go = before % MT == 0;
      for (int i = lane; i < MT; i += 32) if (i >= n) rows[i] = -1;
    }
    if (lane == 0) found = go ? mine : -1;
  }
  __syncthreads();
  adapter = found;
  return adapter >= 0;
}

// grid (tile, part of the width, 64 of the rank's values): the warps take every WARPS-th 32 of the width.
template <int M16, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) shrink_mma_kernel(const __grid_constant__ Mma m) {
  constexpr int MT = 16 * M16;
  __shared__ int rows[MT];
  extern __shared__ float sums[];                // [WARPS / 2][MT][RB]
  int adapter;
  griddep_launch();
  if (m.order != nullptr) griddep_wait();        // (the tiles are the kernel's before this)
  if (!find_tile<MT>(m, rows, adapter)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.y, r0 = blockIdx.z * RB, blocks = min(RB / 8, (m.rank - r0 + 7) / 8);
  const int per = ((m.width + m.splits - 1) / m.splits + 31) / 32 * 32, from = split * per, to = min(m.width, from + per);
  const bf16* xr[2 * M16];
#pragma unroll
  for (int i = 0; i < 2 * M16; ++i) {
    const int row = rows[i * 8 + g];
    xr[i] = row < 0 ? nullptr : m.x + row * m.x_stride;
  }
  const bf16* ar = m.a + (static_cast<long long>(adapter) * m.rank + r0 + g) * m.width;
  float acc[M16][RB / 8][4];
#pragma unroll
  for (int i = 0; i < M16; ++i)
#pragma unroll
    for (int n = 0; n < RB / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][n][e] = 0.f;
#pragma unroll 2
  for (int k0 = from + warp * 32; k0 < to; k0 += WARPS * 32) {
    const int k = k0 + c * 8, left = to - k;
    uint4 xv[2 * M16];
#pragma unroll
    for (int i = 0; i < 2 * M16; ++i) xv[i] = xr[i] == nullptr ? make_uint4(0, 0, 0, 0) : load8(xr[i] + k, left, m.wide_x);
#pragma unroll
    for (int n = 0; n < RB / 8; ++n) {
      if (n >= blocks) break;
      const uint4 av = r0 + n * 8 + g < m.rank ? load8(ar + static_cast<long long>(n) * 8 * m.width + k, left, m.wide_x) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < M16; ++i) {
        const uint32_t one[4] = {xv[2 * i].x, xv[2 * i + 1].x, xv[2 * i].y, xv[2 * i + 1].y}, two[4] = {xv[2 * i].z, xv[2 * i + 1].z, xv[2 * i].w, xv[2 * i + 1].w};
        mma16::mma(acc[i][n], one, av.x, av.y);
        mma16::mma(acc[i][n], two, av.z, av.w);
      }
    }
  }
  // the warps' sums, halving their number: the upper half writes, the lower half adds
#pragma unroll
  for (int half = WARPS / 2; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) {
      float* to_sum = sums + (warp - half) * MT * RB;
#pragma unroll
      for (int i = 0; i < M16; ++i)
#pragma unroll
        for (int n = 0; n < RB / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) to_sum[((i * (RB / 8) + n) * 4 + e) * 32 + lane] = acc[i][n][e];
    }
    __syncthreads();
    if (warp < half) {
      const float* add = sums + warp * MT * RB;
#pragma unroll
      for (int i = 0; i < M16; ++i)
#pragma unroll
        for (int n = 0; n < RB / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][n][e] += add[((i * (RB / 8) + n) * 4 + e) * 32 + lane];
    }
    __syncthreads();
  }
  if (warp != 0) return;
#pragma unroll
  for (int i = 0; i < M16; ++i)
#pragma unroll
    for (int n = 0; n < RB / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = rows[i * 16 + g + (e >> 1) * 8], r = r0 + n * 8 + 2 * c + (e & 1);
        if (row >= 0 && r < m.rank) m.low[(static_cast<long long>(split) * m.tokens + row) * m.rank + r] = acc[i][n][e];
      }
}

// grid (tile, COLS columns of y): a warp takes every fourth 32 columns.
template <int M16>
__global__ void __launch_bounds__(128) expand_mma_kernel(const __grid_constant__ Mma m) {
  constexpr int MT = 16 * M16;
  __shared__ int rows[MT];
  extern __shared__ uint4 low16[];               // [MT][rank in whole 32s] bf16, + 8 a row (bank spacing)
  bf16* low = reinterpret_cast<bf16*>(low16);
  int adapter;
  if (m.order != nullptr) griddep_wait();
  if (!find_tile<MT>(m, rows, adapter)) return;
  if (m.order == nullptr) griddep_wait();        // (the ids are older than the kernel before this, which makes the rank's values)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int wide = (m.rank + 31) / 32 * 32, pitch = wide + 8;
  const float by = m.scale[adapter];
  for (int i = threadIdx.x; i < MT * wide; i += 128) {
    const int t = i / wide, r = i - t * wide, row = rows[t];
    float s = 0.f;
    if (row >= 0 && r < m.rank)
      for (int k = 0; k < m.splits; ++k) s += m.low[(static_cast<long long>(k) * m.tokens + row) * m.rank + r];
    low[t * pitch + r] = __float2bfloat16(s * by);
  }
  __syncthreads();
  int row[2 * M16];
#pragma unroll
  for (int i = 0; i < 2 * M16; ++i) row[i] = rows[i * 8 + g];
  const bf16* b = m.b + static_cast<long long>(adapter) * m.out * m.rank;
#pragma unroll 1
  for (int n0 = blockIdx.y * COLS + warp * 32; n0 < min(m.out, (static_cast<int>(blockIdx.y) + 1) * COLS); n0 += 128) {
    float acc[M16][4][4];
#pragma unroll
    for (int i = 0; i < M16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
    // y is on its way meanwhile: this lane's eight columns of each row
    const int col = n0 + c * 8, left = m.out - col;
    uint4 old[2 * M16];
#pragma unroll
    for (int i = 0; i < 2 * M16; ++i) {
      const bf16* p = m.y + static_cast<long long>(max(row[i], 0)) * m.out + col;
      old[i] = row[i] < 0 ? make_uint4(0, 0, 0, 0) : m.wide_y && left >= 8 ? *reinterpret_cast<const uint4*>(p) : load8(p, left, false);
    }
#pragma unroll 2
    for (int k0 = 0; k0 < m.rank; k0 += 32) {
      const int k = k0 + c * 8;
      uint4 bv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + (g >> 1) * 8 + j * 2 + (g & 1);           // block j's column g
        bv[j] = n < m.out ? load8(b + static_cast<long long>(n) * m.rank + k, m.rank - k, m.wide_b) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < M16; ++i) {
        const uint4 lo = *reinterpret_cast<const uint4*>(low + (i * 16 + g) * pitch + k), hi = *reinterpret_cast<const uint4*>(low + (i * 16 + 8 + g) * pitch + k);
        const uint32_t one[4] = {lo.x, hi.x, lo.y, hi.y}, two[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma16::mma(acc[i][j], one, bv[j].x, bv[j].y);
          mma16::mma(acc[i][j], two, bv[j].z, bv[j].w);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * M16; ++i) {
      if (row[i] < 0 || left <= 0) continue;
      const uint32_t was[4] = {old[i].x, old[i].y, old[i].z, old[i].w};
      uint32_t now[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) now[j] = pack_bf16(bf16_lo(was[j]) + acc[i / 2][j][2 * (i & 1)], bf16_hi(was[j]) + acc[i / 2][j][2 * (i & 1) + 1]);
      bf16* p = m.y + static_cast<long long>(row[i]) * m.out + col;
      if (m.wide_y && left >= 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(now[0], now[1], now[2], now[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) p[e] = __ushort_as_bfloat16(static_cast<unsigned short>(now[e >> 1] >> (e & 1) * 16));
      }
    }
  }
}

// One CTA: the tokens by adapter, and tiles of up to `tall` of them.  (Where a token stands among its adapter's does not change its result.)
__global__ void __launch_bounds__(1024) group_tokens_kernel(const int* __restrict__ ids, int tokens, int adapters, int tall, int* __restrict__ order, int* __restrict__ tiles_n,
                                                            Tile* __restrict__ tiles, int* __restrict__ err) {
  extern __shared__ int at[];                    // [adapters]: counts, then where the next token goes
  __shared__ int totals[32][2], carry[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_launch();
  for (int i = tid; i < adapters; i += 1024) at[i] = 0;
  if (tid == 0) carry[0] = carry[1] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < tokens; i0 += 1024) {
    const int i = i0 + tid, id = i < tokens ? ids[i] : -1;
    const bool there = id >= 0 && id < adapters;
    if (id >= adapters) atomicCAS(err, 0, static_cast<int>(ERR_BAD_ARG));
    const unsigned same = __match_any_sync(0xffffffffu, there ? id : -1);
    if (there && lane == __ffs(same) - 1) atomicAdd(&at[id], __popc(same));
  }
  __syncthreads();
  for (int i0 = 0; i0 < adapters; i0 += 1024) {
    const int i = i0 + tid, n = i < adapters ? at[i] : 0, t = (n + tall - 1) / tall;
    int sn = n, st = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int vn = __shfl_up_sync(0xffffffffu, sn, o), vt = __shfl_up_sync(0xffffffffu, st, o);
      if (lane >= o) { sn += vn; st += vt; }
    }
    if (lane == 31) { totals[warp][0] = sn; totals[warp][1] = st; }
    __syncthreads();
    int bn = carry[0], bt = carry[1];
    for (int w = 0; w < warp; ++w) { bn += totals[w][0]; bt += totals[w][1]; }
    __syncthreads();
    if (tid == 1023) { carry[0] = bn + sn; carry[1] = bt + st; }
    if (i < adapters) {
      at[i] = bn + sn - n;
      for (int j = 0; j < t; ++j) tiles[bt + st - t + j] = Tile{i, bn + sn - n + j * tall, min(tall, n - j * tall), 0};
    }
    __syncthreads();
  }
  if (tid == 0) *tiles_n = carry[1];
  for (int i0 = 0; i0 < tokens; i0 += 1024) {
    const int i = i0 + tid, id = i < tokens ? ids[i] : -1;
    const bool there = id >= 0 && id < adapters;
    const unsigned same = __match_any_sync(0xffffffffu, there ? id : -1);
    int base = 0;
    if (there && lane == __ffs(same) - 1) base = atomicAdd(&at[id], __popc(same));
    base = __shfl_sync(0xffffffffu, base, __ffs(same) - 1);
    if (there) order[base + __popc(same & ((1u << lane) - 1))] = i;
  }
}

template <typename K>
int launch_early(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, const Mma& m) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, m));
}

template <int M16, int WARPS>
int launch_mma(const Mma& m, int tiles, cudaStream_t stream) {
  constexpr int MT = 16 * M16;
  constexpr int sums = WARPS / 2 * MT * RB * 4;
  const int low = MT * ((m.rank + 31) / 32 * 32 + 8) * 2;
  cudaError_t e;
  if ((e = cudaFuncSetAttribute(shrink_mma_kernel<M16, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, sums)) != cudaSuccess) return static_cast<int>(e);
  if ((e = cudaFuncSetAttribute(expand_mma_kernel<M16>, cudaFuncAttributeMaxDynamicSharedMemorySize, low)) != cudaSuccess) return static_cast<int>(e);
  const dim3 first(tiles, m.splits, (m.rank + RB - 1) / RB), second(tiles, (m.out + COLS - 1) / COLS);
  if (m.order != nullptr) {
    if (int rc = launch_early(shrink_mma_kernel<M16, WARPS>, first, WARPS * 32, sums, stream, m)) return rc;
  } else {
    shrink_mma_kernel<M16, WARPS><<<first, WARPS * 32, sums, stream>>>(m);
    if ((e = cudaGetLastError()) != cudaSuccess) return static_cast<int>(e);
  }
  return launch_early(expand_mma_kernel<M16>, second, 128, low, stream, m);
}

}  // namespace adapters
}  // namespace dewb

// y [tokens, out] += scale[id] (x [tokens, width; x_stride] a[id]^T) b[id]^T with a [adapters, rank, width], b [adapters, out, rank], ids int32 [tokens]; low: scratch, splits x
// tokens x rank floats.  An id past the last adapter is reported by the status word and adds nothing.
extern "C" int dewb_add_adapters(const void* x, long long x_stride, const void* a, const void* b, const float* scale, const int* ids, float* low, void* y, int tokens, int adapters,
                                 int rank, int width, int out, int splits, int fp32, int* err, void* stream_ptr) {
  using namespace dewb::adapters;
  if (tokens <= 0 || out <= 0) return 0;
  if (adapters <= 0 || rank <= 0 || rank > 4096 || width <= 0 || splits < 1 || splits > 65535 || out > 65535 * 128) return -3;
  const Args args{x, a, b, scale, ids, low, y, x_stride, tokens, adapters, rank, width, out, splits, err};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  const dim3 first(tokens, splits), second(tokens, (out + 127) / 128);
  if (fp32) {
    shrink_kernel<float><<<first, 128, 0, stream>>>(args);
    expand_kernel<float><<<second, 128, rank * 4, stream>>>(args);
  } else {
    shrink_kernel<__nv_bfloat16><<<first, 128, 0, stream>>>(args);
    expand_kernel<__nv_bfloat16><<<second, 128, rank * 4, stream>>>(args);
  }
  return static_cast<int>(cudaGetLastError());
}

// The same on the tensor cores: bf16, rank up to 512, up to 4096 adapters, any widths.  Up to 512 tokens: two launches; more: three, and order (tokens integers), then tiles (one
// integer on a 16-byte boundary, 12 bytes unused, then 16 bytes for each of tokens / 64 + min(adapters, tokens) + 1).
extern "C" int dewb_add_adapters_mma(const void* x, long long x_stride, const void* a, const void* b, const float* scale, const int* ids, int* order, void* tiles, float* low, void* y,
                                     int tokens, int adapters, int rank, int width, int out, int splits, int* err, void* stream_ptr) {
  using namespace dewb::adapters;
  if (tokens <= 0 || out <= 0) return 0;
  if (adapters <= 0 || adapters > MOST_ADAPTERS || rank <= 0 || rank > 512 || width <= 0 || splits < 1 || splits > 65535 || out > 65535 * COLS || (tokens > SCANNED && order == nullptr)) return -3;
  auto whole = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  int* n = static_cast<int*>(tiles);
  Mma m{static_cast<const bf16*>(x), static_cast<const bf16*>(a), static_cast<const bf16*>(b), scale, ids, nullptr, n, reinterpret_cast<const Tile*>(n + 4), low, static_cast<bf16*>(y),
        x_stride, tokens, adapters, rank, width, out, splits,
        width % 8 == 0 && x_stride % 8 == 0 && whole(x) && whole(a), rank % 8 == 0 && whole(b), out % 8 == 0 && whole(y), err};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (tokens <= SCANNED) return launch_mma<1, 4>(m, tokens, stream);
  group_tokens_kernel<<<1, 1024, adapters * 4, stream>>>(ids, tokens, adapters, 64, order, n, reinterpret_cast<Tile*>(n + 4), err);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  m.order = order;
  return launch_mma<4, 4>(m, tokens / 64 + (adapters < tokens ? adapters : tokens) + 1, stream);
}
