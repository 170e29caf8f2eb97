// Low-rank adapters of many requests beside one projection:  y_t += s_i B_i (A_i x_t),  i the adapter of token t (below 0: none).
//
// An adapter's tokens are worked on together, so that its A and B come from memory once for all of them.
//
// STEPS OF GENERATION, up to 512 tokens: one kernel.  A cluster of eight CTAs takes up to 16 tokens of an adapter: each makes the products with A over its part
// of the width, they add them up through one another's shared memory, and each multiplies with its part of B's rows.  Cluster t takes the t-th such tile in the order of their first
// tokens, which it finds out by looking through the ids.  Operands go from memory to registers as the warp-level products take them (16 rows are too few for the others): a lane of m16n8k16 holds
// two pairs of neighbouring elements of a row, and which elements of the sum they are does not matter as long as both operands agree.  So a lane takes eight in a row (16 bytes),
// four lanes 32, and calls them two products' worth.  B and y are on their way while A's products are added up.  The columns of four n8 blocks are dealt so that a lane's eight
// are neighbours: y is read and written 16 bytes at a time.  Bound by latency (ids, operands, one cluster barrier, results) and, with many adapters, by reading A and B.
//
// PROMPTS: three kernels.  One CTA puts the tokens in the order of their adapters and writes down tiles of up to 128.  Then 128 x 64 x width products on the tensor cores; tokens
// come by TMA, as a block where a tile's are neighbours, else four at a time by their numbers.  A tile's width is shared out over a cluster, whose CTAs add up through one another's
// shared memory and write the rank's values, times the scale, in bf16 and in the tiles' order: the second product's operand as it stands.  Then pieces of 128 columns of all tiles,
// shared evenly by as many CTAs as fit the SMs: times B on the tensor cores, added to y, whose piece has come to shared memory meanwhile and leaves from there.
// Bound by x and twice y, and by the latencies of three kernels.
//
// The values between the two products are rounded to bf16 after their sum and scale in fp32: what an adapter adds is off by at most half a step of each rank's share.
#include <algorithm>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../common/mma_bf16.cuh"
#include "../common/ptx.cuh"
#include "../common/tmap.h"

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
constexpr int SCANNED = 512;     // tokens whose ids each CTA looks through (just past it, by three kernels: 15 instead of 12 us for one adapter, 35 instead of 17 for 48)
constexpr int MOST_ADAPTERS = 3500,            // (16 counts each fit a CTA's shared memory)
              MOST_RANK = 512;
constexpr uint32_t FULL = 0xffffffffu;

struct Tile { int adapter, begin, count, pad; };

struct Mma {
  const bf16 *x, *a, *b;
  const float* scale;
  const int* ids;
  const int *order, *tiles_n;    // prompts: the tokens by adapter, and their tiles
  const Tile* tiles;
  bf16* low;                     // prompts: [tokens, wide], an adapter's tokens together: the rank's values times the scale, zeros behind them
  bf16* y;
  long long x_stride;
  int tokens, adapters, rank, width, out, splits, wide;
  bool wide_x, wide_b, wide_y;   // whether rows of x and a, of b, of y can be taken 16 bytes at a time
  int* err;
};

// Eight elements of a row, the first `n` of which exist.
__device__ __forceinline__ uint4 load8(const bf16* p, int n, bool wide) {
  if (n <= 0) return make_uint4(0, 0, 0, 0);
  if (wide && n >= 8) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = 2 * i < n ? __bfloat16_as_ushort(p[2 * i]) : 0u, hi = 2 * i + 1 < n ? __bfloat16_as_ushort(p[2 * i + 1]) : 0u;
    w[i] = lo | hi << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(bf16* p, const uint32_t (&w)[4], int n, bool wide) {
  if (wide && n >= 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = __ushort_as_bfloat16(static_cast<unsigned short>(w[e >> 1] >> (e & 1) * 16));
  }
}

// ---------------------------------------------------------------------------------------------------------- steps of generation
constexpr int CLUSTER = 8, STEP_WARPS = 4, STEP_THREADS = STEP_WARPS * 32, MT = 16;
constexpr int RB = 64;           // rank's values at a time (steps: 32 where there are no more)

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ void st_cluster4(uint32_t addr, const uint32_t* v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// grid (CLUSTER, as many tiles as there can be); four CTAs an SM, with a few values of the ids' count spilled (three, of 156 registers: 512 tokens of 48 adapters 26 us instead of
// 17, one token 8.8 instead of 9.2).  Clusters of four instead of eight: 128 tokens 33 us instead of 26.7 with the projection.
template <int CLUSTER, int RB>
__global__ void __launch_bounds__(STEP_THREADS, 4) adapters_step_kernel(const __grid_constant__ Mma m) {
  extern __shared__ __align__(16) float sums[];  // [wide / 8][16][8]: this CTA's share of the rank's values; then as bf16 [16][wide + 8]; in front, the warps' shares
  __shared__ unsigned first[SCANNED / 32];
  __shared__ int adapter_at[2];                  // the tile's adapter, and how many of its tokens come before
  __shared__ int rows[MT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int part = cluster_ctarank(), tile = blockIdx.y;
  griddep_wait();
  // which tokens begin a tile: those with no token of their adapter before them, or 16, 32, ... of them.  A warp counts a quarter of the tokens by adapter
  constexpr int HELD = SCANNED / STEP_THREADS;
  unsigned short* counts = reinterpret_cast<unsigned short*>(sums);                  // [adapters][STEP_WARPS], those of adapters that occur
  const int quarter = (m.tokens + STEP_THREADS - 1) / STEP_THREADS * 32, from_token = warp * quarter;
  int id[HELD], before[HELD];
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    const int i = from_token + e * 32 + lane;
    id[e] = e * 32 < quarter && i < m.tokens ? m.ids[i] : -1;
    if (id[e] >= m.adapters) {
      if (tile == 0 && part == 0) atomicCAS(m.err, 0, static_cast<int>(ERR_BAD_ARG));
      id[e] = -1;
    }
    if (id[e] >= 0) *reinterpret_cast<uint2*>(counts + STEP_WARPS * id[e]) = make_uint2(0, 0);
  }
  if (tid < MT) rows[tid] = -1;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    if (e * 32 >= quarter) break;
    const unsigned same = __match_any_sync(FULL, id[e]);
    const int mine_at = STEP_WARPS * id[e] + warp, so_far = id[e] >= 0 ? counts[mine_at] : 0;
    before[e] = so_far + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (id[e] >= 0 && lane == __ffs(same) - 1) counts[mine_at] = static_cast<unsigned short>(so_far + __popc(same));
    __syncwarp();
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    if (e * 32 >= quarter) break;
    if (id[e] >= 0)
#pragma unroll
      for (int w = 0; w < STEP_WARPS - 1; ++w) before[e] += w < warp ? counts[STEP_WARPS * id[e] + w] : 0;
    const unsigned begin = __ballot_sync(FULL, id[e] >= 0 && before[e] % MT == 0);
    if (lane == 0) first[from_token / 32 + e] = begin;
  }
  __syncthreads();
  // this cluster's: the tile that begins with the `tile`-th of them
  const int blocks_of_32 = STEP_WARPS * (quarter / 32);
  int w32 = 0, left_of = tile;
#pragma unroll 1
  while (w32 < blocks_of_32 && left_of >= __popc(first[w32])) left_of -= __popc(first[w32++]);
  if (w32 >= blocks_of_32) return;               // (all CTAs of a cluster, or none)
  unsigned begin = first[w32];
#pragma unroll 1
  for (; left_of > 0; --left_of) begin &= begin - 1;
#pragma unroll
  for (int e = 0; e < HELD; ++e)
    if (e * 32 < quarter && from_token + e * 32 + lane == w32 * 32 + __ffs(begin) - 1) { adapter_at[0] = id[e]; adapter_at[1] = before[e]; }
  __syncthreads();
  const int mine = adapter_at[0];
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    const int n = before[e] - adapter_at[1];
    if (e * 32 < quarter && id[e] == mine && n >= 0 && n < MT) rows[n] = from_token + e * 32 + lane;
  }
  __syncthreads();
  const int row0 = rows[g], row1 = rows[g + 8];
  const int wide = (m.rank + 31) / 32 * 32;
  float* share = sums + STEP_WARPS * MT * RB;    // [MT][wide]
  // ---- x A^T over this CTA's part of the width
  {
    const int per = ((m.width + CLUSTER - 1) / CLUSTER + 31) / 32 * 32, from = part * per, to = min(m.width, from + per);
    const bf16 *x0 = m.x + max(row0, 0) * m.x_stride, *x1 = m.x + max(row1, 0) * m.x_stride;
#pragma unroll 1
    for (int r0 = 0; r0 < wide; r0 += RB) {
      const bf16* ar = m.a + (static_cast<long long>(mine) * m.rank + r0 + g) * m.width;
      const int blocks = min(RB / 8, (m.rank - r0 + 7) / 8);
      float acc[RB / 8][4];
#pragma unroll
      for (int n = 0; n < RB / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
      // (as many operands on their way as there are registers for: 128 columns of 32 ranks, 64 of 64)
      constexpr int DEEP = 128 / RB;
#pragma unroll 1
      for (int k0 = from + warp * 32; k0 < to; k0 += STEP_WARPS * 32 * DEEP) {
        uint4 lo[DEEP], hi[DEEP], av[DEEP][RB / 8];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
          const int k = k0 + d * STEP_WARPS * 32 + c * 8, left = to - k;
          lo[d] = row0 < 0 ? make_uint4(0, 0, 0, 0) : load8(x0 + k, left, m.wide_x);
          hi[d] = row1 < 0 ? make_uint4(0, 0, 0, 0) : load8(x1 + k, left, m.wide_x);
#pragma unroll
          for (int n = 0; n < RB / 8; ++n)
            av[d][n] = n < blocks && r0 + n * 8 + g < m.rank ? load8(ar + static_cast<long long>(n) * 8 * m.width + k, left, m.wide_x) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
          const uint32_t one[4] = {lo[d].x, hi[d].x, lo[d].y, hi[d].y}, two[4] = {lo[d].z, hi[d].z, lo[d].w, hi[d].w};
#pragma unroll
          for (int n = 0; n < RB / 8; ++n) {
            if (n >= blocks) break;
            mma16::mma(acc[n], one, av[d][n].x, av[d][n].y);
            mma16::mma(acc[n], two, av[d][n].z, av[d][n].w);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < RB / 8; ++n)
        if (n < blocks) *reinterpret_cast<float4*>(sums + ((warp * (RB / 8) + n) * 32 + lane) * 4) = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
      __syncthreads();
      // the warps' shares: value e of lane l in block n is row l / 4 + 8 (e / 2), column 8 n + 2 (l % 4) + e % 2
#pragma unroll 1
      for (int i = tid; i < blocks * 32; i += STEP_THREADS) {
        const int n = i >> 5, l = i & 31;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < STEP_WARPS; ++w) {
          const float4 u = *reinterpret_cast<const float4*>(sums + ((w * (RB / 8) + n) * 32 + l) * 4);
          v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
        }
        float* to_share = share + (l >> 2) * wide + r0 + n * 8 + 2 * (l & 3);
        to_share[0] = v.x; to_share[1] = v.y; to_share[8 * wide] = v.z; to_share[8 * wide + 1] = v.w;
      }
      __syncthreads();
    }
  }
  cluster_arrive();
  // ---- meanwhile, this warp's first columns of B and y are fetched: PIECES of 32 of the rank for 32 columns, in the order of their use
  constexpr int PIECES = 3;
  const int per = ((m.out + CLUSTER - 1) / CLUSTER + 31) / 32 * 32, n_end = min(m.out, (part + 1) * per), n_first = part * per + warp * 32;
  const int kblocks = wide / 32, pieces = n_first < n_end ? (n_end - n_first + STEP_THREADS - 1) / STEP_THREADS * kblocks : 0;
  const bf16* b = m.b + static_cast<long long>(mine) * m.out * m.rank;
  uint4 bv[PIECES][4], old[PIECES][2];
  auto fetch = [&](int i, uint4 (&bp)[4], uint4 (&yp)[2]) {
    if (i >= pieces) return;
    const int nt = i / kblocks, kb = i - nt * kblocks, n0 = n_first + nt * STEP_THREADS, k = kb * 32 + c * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + (g >> 1) * 8 + j * 2 + (g & 1);             // block j's column g
      bp[j] = n < n_end ? load8(b + static_cast<long long>(n) * m.rank + k, m.rank - k, m.wide_b) : make_uint4(0, 0, 0, 0);
    }
    if (kb != 0) return;
    const int col = n0 + c * 8, left = m.out - col;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = h == 0 ? row0 : row1;
      const bf16* p = m.y + static_cast<long long>(max(row, 0)) * m.out + col;
      yp[h] = row < 0 ? make_uint4(0, 0, 0, 0) : m.wide_y && left >= 8 ? *reinterpret_cast<const uint4*>(p) : load8(p, left, false);
    }
  };
#pragma unroll
  for (int i = 0; i < PIECES; ++i) fetch(i, bv[i], old[i]);
  const float by = m.scale[mine];
  cluster_wait();
  // ---- the CTAs' shares, their sum times the scale to bf16 (behind the shares)
  const int pitch = wide + 8;
  bf16* low = reinterpret_cast<bf16*>(share + MT * wide);
  {
    const uint32_t at = smem_u32(share);
#pragma unroll 1
    for (int i = tid; i < MT * wide; i += STEP_THREADS) {
      const int t = i / wide, r = i - t * wide;
      float v = 0.f;
#pragma unroll
      for (int p = 0; p < CLUSTER; ++p) v += ld_cluster(map_to_cta(at + i * 4, p));
      low[t * pitch + r] = __float2bfloat16(r < m.rank ? v * by : 0.f);
    }
  }
  cluster_arrive();                              // (its share is read by others until here)
  __syncthreads();
  float acc[4][4];
#pragma unroll 1
  for (int i0 = 0; i0 < pieces; i0 += PIECES) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int i = i0 + p;
      if (i >= pieces) break;
      const int nt = i / kblocks, kb = i - nt * kblocks;
      if (kb == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] = e & 1 ? bf16_hi(word(old[p][e >> 1], j)) : bf16_lo(word(old[p][e >> 1], j));
      }
      const uint4 lo = *reinterpret_cast<const uint4*>(low + g * pitch + kb * 32 + c * 8), hi = *reinterpret_cast<const uint4*>(low + (8 + g) * pitch + kb * 32 + c * 8);
      const uint32_t one[4] = {lo.x, hi.x, lo.y, hi.y}, two[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mma16::mma(acc[j], one, bv[p][j].x, bv[p][j].y);
        mma16::mma(acc[j], two, bv[p][j].z, bv[p][j].w);
      }
      fetch(i + PIECES, bv[p], old[p]);
      if (kb != kblocks - 1) continue;
      const int col = n_first + nt * STEP_THREADS + c * 8, left = m.out - col;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = h == 0 ? row0 : row1;
        uint32_t now[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) now[j] = pack_bf16(acc[j][2 * h], acc[j][2 * h + 1]);
        if (row >= 0 && left > 0) store8(m.y + static_cast<long long>(row) * m.out + col, now, left, m.wide_y);
      }
    }
  }
  cluster_wait();                                // (no CTA's memory goes while another reads it)
}

// ---------------------------------------------------------------------------------------------------------- prompts
constexpr int TALL = 128;        // tokens a tile
constexpr int KB = 64;           // columns of an operand's slot (128 bytes)
constexpr int MAKE_STAGES = 3, AHEAD = 2;
constexpr int LOW_PITCH = RB + 4;                // floats of a token's row in shared memory
constexpr int X_SLOT = TALL * KB * 2, A_SLOT = RB * KB * 2, MAKE_SMEM = MAKE_STAGES * (X_SLOT + A_SLOT);
static_assert(TALL * LOW_PITCH * 4 <= MAKE_SMEM, "the values lie where the operands were");
constexpr int ADD_N = 128, ADD_STAGES = 2, B_SLOT = ADD_N * KB * 2, Y_SLOT = TALL * ADD_N * 2;

// Four rows of 64 columns (128-byte swizzle), each by its number; rows and columns outside the matrix are zeros.
__device__ __forceinline__ void tma_gather4(void* to, const CUtensorMap* map, uint64_t* bar, int col, int r0, int r1, int r2, int r3) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(to)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar))
               : "memory");
}

// 16 bytes (8 elements, the first n of which exist) to shared memory, as zeros where there are none
__device__ __forceinline__ void copy8(uint32_t to, const bf16* p, int n, bool wide) {
  if (wide) {
    const int bytes = max(0, min(n, 8)) * 2;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(p), "r"(bytes) : "memory");
  } else {
    const uint4 v = load8(p, n, false);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
  }
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

struct alignas(16) Bars {
  uint64_t full[4], empty[4], acc_full[2], acc_empty[2], y_full[2], y_done[2], y_free[2], low_full;
  uint32_t tmem;
  int abort_flag, poisoned;
  alignas(16) int rows[TALL];      // (read four at a time)
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code, int lane) {
  if (mbar_wait_warp(bar, parity, abort_flag)) return true;
  if (lane == 0) atomicCAS(err, 0, code);
  return false;
}

// After a wait that ran out: what is on its way to shared memory gets 20 ms to land before that memory is another's.
__device__ __noinline__ void let_copies_land(volatile int* abort_flag) {
  if (*abort_flag == 0) return;
  const unsigned long long from = globaltimer_ns();
  while (globaltimer_ns() - from < 20000000ull) __nanosleep(1000);
}

// whether a tile's tokens are neighbours (all threads)
__device__ __forceinline__ bool neighbours(const int* rows, int count, int tid) { return __syncthreads_and(tid >= count || rows[tid] == rows[0] + tid) != 0; }

// a lane's four rows of a tile (the first one's where there are no more: what comes of those goes nowhere)
__device__ __forceinline__ int4 four_rows(const int* rows, int lane) {
  const int4 v = *reinterpret_cast<const int4*>(rows + 4 * lane);
  return make_int4(v.x < 0 ? rows[0] : v.x, v.y < 0 ? rows[0] : v.y, v.z < 0 ? rows[0] : v.z, v.w < 0 ? rows[0] : v.w);
}

// grid (tile, part of the width, 64 of the rank's values); warps 0..3 write results, warp 4 issues products, warp 5 fetches tokens (a lane four of them) and A.  Without TMA, for
// rows that do not begin at 16 bytes, warps 0..3 fetch: each step then waits for all of a thread's copies at the fence between them and the products.
template <bool TMA>
__global__ void __launch_bounds__(192) make_low_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tx_block, const __grid_constant__ CUtensorMap ta, const __grid_constant__ Mma m) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Bars bars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < MAKE_STAGES; ++i) { mbar_init(&bars.full[i], TMA ? 1 : 4); mbar_init(&bars.empty[i], 1); }
    mbar_init(&bars.acc_full[0], 1);
    bars.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  griddep_wait();                                // (the tiles are the kernel's before this)
  griddep_launch();                              // (and of use to the next one from here on)
  const int tiles = *m.tiles_n;
  const int4 what = *reinterpret_cast<const int4*>(m.tiles + blockIdx.x);          // (there are as many as CTAs, written or not)
  __syncthreads();
  if (static_cast<int>(blockIdx.x) >= tiles) return;             // (all CTAs of a cluster, or none)
  if ((smem_u32(smem) & 1023u) != 0) {
    if (tid == 0) atomicCAS(m.err, 0, static_cast<int>(ERR_BAD_ARG));
    return;
  }
  if (TMA && warp == 5 && lane == 0) { tma_prefetch_desc(&tx); tma_prefetch_desc(&tx_block); tma_prefetch_desc(&ta); }
  const Tile tile{what.x, what.y, what.z, 0};
  const float by = m.scale[tile.adapter];
  if (tid < TALL) bars.rows[tid] = tid < tile.count ? m.order[tile.begin + tid] : -1;
  if (warp == 4) { tmem_alloc(&bars.tmem, 64); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const bool block = TMA && neighbours(bars.rows, tile.count, tid);
  const uint32_t tmem = bars.tmem;
  volatile int* abort_flag = &bars.abort_flag;
  const int split = blockIdx.y, r0 = blockIdx.z * RB, ranks = min(RB, m.rank - r0), n16 = (ranks + 15) / 16;
  const int per = ((m.width + m.splits - 1) / m.splits + KB - 1) / KB * KB, from = split * per, to = min(m.width, from + per);
  const int steps = max(0, (to - from + KB - 1) / KB), share = TALL / m.splits;
  uint8_t *sx = smem, *sa = smem + MAKE_STAGES * X_SLOT;
  if (TMA && warp == 5) {
    const int4 four = four_rows(bars.rows, lane);
    const bool there = 4 * lane < tile.count;
    const uint32_t bytes = (block ? X_SLOT : (tile.count + 3) / 4 * 512) + A_SLOT;
    bool ok = true;
#pragma unroll 1
    for (int s = 0; s < steps && ok; ++s) {
      const int slot = s % MAKE_STAGES;
      ok = wait(&bars.empty[slot], ((s / MAKE_STAGES) & 1) ^ 1, abort_flag, m.err, ERR_WAIT_EMPTY, lane);
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(&bars.full[slot], bytes);
        tma_load_2d(sa + slot * A_SLOT, &ta, &bars.full[slot], from + s * KB, tile.adapter * m.rank + r0);
        if (block) tma_load_2d(sx + slot * X_SLOT, &tx_block, &bars.full[slot], from + s * KB, bars.rows[0]);
      }
      __syncwarp();
      if (there && !block) tma_gather4(sx + slot * X_SLOT + lane * 512, &tx, &bars.full[slot], from + s * KB, four.x, four.y, four.z, four.w);
      __syncwarp();
    }
  } else if (warp < 4) {
   if constexpr (!TMA) {
    const int c = tid & 7;
    const bf16* xr[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int row = bars.rows[(tid >> 3) + 16 * e];
      xr[e] = row < 0 ? nullptr : m.x + row * m.x_stride + c * 8;
    }
    const bf16* ar = m.a + (static_cast<long long>(tile.adapter) * m.rank + r0 + (tid >> 3)) * m.width + c * 8;
    bool ok = true;
#pragma unroll 1
    for (int s = 0; s < steps + AHEAD; ++s) {
      if (s < steps) {
        const int slot = s % MAKE_STAGES;
        ok = ok && wait(&bars.empty[slot], ((s / MAKE_STAGES) & 1) ^ 1, abort_flag, m.err, ERR_WAIT_EMPTY, lane);
        const int k = from + s * KB, left = to - k - c * 8;
        const uint32_t xs = smem_u32(sx + slot * X_SLOT) + (tid >> 3) * 128 + ((c ^ ((tid >> 3) & 7)) << 4);
        const uint32_t as = smem_u32(sa + slot * A_SLOT) + (tid >> 3) * 128 + ((c ^ ((tid >> 3) & 7)) << 4);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (xr[e] != nullptr) copy8(xs + e * 2048, left > 0 ? xr[e] + k : xr[e], left, m.wide_x);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((tid >> 3) + 16 * e < ranks) copy8(as + e * 2048, left > 0 ? ar + static_cast<long long>(e) * 16 * m.width + k : m.a, left, m.wide_x);
      }
      copies_end_group();
      if (s >= AHEAD) {
        copies_wait<AHEAD>();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.full[(s - AHEAD) % MAKE_STAGES]);
      }
    }
   }
    if (steps > 0) wait(&bars.acc_full[0], 0, abort_flag, m.err, ERR_WAIT_TMEM_FULL, lane);
    tc_fence_after();
    let_copies_land(abort_flag);
    // this part's values to the CTA that adds up this thread's token, where its operands were (in room of their own, 106 KB a CTA and two instead of three an SM: 29 us instead of 24)
    cluster_arrive();
    cluster_wait();                              // (all are done with their operands)
    const uint32_t theirs = map_to_cta(smem_u32(smem) + (split * share + tid % share) * LOW_PITCH * 4, tid / share);
#pragma unroll 1
    for (int c16 = 0; c16 < n16; ++c16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c16 * 16, v);
      tmem_ld_wait();
      if (steps == 0)
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0;
#pragma unroll
      for (int i = 0; i < 16; i += 4) st_cluster4(theirs + (c16 * 16 + i) * 4, v + i);
    }
  } else if (warp == 4) {
    const uint32_t idesc = make_idesc(TALL, 16, 1, 1, 0, 0) + (static_cast<uint32_t>((n16 - 1) * 16 >> 3) << 17);
    bool ok = true;
#pragma unroll 1
    for (int s = 0; s < steps && ok; ++s) {
      const int slot = s % MAKE_STAGES;
      ok = wait(&bars.full[slot], (s / MAKE_STAGES) & 1, abort_flag, m.err, ERR_WAIT_FULL, lane);
      if (!ok) break;
      tc_fence_after();
      const uint32_t xa = smem_u32(sx + slot * X_SLOT), aa = smem_u32(sa + slot * A_SLOT);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < KB / 16; ++kk)
          umma_bf16_ss(tmem, make_sdesc_sw128(xa + kk * 32, 16, 1024), make_sdesc_sw128(aa + kk * 32, 16, 1024), idesc, s > 0 || kk > 0 ? 1u : 0u);
        umma_commit(&bars.empty[slot]);
        if (s == steps - 1) umma_commit(&bars.acc_full[0]);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  if (warp >= 4) { __syncwarp(); cluster_arrive(); cluster_wait(); }
  // ---- each CTA adds up its share of the tokens: eight of the rank's values a thread, times the scale, to bf16
  cluster_arrive();
  cluster_wait();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, 64);
  }
  const float* parts = reinterpret_cast<const float*>(smem);
  const int count = min(share, tile.count - split * share), columns = min(RB, m.wide - r0) / 8;
#pragma unroll 1
  for (int i = tid; i < count * columns; i += 192) {
    const int t = i / columns, k = i % columns * 8;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < n16 * 16) {
#pragma unroll 4
      for (int p = 0; p < m.splits; ++p) {
        const float4* from_part = reinterpret_cast<const float4*>(parts + (p * share + t) * LOW_PITCH + k);
        const float4 u = from_part[0], v = from_part[1];
        f[0] += u.x; f[1] += u.y; f[2] += u.z; f[3] += u.w; f[4] += v.x; f[5] += v.y; f[6] += v.z; f[7] += v.w;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = k + e < ranks ? f[e] * by : 0.f;
    *reinterpret_cast<uint4*>(m.low + static_cast<long long>(tile.begin + split * share + t) * m.wide + r0 + k) =
        make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
}

// Told of when this thread's copies have come.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory"); }

// Pieces of 128 tokens and 128 columns; warps 0..3 add to y in shared memory, 4..7 put it back (one thread each half, where a tile is a block), 8 issues products, 9 fetches the
// rank's values, B and y: a tile of neighbours as a block, else four rows at a time.  (Fetched by the threads that put it back, 16 bytes each: 144 us instead of 90 for 8192 tokens
// and 8192 columns.)  Without TMA (rows of B or y that do not begin at 16 bytes) warps 4..7 fetch both.
template <bool TMA>
__global__ void __launch_bounds__(320, 1) add_columns_kernel(const __grid_constant__ CUtensorMap tl, const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap ty,
                                                             const __grid_constant__ CUtensorMap ty_block, const __grid_constant__ Mma m) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Bars bars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.full[i], TMA ? 1 : 4); mbar_init(&bars.empty[i], 1);
      mbar_init(&bars.acc_full[i], 1); mbar_init(&bars.acc_empty[i], 4);
      mbar_init(&bars.y_full[i], TMA ? 1 : 128); mbar_init(&bars.y_done[i], 4); mbar_init(&bars.y_free[i], 4);
    }
    mbar_init(&bars.low_full, 1);
    bars.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
    bars.poisoned = *reinterpret_cast<volatile int*>(m.err);
  }
  // (the tiles are complete when this kernel may begin; the rank's values, and y, after the wait)
  const int kblocks = m.wide / KB, n_tiles = (m.out + ADD_N - 1) / ADD_N;
  const long long units = static_cast<long long>(__ldcg(m.tiles_n)) * n_tiles, each = (units + gridDim.x - 1) / gridDim.x;
  const long long u0 = min(units, blockIdx.x * each), u1 = min(units, u0 + each);
  __syncthreads();
  if (bars.poisoned != 0 || u0 >= u1 || (smem_u32(smem) & 1023u) != 0) {
    if (u0 < u1 && bars.poisoned == 0 && tid == 0) atomicCAS(m.err, 0, static_cast<int>(ERR_BAD_ARG));
    griddep_wait();
    return;
  }
  if (warp == 9 && lane == 0) { tma_prefetch_desc(&tl); if (TMA) { tma_prefetch_desc(&tb); tma_prefetch_desc(&ty); tma_prefetch_desc(&ty_block); } }
  if (warp == 8) { tmem_alloc(&bars.tmem, 2 * ADD_N); tmem_relinquish(); }
  uint8_t *sl = smem, *sb = smem + kblocks * X_SLOT, *sy = sb + ADD_STAGES * B_SLOT;
  volatile int* abort_flag = &bars.abort_flag;
  bool ok = true;
  int piece = 0, tile_at = 0;                    // of this CTA's, the pieces counted over its tiles
#pragma unroll 1
  for (long long u = u0; u < u1; ++tile_at) {
    const int at = static_cast<int>(u / n_tiles), first = static_cast<int>(u - static_cast<long long>(at) * n_tiles);
    const int n = static_cast<int>(min(u1 - u, static_cast<long long>(n_tiles - first))), steps = n * kblocks;
    u += n;
    const int4 what = __ldcg(reinterpret_cast<const int4*>(m.tiles + at));
    const Tile tile{what.x, what.y, what.z, 0};
    __syncthreads();                             // (the tile before is done with)
    if (tid < TALL) bars.rows[tid] = tid < tile.count ? __ldcg(m.order + tile.begin + tid) : -1;
    tc_fence_before();
    __syncthreads();
    const bool block = TMA && neighbours(bars.rows, tile.count, tid);
    tc_fence_after();
    if (tile_at == 0) griddep_wait();
    const uint32_t tmem = bars.tmem;
    if (warp >= 4 && warp < 8) {
      const int p = tid - 128, c = p & 7, yc = p & 15;
      const bf16* b = m.b + static_cast<long long>(tile.adapter) * m.out * m.rank;
      // y's piece i (of this tile's), 16 bytes of 16 rows a thread: fetched, and put back by the thread that fetched it
      auto fetch_y = [&](int i) {
        const int buf = (piece + i) & 1, col = (first + i) * ADD_N + yc * 8, left = m.out - col;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int t = (p >> 4) + 8 * e, row = bars.rows[t];
          if (row >= 0) copy8(smem_u32(sy + buf * Y_SLOT + (yc >> 3) * (TALL * 128) + t * 128 + (((yc & 7) ^ (t & 7)) << 4)), left > 0 ? m.y + static_cast<long long>(row) * m.out + col : m.y, left, m.wide_y);
        }
        if (m.wide_y) copies_arrive(&bars.y_full[buf]);
        else mbar_arrive(&bars.y_full[buf]);
      };
      auto put_back = [&](int i) {
        const int buf = (piece + i) & 1, col = (first + i) * ADD_N + yc * 8, left = m.out - col;
        ok = ok && wait(&bars.y_done[buf], ((piece + i) >> 1) & 1, abort_flag, m.err, ERR_WAIT_OTHER, lane);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int t = (p >> 4) + 8 * e, row = bars.rows[t];
          const uint4 v = *reinterpret_cast<const uint4*>(sy + buf * Y_SLOT + (yc >> 3) * (TALL * 128) + t * 128 + (((yc & 7) ^ (t & 7)) << 4));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
          if (row >= 0 && left > 0 && ok) store8(m.y + static_cast<long long>(row) * m.out + col, w, left, m.wide_y);
        }
      };
      if constexpr (TMA) {
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
          const int buf = (piece + i) & 1, half = warp - 4, col = (first + i) * ADD_N + half * 64;
          if (block && tile.count == TALL) {
            ok = ok && wait(&bars.y_done[buf], ((piece + i) >> 1) & 1, abort_flag, m.err, ERR_WAIT_OTHER, lane);
            if (ok && half < 2 && col < m.out && lane == 0) {
              tma_store_2d(&ty_block, sy + buf * Y_SLOT + half * (TALL * 128), col, bars.rows[0]);
              tma_store_commit();
              tma_store_wait_read<0>();
            }
          } else {
            put_back(i);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.y_free[buf]);
        }
      } else {
        // a slot of B a step (64 of the rank); told of when the next one is on its way
#pragma unroll 1
        for (int step = 0; step <= steps; ++step) {
          const int i = step / kblocks, kb = step - i * kblocks;
          if (step < steps) {
            if (kb == 0) {
              if (i >= 2) put_back(i - 2);
              fetch_y(i);
            }
            const int s = piece * kblocks + step, slot = s % ADD_STAGES, k = kb * KB + c * 8, k_left = m.rank - k;
            ok = ok && wait(&bars.empty[slot], ((s / ADD_STAGES) & 1) ^ 1, abort_flag, m.err, ERR_WAIT_EMPTY, lane);
            const uint32_t bs = smem_u32(sb + slot * B_SLOT) + (p >> 3) * 128 + ((c ^ ((p >> 3) & 7)) << 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int row = (first + i) * ADD_N + (p >> 3) + 16 * e;
              const bool there = row < m.out && k_left > 0;
              copy8(bs + e * 2048, there ? b + static_cast<long long>(row) * m.rank + k : m.b, there ? k_left : 0, m.wide_b);
            }
          }
          copies_end_group();
          if (step == 0) continue;
          copies_wait<1>();
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.full[(piece * kblocks + step - 1) % ADD_STAGES]);
        }
      }
      if constexpr (!TMA) {
        if (n >= 2) put_back(n - 2);
        put_back(n - 1);
      }
    } else if (warp == 9) {
      if (lane == 0) {
        mbar_expect_tx(&bars.low_full, kblocks * X_SLOT);
#pragma unroll 1
        for (int kb = 0; kb < kblocks; ++kb) tma_load_2d(sl + kb * X_SLOT, &tl, &bars.low_full, kb * KB, tile.begin);
      }
      __syncwarp();
      if constexpr (TMA) {
        const int4 four = four_rows(bars.rows, lane);
#pragma unroll 1
        for (int step = 0; step < steps && ok; ++step) {
          const int i = step / kblocks, kb = step - i * kblocks, s = piece * kblocks + step, slot = s % ADD_STAGES, buf = (piece + i) & 1;
          if (kb == 0) {
            ok = wait(&bars.y_free[buf], (((piece + i) >> 1) & 1) ^ 1, abort_flag, m.err, ERR_WAIT_EMPTY, lane);
            if (!ok) break;
            fence_proxy_async();                 // (what threads read and wrote there is behind us)
            if (lane == 0) mbar_expect_tx(&bars.y_full[buf], block ? Y_SLOT : (tile.count + 3) / 4 * 1024);
            __syncwarp();
            if (block && lane < 2) tma_load_2d(sy + buf * Y_SLOT + lane * (TALL * 128), &ty_block, &bars.y_full[buf], (first + i) * ADD_N + lane * 64, bars.rows[0]);
            if (!block && 4 * lane < tile.count) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
                tma_gather4(sy + buf * Y_SLOT + h * (TALL * 128) + lane * 512, &ty, &bars.y_full[buf], (first + i) * ADD_N + h * 64, four.x, four.y, four.z, four.w);
            }
            __syncwarp();
          }
          ok = wait(&bars.empty[slot], ((s / ADD_STAGES) & 1) ^ 1, abort_flag, m.err, ERR_WAIT_EMPTY, lane);
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(&bars.full[slot], B_SLOT);
            tma_load_2d(sb + slot * B_SLOT, &tb, &bars.full[slot], kb * KB, tile.adapter * m.out + (first + i) * ADD_N);
          }
          __syncwarp();
        }
      }
    } else if (warp == 8) {
      constexpr uint32_t idesc = make_idesc(TALL, ADD_N, 1, 1, 0, 0);
      ok = ok && wait(&bars.low_full, tile_at & 1, abort_flag, m.err, ERR_WAIT_FULL, lane);
#pragma unroll 1
      for (int i = 0; i < steps && ok; ++i) {
        const int s = piece * kblocks + i, slot = s % ADD_STAGES, nt = i / kblocks, kb = i - nt * kblocks, buf = (piece + nt) & 1;
        if (kb == 0) ok = wait(&bars.acc_empty[buf], (((piece + nt) >> 1) & 1) ^ 1, abort_flag, m.err, ERR_WAIT_TMEM_EMPTY, lane);
        ok = ok && wait(&bars.full[slot], (s / ADD_STAGES) & 1, abort_flag, m.err, ERR_WAIT_FULL, lane);
        if (!ok) break;
        tc_fence_after();
        const uint32_t la = smem_u32(sl + kb * X_SLOT), ba = smem_u32(sb + slot * B_SLOT);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < KB / 16; ++kk)
            umma_bf16_ss(tmem + buf * ADD_N, make_sdesc_sw128(la + kk * 32, 16, 1024), make_sdesc_sw128(ba + kk * 32, 16, 1024), idesc, kb > 0 || kk > 0 ? 1u : 0u);
          umma_commit(&bars.empty[slot]);
          if (kb == kblocks - 1) umma_commit(&bars.acc_full[buf]);
        }
        __syncwarp();
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int buf = (piece + i) & 1, phase = ((piece + i) >> 1) & 1;
        ok = ok && wait(&bars.acc_full[buf], phase, abort_flag, m.err, ERR_WAIT_TMEM_FULL, lane) && wait(&bars.y_full[buf], phase, abort_flag, m.err, ERR_WAIT_FULL, lane);
        tc_fence_after();
        uint8_t* mine = sy + buf * Y_SLOT + tid * 128;
#pragma unroll
        for (int c = 0; c < ADD_N / 32; ++c) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(warp * 32) << 16) + buf * ADD_N + c * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4* y = reinterpret_cast<uint4*>(mine + (c >> 1) * (TALL * 128) + ((((c & 1) * 4 + q) ^ (tid & 7)) << 4));
            const uint4 was = *y;
            const uint32_t w[4] = {was.x, was.y, was.z, was.w};
            uint32_t now[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) now[j] = pack_bf16(bf16_lo(w[j]) + __uint_as_float(v[q * 8 + 2 * j]), bf16_hi(w[j]) + __uint_as_float(v[q * 8 + 2 * j + 1]));
            *y = make_uint4(now[0], now[1], now[2], now[3]);
          }
        }
        tc_fence_before();
        if (TMA && block) fence_proxy_async();   // (a copy takes it from there)
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.acc_empty[buf]);
          mbar_arrive(&bars.y_done[buf]);
        }
      }
    }
    piece += n;
  }
  let_copies_land(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(bars.tmem, 2 * ADD_N);
  }
}

// One CTA: the tokens by adapter, each adapter's in their order (a run of neighbours is fetched as a block then), and tiles of up to TALL of them.  A warp looks through a
// sixteenth of the tokens, and counts them by adapter for itself.
constexpr int GROUP_WARPS = 16;
__global__ void __launch_bounds__(GROUP_WARPS * 32) group_tokens_kernel(const int* __restrict__ ids, int tokens, int adapters, int* __restrict__ order, int* __restrict__ tiles_n,
                                                                        Tile* __restrict__ tiles, int* __restrict__ err) {
  extern __shared__ int at[];                    // [GROUP_WARPS][adapters]: counts, then where the next token goes
  __shared__ int totals[GROUP_WARPS][2], carry[2];
  constexpr int HELD = 16;                       // ids that a lane keeps
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  griddep_launch();
  const int per = ((tokens + GROUP_WARPS - 1) / GROUP_WARPS + 31) / 32 * 32, from = warp * per, to = min(tokens, from + per);
  int held[HELD];
#pragma unroll
  for (int e = 0; e < HELD; ++e) held[e] = from + e * 32 + lane < to ? ids[from + e * 32 + lane] : -1;
  for (int i = tid; i < GROUP_WARPS * adapters; i += GROUP_WARPS * 32) at[i] = 0;
  if (tid == 0) carry[0] = carry[1] = 0;
  __syncthreads();
  int* mine = at + warp * adapters;
  auto each = [&](auto take) {
#pragma unroll
    for (int e = 0; e < HELD; ++e)
      if (from + e * 32 < to) take(from + e * 32 + lane, held[e]);
#pragma unroll 1
    for (int i0 = from + HELD * 32; i0 < to; i0 += 32) take(i0 + lane, i0 + lane < to ? ids[i0 + lane] : -1);
  };
  each([&](int, int id) {
    const bool there = id >= 0 && id < adapters;
    if (id >= adapters) atomicCAS(err, 0, static_cast<int>(ERR_BAD_ARG));
    const unsigned same = __match_any_sync(FULL, there ? id : -1);
    if (there && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
  });
  __syncthreads();
  for (int i0 = 0; i0 < adapters; i0 += GROUP_WARPS * 32) {
    const int i = i0 + tid;
    int n = 0;
    if (i < adapters)
      for (int w = 0; w < GROUP_WARPS; ++w) {
        const int v = at[w * adapters + i];
        at[w * adapters + i] = n;
        n += v;
      }
    const int t = (n + TALL - 1) / TALL;
    int sn = n, st = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int vn = __shfl_up_sync(FULL, sn, o), vt = __shfl_up_sync(FULL, st, o);
      if (lane >= o) { sn += vn; st += vt; }
    }
    if (lane == 31) { totals[warp][0] = sn; totals[warp][1] = st; }
    __syncthreads();
    int bn = carry[0], bt = carry[1];
    for (int w = 0; w < warp; ++w) { bn += totals[w][0]; bt += totals[w][1]; }
    __syncthreads();
    if (tid == GROUP_WARPS * 32 - 1) { carry[0] = bn + sn; carry[1] = bt + st; }
    if (i < adapters) {
      for (int w = 0; w < GROUP_WARPS; ++w) at[w * adapters + i] += bn + sn - n;
      for (int j = 0; j < t; ++j) tiles[bt + st - t + j] = Tile{i, bn + sn - n + j * TALL, min(TALL, n - j * TALL), 0};
    }
    __syncthreads();
  }
  if (tid == 0) *tiles_n = carry[1];
  each([&](int i, int id) {
    const bool there = id >= 0 && id < adapters;
    const unsigned same = __match_any_sync(FULL, there ? id : -1);
    const int place = there ? mine[id] + __popc(same & ((1u << lane) - 1)) : tokens;
    if (place < tokens) order[place] = i;          // (past the end: never, unless someone writes the ids meanwhile)
    __syncwarp();
    if (there && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
  });
}

int multiprocessors() {
  static int n[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (n[dev] == 0) {
    int v = 0;
    n[dev] = cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0 ? v : 148;
  }
  return n[dev];
}

template <typename K, typename... A>
int launch_early(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, dim3 cluster, const A&... args) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute with[2] = {};
  with[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  with[0].val.programmaticStreamSerializationAllowed = 1;
  with[1].id = cudaLaunchAttributeClusterDimension;
  with[1].val.clusterDim.x = cluster.x;
  with[1].val.clusterDim.y = cluster.y;
  with[1].val.clusterDim.z = 1;
  cfg.attrs = with;
  cfg.numAttrs = cluster.x * cluster.y > 1 ? 2 : 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, args...));
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

// The same on the tensor cores: bf16, rank up to 512, up to 3500 adapters, any widths.  Up to 512 tokens: one launch, no scratch.  More: three, and scratch: low (tokens x rank
// rounded up to 64, bf16), order (tokens integers), tiles (4 integers, then 4 for each of tokens / 128 + min(adapters, tokens) + 1), low and tiles on 16-byte boundaries; splits 1, 2, 4 or 8.
extern "C" int dewb_add_adapters_mma(const void* x, long long x_stride, const void* a, const void* b, const float* scale, const int* ids, int* order, void* tiles, void* low, void* y,
                                     int tokens, int adapters, int rank, int width, int out, int splits, int* err, void* stream_ptr) {
  using namespace dewb::adapters;
  if (tokens <= 0 || out <= 0) return 0;
  if (adapters <= 0 || adapters > MOST_ADAPTERS || rank <= 0 || rank > MOST_RANK || width <= 0 || splits < 1 || splits > 8 || (splits & (splits - 1))) return -3;
  auto whole = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  int* n = static_cast<int*>(tiles);
  const int wide = (rank + KB - 1) / KB * KB;
  const Mma m{static_cast<const bf16*>(x), static_cast<const bf16*>(a), static_cast<const bf16*>(b), scale, ids, order, n, n == nullptr ? nullptr : reinterpret_cast<const Tile*>(n + 4),
              static_cast<bf16*>(low), static_cast<bf16*>(y), x_stride, tokens, adapters, rank, width, out, splits, wide,
              width % 8 == 0 && x_stride % 8 == 0 && whole(x) && whole(a), rank % 8 == 0 && whole(b), out % 8 == 0 && whole(y), err};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (tokens <= SCANNED) {
    const int pad = (rank + 31) / 32 * 32, ranks = rank <= 32 ? 32 : 64, smem = std::max(4 * (STEP_WARPS * MT * ranks + MT * pad) + 2 * MT * (pad + 8), 2 * STEP_WARPS * adapters);
    const dim3 grid(CLUSTER, std::min(tokens, std::min(adapters, tokens) + tokens / MT));
    return rank <= 32 ? launch_early(adapters_step_kernel<CLUSTER, 32>, grid, STEP_THREADS, smem, stream, dim3(CLUSTER), m)
                      : launch_early(adapters_step_kernel<CLUSTER, 64>, grid, STEP_THREADS, smem, stream, dim3(CLUSTER), m);
  }
  if (order == nullptr || tiles == nullptr || low == nullptr || !whole(tiles) || !whole(low)) return -3;
  int rc = launch_early(group_tokens_kernel, dim3(1), GROUP_WARPS * 32, GROUP_WARPS * adapters * 4, stream, dim3(1), ids, tokens, adapters, order, n, reinterpret_cast<Tile*>(n + 4), err);
  if (rc) return rc;
  const int most = tokens / TALL + std::min(adapters, tokens) + 1;
  CUtensorMap t0 = {}, t1 = {}, t2 = {}, t3 = {};
  const uint64_t rows = tokens, ranks = static_cast<uint64_t>(adapters) * rank, outs = static_cast<uint64_t>(adapters) * out;
  const dim3 first(most, splits, (rank + RB - 1) / RB), together(1, splits);
  if (m.wide_x) {
    if ((rc = dewb::make_tmap_2d(&t0, x, rows, width, x_stride, 1, KB, 2, true))) return 1000 + rc;
    if ((rc = dewb::make_tmap_2d(&t1, x, rows, width, x_stride, TALL, KB, 2, true))) return 1000 + rc;
    if ((rc = dewb::make_tmap_2d(&t2, a, ranks, width, width, RB, KB, 2, true))) return 2000 + rc;
    rc = launch_early(make_low_kernel<true>, first, 192, MAKE_SMEM, stream, together, t0, t1, t2, m);
  } else {
    rc = launch_early(make_low_kernel<false>, first, 192, MAKE_SMEM, stream, together, t0, t1, t2, m);
  }
  if (rc) return rc;
  // two CTAs an SM where their memory fits
  const int smem = wide / KB * X_SLOT + ADD_STAGES * B_SLOT + 2 * Y_SLOT, ctas = multiprocessors() * (2 * (smem + 2048) <= 228 * 1024 ? 2 : 1);
  if ((rc = dewb::make_tmap_2d(&t0, low, rows, wide, wide, TALL, KB, 2, true))) return 3000 + rc;
  if (m.wide_b && m.wide_y && outs < 0x7fffff00ull) {
    if ((rc = dewb::make_tmap_2d(&t1, b, outs, rank, rank, ADD_N, KB, 2, true))) return 4000 + rc;
    if ((rc = dewb::make_tmap_2d(&t2, y, rows, out, out, 1, KB, 2, true))) return 5000 + rc;
    if ((rc = dewb::make_tmap_2d(&t3, y, rows, out, out, TALL, KB, 2, true))) return 5000 + rc;
    return launch_early(add_columns_kernel<true>, dim3(ctas), 320, smem, stream, dim3(1), t0, t1, t2, t3, m);
  }
  return launch_early(add_columns_kernel<false>, dim3(ctas), 320, smem, stream, dim3(1), t0, t1, t2, t3, m);
}
