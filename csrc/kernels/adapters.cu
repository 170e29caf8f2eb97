// Low-rank adapters of many requests beside one projection:  y_t += s_i B_i (A_i x_t),  i the adapter of token t (below 0: none).
//
// An adapter's tokens are worked on together, so that its A and B come from memory once for all of them.
//
// STEPS OF GENERATION, up to 512 tokens: one kernel.  A cluster of eight CTAs (four, from 33 tokens on) takes up to 16 tokens of an adapter: each makes the products with A over its part
// of the width, they add them up through one another's shared memory, and each multiplies with its part of B's rows.  Cluster t goes on if token t is the first, 17th, 33rd ... of its adapter, which
// it finds out by looking through the ids.  Operands go from memory to registers as the warp-level products take them (16 rows are too few for the others): a lane of m16n8k16 holds
// two pairs of neighbouring elements of a row, and which elements of the sum they are does not matter as long as both operands agree.  So a lane takes eight in a row (16 bytes),
// four lanes 32, and calls them two products' worth.  B and y are on their way while A's products are added up.  The columns of four n8 blocks are dealt so that a lane's eight
// are neighbours: y is read and written 16 bytes at a time.  Bound by latency (ids, operands, one cluster barrier, results) and, with many adapters, by reading A and B.
//
// PROMPTS: three kernels.  One CTA counts the tokens of each adapter and writes down tiles of up to 128.  Then 128 x 64 x width products, tokens gathered by 16-byte copies, the
// width in parts; then the
// pieces of 128 columns of all tiles, shared evenly by as many CTAs as fit the SMs: the parts' sum times the scale, rounded to bf16, times B on the tensor cores, added to y, whose
// piece has come to shared memory meanwhile and leaves from there (a row's 256 bytes at a time: with 64, from registers, 62 us instead of @@ for 8192 x 4096).  Bound by x and twice y.
//
// The values between the two products are rounded to bf16 after their sum and scale in fp32: what an adapter adds is off by at most half a step of each rank's share.
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
constexpr int SCANNED = 512;     // tokens whose ids each CTA looks through
constexpr int MOST_ADAPTERS = 4096, MOST_RANK = 512;
constexpr uint32_t FULL = 0xffffffffu;

struct Tile { int adapter, begin, count, pad; };

struct Mma {
  const bf16 *x, *a, *b;
  const float* scale;
  const int* ids;
  const int *order, *tiles_n;    // prompts: the tokens by adapter, and their tiles
  const Tile* tiles;
  float* low;                    // prompts: [splits, tokens, rank]
  bf16* y;
  long long x_stride;
  int tokens, adapters, rank, width, out, splits;
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
constexpr int STEP_WARPS = 4, STEP_THREADS = STEP_WARPS * 32, MT = 16;
constexpr int RB = 64;           // rank's values at a time

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// grid (CLUSTER, tokens), clusters of the CTAs of a token
template <int CLUSTER>
__global__ void __launch_bounds__(STEP_THREADS) adapters_step_kernel(const __grid_constant__ Mma m) {
  extern __shared__ __align__(16) float sums[];  // [wide / 8][16][8]: this CTA's share of the rank's values; then as bf16 [16][wide + 8]; in front, the warps' shares
  __shared__ unsigned same[SCANNED / 32];
  __shared__ int rows[MT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int part = cluster_ctarank(), t0 = blockIdx.y;
  griddep_wait();
  // the tokens of this one's adapter
  const int mine = m.ids[t0];
#pragma unroll 1
  for (int i0 = warp * 32; i0 < m.tokens; i0 += STEP_THREADS) {
    const unsigned w = __ballot_sync(FULL, i0 + lane < m.tokens && m.ids[i0 + lane] == mine);
    if (lane == 0) same[i0 >> 5] = w;
  }
  if (mine >= m.adapters && tid == 0 && part == 0) atomicCAS(m.err, 0, static_cast<int>(ERR_BAD_ARG));
  if (tid < MT) rows[tid] = -1;
  __syncthreads();
  if (mine < 0 || mine >= m.adapters) return;
  int before = 0;
#pragma unroll 1
  for (int w = 0; w < t0 >> 5; ++w) before += __popc(same[w]);
  before += __popc(same[t0 >> 5] & ((1u << (t0 & 31)) - 1));
  if (before % MT != 0) return;                  // (all CTAs of a cluster, or none)
#pragma unroll 1
  for (int i = tid; i < m.tokens; i += STEP_THREADS) {
    if (i < t0 || !(same[i >> 5] >> (i & 31) & 1)) continue;
    int rank_of = __popc(same[i >> 5] & ((1u << (i & 31)) - 1)) - before;
#pragma unroll 1
    for (int w = 0; w < i >> 5; ++w) rank_of += __popc(same[w]);
    if (rank_of < MT) rows[rank_of] = i;
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
#pragma unroll 2
      for (int k0 = from + warp * 32; k0 < to; k0 += STEP_WARPS * 32) {
        const int k = k0 + c * 8, left = to - k;
        const uint4 lo = row0 < 0 ? make_uint4(0, 0, 0, 0) : load8(x0 + k, left, m.wide_x), hi = row1 < 0 ? make_uint4(0, 0, 0, 0) : load8(x1 + k, left, m.wide_x);
        const uint32_t one[4] = {lo.x, hi.x, lo.y, hi.y}, two[4] = {lo.z, hi.z, lo.w, hi.w};
        uint4 av[RB / 8];
#pragma unroll
        for (int n = 0; n < RB / 8; ++n)
          av[n] = n < blocks && r0 + n * 8 + g < m.rank ? load8(ar + static_cast<long long>(n) * 8 * m.width + k, left, m.wide_x) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < RB / 8; ++n) {
          if (n >= blocks) break;
          mma16::mma(acc[n], one, av[n].x, av[n].y);
          mma16::mma(acc[n], two, av[n].z, av[n].w);
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
  // ---- meanwhile, this warp's first columns of B and y are fetched
  const int per = ((m.out + CLUSTER - 1) / CLUSTER + 31) / 32 * 32, n_end = min(m.out, (part + 1) * per);
  const bf16* b = m.b + static_cast<long long>(mine) * m.out * m.rank;
  uint4 bv[4], old[2];
  auto fetch_b = [&](int n0, int k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + (g >> 1) * 8 + j * 2 + (g & 1);             // block j's column g
      bv[j] = n < n_end ? load8(b + static_cast<long long>(n) * m.rank + k, m.rank - k, m.wide_b) : make_uint4(0, 0, 0, 0);
    }
  };
  auto fetch_y = [&](int n0) {
    const int col = n0 + c * 8, left = m.out - col;
    old[0] = row0 < 0 ? make_uint4(0, 0, 0, 0) : m.wide_y && left >= 8 ? *reinterpret_cast<const uint4*>(m.y + static_cast<long long>(row0) * m.out + col)
                                                                        : load8(m.y + static_cast<long long>(row0) * m.out + col, left, false);
    old[1] = row1 < 0 ? make_uint4(0, 0, 0, 0) : m.wide_y && left >= 8 ? *reinterpret_cast<const uint4*>(m.y + static_cast<long long>(row1) * m.out + col)
                                                                        : load8(m.y + static_cast<long long>(row1) * m.out + col, left, false);
  };
  int n0 = part * per + warp * 32;
  if (n0 < n_end) {
    fetch_b(n0, c * 8);
    fetch_y(n0);
  }
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
#pragma unroll 1
  for (; n0 < n_end; n0 += STEP_THREADS) {
    float acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
#pragma unroll 1
    for (int k0 = 0; k0 < m.rank; k0 += 32) {
      const uint4 lo = *reinterpret_cast<const uint4*>(low + g * pitch + k0 + c * 8), hi = *reinterpret_cast<const uint4*>(low + (8 + g) * pitch + k0 + c * 8);
      const uint32_t one[4] = {lo.x, hi.x, lo.y, hi.y}, two[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mma16::mma(acc[j], one, bv[j].x, bv[j].y);
        mma16::mma(acc[j], two, bv[j].z, bv[j].w);
      }
      const bool same_columns = k0 + 32 < m.rank;
      if (same_columns || n0 + STEP_THREADS < n_end) fetch_b(same_columns ? n0 : n0 + STEP_THREADS, (same_columns ? k0 + 32 : 0) + c * 8);
    }
    const int col = n0 + c * 8, left = m.out - col;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = i == 0 ? row0 : row1;
      const uint32_t was[4] = {old[i].x, old[i].y, old[i].z, old[i].w};
      uint32_t now[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) now[j] = pack_bf16(bf16_lo(was[j]) + acc[j][2 * i], bf16_hi(was[j]) + acc[j][2 * i + 1]);
      if (row >= 0 && left > 0) store8(m.y + static_cast<long long>(row) * m.out + col, now, left, m.wide_y);
    }
    if (n0 + STEP_THREADS < n_end) fetch_y(n0 + STEP_THREADS);
  }
  cluster_wait();                                // (no CTA's memory goes while another reads it)
}

// ---------------------------------------------------------------------------------------------------------- prompts
constexpr int TALL = 128;        // tokens a tile
constexpr int KB = 64;           // columns of an operand's slot (128 bytes)
constexpr int MAKE_STAGES = 3, AHEAD = 2;
constexpr int X_SLOT = TALL * KB * 2, A_SLOT = RB * KB * 2, MAKE_SMEM = MAKE_STAGES * (X_SLOT + A_SLOT);
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
  uint64_t full[4], empty[4], acc_full[2], acc_empty[2], y_full[2], y_done[2], y_free[2];
  uint32_t tmem;
  int abort_flag, poisoned;
  alignas(16) int rows[TALL];      // (read four at a time)
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code, int lane) {
  if (mbar_wait_warp(bar, parity, abort_flag)) return true;
  if (lane == 0) atomicCAS(err, 0, code);
  return false;
}

// a lane's four rows of a tile (the first one's where there are no more: what comes of those goes nowhere)
__device__ __forceinline__ int4 four_rows(const int* rows, int lane) {
  const int4 v = *reinterpret_cast<const int4*>(rows + 4 * lane);
  return make_int4(v.x < 0 ? rows[0] : v.x, v.y < 0 ? rows[0] : v.y, v.z < 0 ? rows[0] : v.z, v.w < 0 ? rows[0] : v.w);
}

// grid (tile, part of the width, 64 of the rank's values); warps 0..3 write results, warp 4 issues products, warp 5 fetches tokens (a lane four of them) and A.  Without TMA, for
// rows that do not begin at 16 bytes, warps 0..3 fetch: each step then waits for all of a thread's copies at the fence between them and the products (33 us instead of @@ for
// 8192 tokens, 4096 wide).
template <bool TMA>
__global__ void __launch_bounds__(192) make_low_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap ta, const __grid_constant__ Mma m) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Bars bars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < MAKE_STAGES; ++i) { mbar_init(&bars.full[i], TMA ? 1 : 4); mbar_init(&bars.empty[i], 1); }
    mbar_init(&bars.acc_full[0], 1);
    bars.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
    bars.poisoned = *reinterpret_cast<volatile int*>(m.err);
  }
  griddep_launch();
  griddep_wait();                                // (the tiles are the kernel's before this)
  __syncthreads();
  if (bars.poisoned != 0 || static_cast<int>(blockIdx.x) >= *m.tiles_n) return;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (tid == 0) atomicCAS(m.err, 0, static_cast<int>(ERR_BAD_ARG));
    return;
  }
  if (TMA && warp == 5 && lane == 0) { tma_prefetch_desc(&tx); tma_prefetch_desc(&ta); }
  const Tile tile = m.tiles[blockIdx.x];
  if (tid < TALL) bars.rows[tid] = tid < tile.count ? m.order[tile.begin + tid] : -1;
  if (warp == 4) { tmem_alloc(&bars.tmem, 64); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  volatile int* abort_flag = &bars.abort_flag;
  const int split = blockIdx.y, r0 = blockIdx.z * RB, ranks = min(RB, m.rank - r0), n16 = (ranks + 15) / 16;
  const int per = ((m.width + m.splits - 1) / m.splits + KB - 1) / KB * KB, from = split * per, to = min(m.width, from + per);
  const int steps = max(0, (to - from + KB - 1) / KB);
  uint8_t *sx = smem, *sa = smem + MAKE_STAGES * X_SLOT;
  if (TMA && warp == 5) {
    const int4 four = four_rows(bars.rows, lane);
    const bool there = 4 * lane < tile.count;
    const uint32_t bytes = (tile.count + 3) / 4 * 512 + A_SLOT;
    bool ok = true;
#pragma unroll 1
    for (int s = 0; s < steps && ok; ++s) {
      const int slot = s % MAKE_STAGES;
      ok = wait(&bars.empty[slot], ((s / MAKE_STAGES) & 1) ^ 1, abort_flag, m.err, ERR_WAIT_EMPTY, lane);
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(&bars.full[slot], bytes);
        tma_load_2d(sa + slot * A_SLOT, &ta, &bars.full[slot], from + s * KB, tile.adapter * m.rank + r0);
      }
      __syncwarp();
      if (there) tma_gather4(sx + slot * X_SLOT + lane * 512, &tx, &bars.full[slot], from + s * KB, four.x, four.y, four.z, four.w);
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
    const int row = bars.rows[tid];
    float* low = m.low + (static_cast<long long>(split) * m.tokens + max(row, 0)) * m.rank + r0;
#pragma unroll 1
    for (int c16 = 0; c16 < n16; ++c16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c16 * 16, v);
      tmem_ld_wait();
      if (row >= 0) {
        if (steps == 0)
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = 0;
        if (m.rank % 4 == 0 && c16 * 16 + 16 <= ranks) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<uint4*>(low + c16 * 16 + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c16 * 16 + i < ranks) low[c16 * 16 + i] = __uint_as_float(v[i]);
        }
      }
      __syncwarp();
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
  __syncthreads();
  if (warp == 4) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 64);
  }
}

// Pieces of 128 tokens and 128 columns; warps 0..3 add to y in shared memory, 4..7 put it back, 8 issues products, 9 fetches B and y.  Without TMA (rows that do not begin at 16
// bytes) warps 4..7 fetch too.
template <bool TMA>
__global__ void __launch_bounds__(320, 1) add_columns_kernel(const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap ty, const __grid_constant__ Mma m) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Bars bars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.full[i], TMA ? 1 : 4); mbar_init(&bars.empty[i], 1);
      mbar_init(&bars.acc_full[i], 1); mbar_init(&bars.acc_empty[i], 4);
      mbar_init(&bars.y_full[i], TMA ? 1 : 4); mbar_init(&bars.y_done[i], 4); mbar_init(&bars.y_free[i], 4);
    }
    bars.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
    bars.poisoned = *reinterpret_cast<volatile int*>(m.err);
  }
  griddep_wait();
  __syncthreads();
  const int kblocks = (m.rank + KB - 1) / KB, n_tiles = (m.out + ADD_N - 1) / ADD_N;
  const long long units = static_cast<long long>(*m.tiles_n) * n_tiles, each = (units + gridDim.x - 1) / gridDim.x;
  const long long u0 = min(units, blockIdx.x * each), u1 = min(units, u0 + each);
  if (bars.poisoned != 0 || u0 >= u1) return;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (tid == 0) atomicCAS(m.err, 0, static_cast<int>(ERR_BAD_ARG));
    return;
  }
  if (TMA && warp == 9 && lane == 0) { tma_prefetch_desc(&tb); tma_prefetch_desc(&ty); }
  if (warp == 8) { tmem_alloc(&bars.tmem, 2 * ADD_N); tmem_relinquish(); }
  uint8_t *sl = smem, *sb = smem + kblocks * X_SLOT, *sy = sb + ADD_STAGES * B_SLOT;
  volatile int* abort_flag = &bars.abort_flag;
  bool ok = true;
  int piece = 0;                                 // of this CTA's, counted over its tiles
#pragma unroll 1
  for (long long u = u0; u < u1;) {
    const int at = static_cast<int>(u / n_tiles), first = static_cast<int>(u - static_cast<long long>(at) * n_tiles);
    const int n = static_cast<int>(min(u1 - u, static_cast<long long>(n_tiles - first))), steps = n * kblocks;
    u += n;
    const Tile tile = m.tiles[at];
    __syncthreads();                             // (the tile before is done with)
    if (tid < TALL) bars.rows[tid] = tid < tile.count ? m.order[tile.begin + tid] : -1;
    __syncthreads();
    {
      // the rank's values: the parts' sum, times the scale, eight a thread
      const float by = m.scale[tile.adapter];
#pragma unroll 1
      for (int i = tid; i < TALL * kblocks * 8; i += 320) {
        const int t = i / (kblocks * 8), k = i - t * kblocks * 8, row = bars.rows[t], left = m.rank - k * 8;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (row >= 0 && left > 0) {
#pragma unroll 4
          for (int p = 0; p < m.splits; ++p) {
            const float* from = m.low + (static_cast<long long>(p) * m.tokens + row) * m.rank + k * 8;
            if (m.rank % 4 == 0 && left >= 8) {
              const float4 a = *reinterpret_cast<const float4*>(from), b = *reinterpret_cast<const float4*>(from + 4);
              f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w; f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) if (e < left) f[e] += from[e];
            }
          }
        }
        *reinterpret_cast<uint4*>(sl + (k >> 3) * X_SLOT + t * 128 + (((k & 7) ^ (t & 7)) << 4)) =
            make_uint4(pack_bf16(f[0] * by, f[1] * by), pack_bf16(f[2] * by, f[3] * by), pack_bf16(f[4] * by, f[5] * by), pack_bf16(f[6] * by, f[7] * by));
      }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;
    if (warp >= 4 && warp < 8) {
      const int p = tid - 128, c = p & 7, yc = p & 15;
      const bf16* b = m.b + static_cast<long long>(tile.adapter) * m.out * m.rank;
      // put back piece i (of this tile's)
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
          put_back(i);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.y_free[(piece + i) & 1]);
        }
      } else {
        // a slot of B a step (64 of the rank), y's piece with a piece's first; told of when the next one is on its way
#pragma unroll 1
        for (int step = 0; step <= steps; ++step) {
          const int i = step / kblocks, kb = step - i * kblocks;
          if (step < steps) {
            if (kb == 0) {
              if (i >= 2) put_back(i - 2);
              const int buf = (piece + i) & 1, col = (first + i) * ADD_N + yc * 8, left = m.out - col;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const int t = (p >> 4) + 8 * e, row = bars.rows[t];
                if (row >= 0) copy8(smem_u32(sy + buf * Y_SLOT + (yc >> 3) * (TALL * 128) + t * 128 + (((yc & 7) ^ (t & 7)) << 4)), left > 0 ? m.y + static_cast<long long>(row) * m.out + col : m.y, left, m.wide_y);
              }
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
          if (lane == 0) {
            const int before = (step - 1) / kblocks;
            mbar_arrive(&bars.full[(piece * kblocks + step - 1) % ADD_STAGES]);
            if ((step - 1) % kblocks == 0) mbar_arrive(&bars.y_full[(piece + before) & 1]);
          }
        }
        if (n >= 2) put_back(n - 2);
        put_back(n - 1);
      }
    } else if (warp == 9) {
      if constexpr (TMA) {
        const int4 four = four_rows(bars.rows, lane);
        const bool there = 4 * lane < tile.count;
#pragma unroll 1
        for (int step = 0; step < steps && ok; ++step) {
          const int i = step / kblocks, kb = step - i * kblocks, s = piece * kblocks + step, slot = s % ADD_STAGES, buf = (piece + i) & 1;
          if (kb == 0) {
            ok = wait(&bars.y_free[buf], (((piece + i) >> 1) & 1) ^ 1, abort_flag, m.err, ERR_WAIT_EMPTY, lane);
            if (!ok) break;
            fence_proxy_async();                 // (what threads read and wrote there is behind us)
            if (lane == 0) mbar_expect_tx(&bars.y_full[buf], (tile.count + 3) / 4 * 1024);
            __syncwarp();
            if (there) {
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
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.acc_empty[buf]);
          mbar_arrive(&bars.y_done[buf]);
        }
      }
    }
    piece += n;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(bars.tmem, 2 * ADD_N);
  }
}

// One CTA: the tokens by adapter, and tiles of up to TALL of them.  (Where a token stands among its adapter's does not change its result.)
__global__ void __launch_bounds__(1024) group_tokens_kernel(const int* __restrict__ ids, int tokens, int adapters, int* __restrict__ order, int* __restrict__ tiles_n,
                                                            Tile* __restrict__ tiles, int* __restrict__ err) {
  extern __shared__ int at[];                    // [adapters]: counts, then where the next token goes
  __shared__ int totals[32][2], carry[2];
  constexpr int HELD = 8;                        // ids that a thread keeps
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_launch();
  int held[HELD];
#pragma unroll
  for (int e = 0; e < HELD; ++e) held[e] = e * 1024 + tid < tokens ? ids[e * 1024 + tid] : -1;
  for (int i = tid; i < adapters; i += 1024) at[i] = 0;
  if (tid == 0) carry[0] = carry[1] = 0;
  __syncthreads();
  auto each = [&](auto take) {
#pragma unroll
    for (int e = 0; e < HELD; ++e)
      if (e * 1024 < tokens) take(e * 1024 + tid, held[e]);
#pragma unroll 1
    for (int i0 = HELD * 1024; i0 < tokens; i0 += 1024) take(i0 + tid, i0 + tid < tokens ? ids[i0 + tid] : -1);
  };
  each([&](int, int id) {
    const bool there = id >= 0 && id < adapters;
    if (id >= adapters) atomicCAS(err, 0, static_cast<int>(ERR_BAD_ARG));
    const unsigned same = __match_any_sync(FULL, there ? id : -1);
    if (there && lane == __ffs(same) - 1) atomicAdd(&at[id], __popc(same));
  });
  __syncthreads();
  for (int i0 = 0; i0 < adapters; i0 += 1024) {
    const int i = i0 + tid, n = i < adapters ? at[i] : 0, t = (n + TALL - 1) / TALL;
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
    if (tid == 1023) { carry[0] = bn + sn; carry[1] = bt + st; }
    if (i < adapters) {
      at[i] = bn + sn - n;
      for (int j = 0; j < t; ++j) tiles[bt + st - t + j] = Tile{i, bn + sn - n + j * TALL, min(TALL, n - j * TALL), 0};
    }
    __syncthreads();
  }
  if (tid == 0) *tiles_n = carry[1];
  each([&](int i, int id) {
    const bool there = id >= 0 && id < adapters;
    const unsigned same = __match_any_sync(FULL, there ? id : -1);
    int base = 0;
    if (there && lane == __ffs(same) - 1) base = atomicAdd(&at[id], __popc(same));
    base = __shfl_sync(FULL, base, __ffs(same) - 1);
    if (there) order[base + __popc(same & ((1u << lane) - 1))] = i;
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
int launch_early(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, int cluster, const A&... args) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute with[2] = {};
  with[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  with[0].val.programmaticStreamSerializationAllowed = 1;
  with[1].id = cudaLaunchAttributeClusterDimension;
  with[1].val.clusterDim.x = cluster;
  with[1].val.clusterDim.y = with[1].val.clusterDim.z = 1;
  cfg.attrs = with;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
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

// The same on the tensor cores: bf16, rank up to 512, up to 4096 adapters, any widths.  Up to 512 tokens: one launch, no scratch.  More: three, and scratch: low (splits x tokens x
// rank floats), order (tokens integers), tiles (4 integers, then 4 for each of tokens / 128 + min(adapters, tokens) + 1, on a 16-byte boundary).
extern "C" int dewb_add_adapters_mma(const void* x, long long x_stride, const void* a, const void* b, const float* scale, const int* ids, int* order, void* tiles, float* low, void* y,
                                     int tokens, int adapters, int rank, int width, int out, int splits, int* err, void* stream_ptr) {
  using namespace dewb::adapters;
  if (tokens <= 0 || out <= 0) return 0;
  if (adapters <= 0 || adapters > MOST_ADAPTERS || rank <= 0 || rank > MOST_RANK || width <= 0 || splits < 1 || splits > 65535 ) return -3;
  auto whole = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  int* n = static_cast<int*>(tiles);
  const Mma m{static_cast<const bf16*>(x), static_cast<const bf16*>(a), static_cast<const bf16*>(b), scale, ids, order, n, n == nullptr ? nullptr : reinterpret_cast<const Tile*>(n + 4), low,
              static_cast<bf16*>(y), x_stride, tokens, adapters, rank, width, out, splits,
              width % 8 == 0 && x_stride % 8 == 0 && whole(x) && whole(a), rank % 8 == 0 && whole(b), out % 8 == 0 && whole(y), err};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (tokens <= SCANNED) {
    const int wide = (rank + 31) / 32 * 32, smem = 4 * (STEP_WARPS * MT * RB + MT * wide) + 2 * MT * (wide + 8);
    // (128 tokens of 48 adapters of rank 32, 4096 to 6144: clusters of eight 18 us, of four @@; one token, 1024 to 2048: @@)
    return tokens <= 32 ? launch_early(adapters_step_kernel<8>, dim3(8, tokens), STEP_THREADS, smem, stream, 8, m) : launch_early(adapters_step_kernel<4>, dim3(4, tokens), STEP_THREADS, smem, stream, 4, m);
  }
  if (order == nullptr || tiles == nullptr || low == nullptr || !whole(tiles) || !whole(low)) return -3;
  group_tokens_kernel<<<1, 1024, adapters * 4, stream>>>(ids, tokens, adapters, order, n, reinterpret_cast<Tile*>(n + 4), err);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  const int most = tokens / TALL + (adapters < tokens ? adapters : tokens) + 1;
  CUtensorMap t0 = {}, t1 = {};
  const uint64_t rows = tokens, ranks = static_cast<uint64_t>(adapters) * rank, outs = static_cast<uint64_t>(adapters) * out;
  int rc;
  const dim3 first(most, splits, (rank + RB - 1) / RB);
  if (m.wide_x) {
    if ((rc = dewb::make_tmap_2d(&t0, x, rows, width, x_stride, 1, KB, 2, true))) return 1000 + rc;
    if ((rc = dewb::make_tmap_2d(&t1, a, ranks, width, width, RB, KB, 2, true))) return 2000 + rc;
    rc = launch_early(make_low_kernel<true>, first, 192, MAKE_SMEM, stream, 1, t0, t1, m);
  } else {
    rc = launch_early(make_low_kernel<false>, first, 192, MAKE_SMEM, stream, 1, t0, t1, m);
  }
  if (rc) return rc;
  // two CTAs an SM where their memory fits
  const int smem = (rank + KB - 1) / KB * X_SLOT + ADD_STAGES * B_SLOT + 2 * Y_SLOT, ctas = multiprocessors() * (2 * (smem + 2048) <= 228 * 1024 ? 2 : 1);
  if (m.wide_b && m.wide_y && outs < 0x7fffff00ull) {
    if ((rc = dewb::make_tmap_2d(&t0, b, outs, rank, rank, ADD_N, KB, 2, true))) return 3000 + rc;
    if ((rc = dewb::make_tmap_2d(&t1, y, rows, out, out, 1, KB, 2, true))) return 4000 + rc;
    return launch_early(add_columns_kernel<true>, dim3(ctas), 320, smem, stream, 1, t0, t1, m);
  }
  return launch_early(add_columns_kernel<false>, dim3(ctas), 320, smem, stream, 1, t0, t1, m);
}
