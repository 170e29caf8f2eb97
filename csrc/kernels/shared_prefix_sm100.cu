// A decode step of rows that share prefixes, on the tensor cores: bf16 queries and pools, heads of 64, 128 or 256, pages of a multiple of 16 tokens.
//
// The work is lists of 64-key tiles.  A group's shared keys (shared_range.cuh) make a list for each key head and each 128 of the group's (row, head) queries on it; a row's own
// keys make one for each key head.  All lists stand behind one another in one sequence, which the CTAs share evenly: a list may begin in one CTA and end in another.  Every
// list is the same work to the kernel: up to 128 queries, a page table's row, a range of keys.
//
//   warps 0..3  softmax: a thread a query; also fetch the queries, and write results
//   warp 4      TMA: keys and values, a 64-key tile a slot of one ring, in the order of their use, across lists
//   warp 5      tensor cores: S = Q K^T of a tile into one of two score buffers, O += P V with P over its scores
//
// A query tile is 128 rows tall however few queries a list has (four, of a row's own keys): the products of 64 keys then take 256 cycles, while an SM's share of the memory
// rate brings those 64 keys and values in 1400 (heads of 128).  What a row of a list does is the business of its lane of tensor memory alone, so lanes without a query hold
// anything.  Two CTAs an SM (one at heads of 256): a tile's chain from scores to products is longer than its products, and the other CTA's lie beside it.
//
// No score needs a mask but at the ends of a list's keys, where it is the same for all queries.  Values there are put to zero in shared memory, since a weight of zero does
// not cancel what is not a number.
//
// A list that is a row's whole attention is finished here.  Otherwise (m, l, sum) of a list, or of the piece of it that a CTA had, goes to scratch, and a second kernel joins
// a query's pieces:  o = sum_i 2^(m_i - M) a_i / sum_i 2^(m_i - M) l_i.  Scratch is bounded by queries and CTAs, whatever the keys' number: a CTA holds at most two lists
// in part (its first and its last), the others' queries have a place of their own.  Nothing is counted with atomics: the same call gives the same bits.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../common/ptx.cuh"
#include "../common/shared_range.cuh"
#include "../common/tmap.h"

namespace dewb {
namespace sharedmma {

constexpr int BM = 128, BN = 64;                  // queries of a list, keys of a tile
constexpr int THREADS = 192, TMA_WARP = 4, MMA_WARP = 5;
constexpr int MOST_ROWS = 512;
constexpr float RESCALE = 8.f;                    // how far (log2) a row's maximum may grow before O is rescaled
constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t FULL = 0xffffffffu;

template <int D>
struct Cfg {
  static constexpr int SUB = D / 64;              // 64-column pieces of a row
  static constexpr int Q_BYTES = BM * D * 2;
  static constexpr int SLOT = BN * D * 2;
  static constexpr int RING = D == 64 ? 8 : 4;
  static constexpr int CTAS = D == 256 ? 1 : 2;   // an SM
  static constexpr int TM_O = 2 * BN, TM_COLS = D == 256 ? 512 : 256;
};

struct Bars {
  uint64_t full[8], empty[8], q_full, s_full[2], p_full[2], done;
  uint32_t tmem;
  int abort_flag, poisoned;
};

// what a CTA knows of all lists
struct Lists {
  int prefix_units, per_cta;
  int first[MOST_ROWS + 1];                       // groups: first place
  int lo[MOST_ROWS], hi[MOST_ROWS];               // groups: shared keys (hi 0: none)
  int at[MOST_ROWS + 1];                          // groups: first unit
  int own[MOST_ROWS + 1];                         // places: own tiles before
  int len[MOST_ROWS];                             // places
  short row[MOST_ROWS], group[MOST_ROWS];         // places (-1: none)
  short through[MOST_ROWS];                       // groups: a row that holds something
};

struct Args {
  const __nv_bfloat16* q;
  long long q_stride;
  const int *table, *lengths, *order, *first, *tokens;
  const float* sinks;
  __nv_bfloat16* out;
  float* acc;                                     // [2 rows heads + 2 ctas 128][D]
  float2* ml;                                     // [the same]: maximum (log2), sum
  int* plan;                                      // for the second kernel: see write_plan
  int rows, heads, kv_heads, page_size, box, max_pages, pages, groups, window, least;
  float scale_log2, cap_log2;
  int* err;
};

struct Ranges {                                   // the keys of a list, [a0, a1) and [b0, b1), and its tiles
  int a0, a1, b0, b1;
  __device__ __forceinline__ int a_tiles() const { return a1 > a0 ? (a1 + BN - 1) / BN - a0 / BN : 0; }
  __device__ __forceinline__ int b_first() const { return a1 > a0 ? max(b0 / BN, (a1 + BN - 1) / BN) : b0 / BN; }
  __device__ __forceinline__ int tiles() const { return a_tiles() + (b1 > b0 ? max(0, (b1 + BN - 1) / BN - b_first()) : 0); }
  __device__ __forceinline__ int tile(int i) const { const int n = a_tiles(); return i < n ? a0 / BN + i : b_first() + i - n; }
  __device__ __forceinline__ bool sees(int key) const { return (key >= a0 && key < a1) || (key >= b0 && key < b1); }
  __device__ __forceinline__ bool whole(int tile) const {
    const int x = tile * BN, y = x + BN;
    return (x >= a0 && y <= a1) || (x >= b0 && y <= b1);
  }
};

__device__ __forceinline__ Ranges own_ranges(int len, int window, int lo, int hi) {
  if (len == 0) return Ranges{0, 0, 0, 0};
  const int first = row_first(len, window);
  if (hi == 0) return Ranges{first, len, 0, 0};
  return Ranges{first, max(first, lo), hi, max(hi, len)};
}

struct Item {
  int place, hk, head0, n;                        // first place, key head, first query head, queries
  int each;                                       // query heads a row
  int row;                                        // whose table
  int from, tiles;                                // of the list's tiles
  int slot;                                       // scratch: >= 0 a CTA's place for a piece, -1 the queries' own places of lists of groups, -2 of rows, -3 finished here
  Ranges keys;
};

__device__ __forceinline__ int last_at_most(const int* x, int n, int v) {      // largest i in [0, n) with x[i] <= v (x[0] <= v)
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

// The piece that begins at unit u and ends with its list or before `end`.
__device__ __forceinline__ Item locate(const Lists& s, const Args& a, int u, int end) {
  const int ratio = a.heads / a.kv_heads, chunks = (ratio + BM - 1) / BM;
  Item w;
  int start, units;
  if (u < s.prefix_units) {
    const int g = last_at_most(s.at, a.groups, u);
    const int queries = (s.first[g + 1] - s.first[g]) * ratio, tall = (queries + BM - 1) / BM;
    w.keys = Ranges{s.lo[g], s.hi[g], 0, 0};
    units = w.keys.tiles();
    const int list = (u - s.at[g]) / units;
    start = s.at[g] + list * units;
    w.hk = list / tall;
    const int m0 = (list - w.hk * tall) * BM;
    w.place = s.first[g] * ratio + m0;            // (counted in queries)
    w.each = ratio;
    w.head0 = w.hk * ratio;
    w.n = min(BM, queries - m0);
    w.row = s.through[g];
    w.slot = -1;
  } else {
    const int lists = a.kv_heads * chunks, v = u - s.prefix_units;
    const int i = last_at_most(s.own, a.rows, v / lists);
    units = s.own[i + 1] - s.own[i];
    start = s.prefix_units + s.own[i] * lists;
    const int list = (u - start) / units;
    start += list * units;
    w.hk = list / chunks;
    const int c = list - w.hk * chunks;
    w.n = min(BM, ratio - c * BM);
    w.each = w.n;
    w.place = i * w.n;
    w.head0 = w.hk * ratio + c * BM;
    w.row = s.row[i];
    const int g = s.group[i];
    w.keys = own_ranges(s.len[i], a.window, s.lo[g], s.hi[g]);
    w.slot = s.hi[g] == 0 ? -3 : -2;
  }
  w.from = u - start;
  w.tiles = min(end, start + units) - u;
  if (w.tiles < units) w.slot = 2 * blockIdx.x + (w.from == 0 ? 1 : 0);
  return w;
}

// the row and head of a list's query
__device__ __forceinline__ void query(const Lists& s, const Item& w, int i, int& row, int& head) {
  const int x = w.place + i;
  const int place = x / w.each;
  row = s.row[place];
  head = w.head0 + x - place * w.each;
}

// What the second kernel needs: units a CTA, units of groups, places' tiles, groups and lengths, groups' first units and tiles.
__device__ __forceinline__ void write_plan(const Lists& s, const Args& a, int tid) {
  int* p = a.plan;
  if (tid == 0) { p[0] = s.per_cta; p[1] = s.prefix_units; }
  p += 2;
  for (int i = tid; i <= a.rows; i += THREADS) p[i] = s.own[i];
  p += a.rows + 1;
  for (int i = tid; i < a.rows; i += THREADS) p[i] = s.group[i];
  p += a.rows;
  for (int g = tid; g <= a.groups; g += THREADS) p[g] = s.at[g];
  p += a.groups + 1;
  for (int g = tid; g < a.groups; g += THREADS) p[g] = Ranges{s.lo[g], s.hi[g], 0, 0}.tiles();
}

// Running sums of n numbers f(i) into x[0..n] by one warp.
template <typename F>
__device__ __forceinline__ void running_sums(int* x, int n, int lane, F f) {
  const int per = (n + 31) / 32, i0 = min(n, lane * per), i1 = min(n, i0 + per);
  int sum = 0;
  for (int i = i0; i < i1; ++i) sum += f(i);
  int to = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(FULL, to, o);
    if (lane >= o) to += v;
  }
  int run = to - sum;
  if (lane == 0) x[0] = 0;
  for (int i = i0; i < i1; ++i) { run += f(i); x[i + 1] = run; }
}

__device__ __forceinline__ void make_lists(Lists& s, const Args& a, int tid, int warp, int lane) {
  const int most = a.max_pages * a.page_size, ratio = a.heads / a.kv_heads;
  int* live = s.at;                               // (until the units are known)
  for (int g = tid; g <= a.groups; g += THREADS) {
    s.first[g] = min(max(a.first[g], 0), a.rows);
    if (g == a.groups) break;
    s.lo[g] = 0;
    s.hi[g] = min(max(a.tokens[g], 0), most);
    live[g] = 0;
    s.through[g] = -1;
  }
  __syncthreads();
  for (int i0 = warp * 32; i0 < a.rows; i0 += THREADS) {
    const int i = i0 + lane;
    int g = -1, row = -1, len = 0;
    if (i < a.rows) {
      g = last_at_most(s.first, a.groups, i);
      row = a.order[i];
      bool bad = row < 0 || row >= a.rows;
      if (i < s.first[g] || i >= s.first[g + 1]) { g = -1; bad = true; }
      if (bad) {
        row = -1;
      } else {
        const int n = a.lengths[row];
        bad = n > most;
        len = min(max(n, 0), most);
      }
      if (bad && blockIdx.x == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
      s.row[i] = static_cast<short>(row);
      s.group[i] = static_cast<short>(max(g, 0));
      s.len[i] = len;
    }
    // groups are neighbouring places: lanes of one group answer together
    const bool holds = len > 0 && g >= 0;
    const unsigned same = __match_any_sync(FULL, holds ? g : -1);
    if (holds) {
      const int lo = __reduce_max_sync(same, row_first(len, a.window)), hi = __reduce_min_sync(same, len);
      if (lane == __ffs(same) - 1) {
        atomicMax(&s.lo[g], lo);
        atomicMin(&s.hi[g], hi);
        atomicAdd(&live[g], __popc(same));
        s.through[g] = static_cast<short>(row);   // (any of them)
      }
    }
  }
  __syncthreads();
  for (int g = tid; g < a.groups; g += THREADS)
    if (live[g] < 2 || s.lo[g] >= s.hi[g]) s.lo[g] = s.hi[g] = 0;
  __syncthreads();
  if (warp == 0) {
    running_sums(s.own, a.rows, lane, [&](int i) { return own_ranges(s.len[i], a.window, s.lo[s.group[i]], s.hi[s.group[i]]).tiles(); });
  } else if (warp == 1) {
    running_sums(s.at, a.groups, lane, [&](int g) {
      return s.hi[g] == 0 ? 0 : a.kv_heads * (((s.first[g + 1] - s.first[g]) * ratio + BM - 1) / BM) * Ranges{s.lo[g], s.hi[g], 0, 0}.tiles();
    });
  }
  __syncthreads();
  if (tid == 0) {
    const int units = s.at[a.groups] + s.own[a.rows] * a.kv_heads * ((ratio + BM - 1) / BM);
    s.prefix_units = s.at[a.groups];
    s.per_cta = max(a.least, (units + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
  }
  __syncthreads();
}

template <int D>
__global__ void __launch_bounds__(THREADS, Cfg<D>::CTAS)
shared_mma_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ Args a) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
    return;
  }
  uint8_t *sQ = smem, *ring = smem + C::Q_BYTES;
  Bars* bars = reinterpret_cast<Bars*>(ring + C::RING * C::SLOT);
  Lists& lists = *reinterpret_cast<Lists*>(bars + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    bars->poisoned = *reinterpret_cast<volatile int*>(a.err);
    for (int i = 0; i < C::RING; ++i) { mbar_init(&bars->full[i], 1); mbar_init(&bars->empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&bars->s_full[i], 1); mbar_init(&bars->p_full[i], 4); }
    mbar_init(&bars->q_full, 4);
    mbar_init(&bars->done, 1);
    bars->abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  __syncthreads();
  if (bars->poisoned != 0) return;
  if (warp == MMA_WARP) { tmem_alloc(&bars->tmem, C::TM_COLS); tmem_relinquish(); }
  make_lists(lists, a, tid, warp, lane);
  if (blockIdx.x == 0) write_plan(lists, a, tid);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  volatile int* abort_flag = &bars->abort_flag;
  const int chunks = (a.heads / a.kv_heads + BM - 1) / BM;
  const int units = lists.prefix_units + lists.own[a.rows] * a.kv_heads * chunks;
  const int u0 = static_cast<int>(min(static_cast<long long>(units), static_cast<long long>(blockIdx.x) * lists.per_cta)), u1 = min(units, u0 + lists.per_cta);

  if (warp == TMA_WARP) {
    // ------------------------------------------------------------------ TMA: a list's K0 K1 V0 K2 V1 ... V(n-1); a lane a box of rows
    if (lane == 0) { tma_prefetch_desc(&tk); tma_prefetch_desc(&tv); }
    int slot = 0;
    uint32_t phase = 1;
    bool ok = true;
    const int boxes = BN / a.box;
    for (int u = u0; u < u1 && ok;) {
      const Item w = locate(lists, a, u, u1);
      u += w.tiles;
      const int* table = a.table + static_cast<long long>(w.row) * a.max_pages;
      int row0 = 0, row1 = 0;                     // pool rows of this lane's box of the last two tiles asked for (even, odd)
      unsigned some0 = 0, some1 = 0;              // lanes whose box holds a key of the list
      auto fetch = [&](const CUtensorMap* map, int row, unsigned lanes) -> bool {
        if (!mbar_wait_warp(&bars->empty[slot], phase, abort_flag)) { if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_WAIT_EMPTY)); return false; }
        if (lane == 0) mbar_expect_tx(&bars->full[slot], static_cast<uint32_t>(__popc(lanes)) * a.box * D * 2);
        __syncwarp();
        if (lanes >> lane & 1) {
          uint8_t* to = ring + slot * C::SLOT + lane * a.box * 128;
#pragma unroll
          for (int t = 0; t < C::SUB; ++t) tma_load_2d(to + t * (BN * 128), map, &bars->full[slot], w.hk * D + t * 64, row);
        }
        __syncwarp();
        if (++slot == C::RING) { slot = 0; phase ^= 1; }
        return true;
      };
      auto keys = [&](int j) -> bool {
        const int key0 = w.keys.tile(w.from + j) * BN + lane * a.box;
        bool any = false;
        int row = 0;
        if (lane < boxes) {
          any = (key0 < w.keys.a1 && key0 + a.box > w.keys.a0 && w.keys.a1 > w.keys.a0) || (key0 < w.keys.b1 && key0 + a.box > w.keys.b0 && w.keys.b1 > w.keys.b0);
          if (any) {
            int page = table[key0 / a.page_size];
            if (page < 0 || page >= a.pages) {    // past the pool's end: zeros
              atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
              row = a.pages * a.page_size;
            } else {
              row = page * a.page_size + key0 % a.page_size;
            }
          }
        }
        const unsigned some = __ballot_sync(FULL, any);
        if (j & 1) { row1 = row; some1 = some; } else { row0 = row; some0 = some; }
        return fetch(&tk, row, some);
      };
      ok = keys(0) && (w.tiles < 2 || keys(1));
      for (int j = 0; ok && j < w.tiles; ++j) {
        ok = fetch(&tv, j & 1 ? row1 : row0, j & 1 ? some1 : some0);
        if (ok && j + 2 < w.tiles) ok = keys(j + 2);
      }
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------------ tensor cores (the warp waits together, one lane issues)
    constexpr uint32_t idesc_qk = make_idesc(BM, BN, 1, 1, 0, 0);
    constexpr uint32_t idesc_pv = make_idesc(BM, D, 1, 1, 0, 1);
    int slot = 0;
    uint32_t phase = 0, q_phase = 0, p_phase = 0;  // (p_phase: a bit for each buffer)
    bool ok = true;
    const uint32_t qa = smem_u32(sQ);
    auto take = [&](int& at) -> bool {
      at = slot;
      if (!mbar_wait_warp(&bars->full[slot], phase, abort_flag)) { if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_WAIT_FULL)); return false; }
      if (++slot == C::RING) { slot = 0; phase ^= 1; }
      return true;
    };
    auto scores = [&](int b) -> bool {
      int at;
      if (!take(at)) return false;
      tc_fence_after();
      const uint32_t ka = smem_u32(ring + at * C::SLOT);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16_ss(tmem + b * BN, make_sdesc_sw128(qa + (kk >> 2) * (BM * 128) + (kk & 3) * 32, 16, 1024),
                       make_sdesc_sw128(ka + (kk >> 2) * (BN * 128) + (kk & 3) * 32, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
        umma_commit(&bars->s_full[b]);
        umma_commit(&bars->empty[at]);
      }
      __syncwarp();
      return true;
    };
    for (int u = u0; u < u1 && ok;) {
      const Item w = locate(lists, a, u, u1);
      u += w.tiles;
      ok = mbar_wait_warp(&bars->q_full, q_phase, abort_flag);
      if (!ok) { if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_WAIT_OTHER)); break; }
      q_phase ^= 1;
      ok = scores(0) && (w.tiles < 2 || scores(1));
      for (int j = 0; ok && j < w.tiles; ++j) {
        const int b = j & 1;
        int at;
        ok = take(at);
        if (!ok) break;
        if (!mbar_wait_warp(&bars->p_full[b], p_phase >> b & 1, abort_flag)) { if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_WAIT_OTHER)); ok = false; break; }
        p_phase ^= 1u << b;
        tc_fence_after();
        const uint32_t va = smem_u32(ring + at * C::SLOT);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            umma_bf16_ts(tmem + C::TM_O, tmem + b * BN + kk * 8, make_sdesc_sw128(va + kk * 2048, BN * 128, 1024), idesc_pv, kk > 0 || j > 0 ? 1u : 0u);
          umma_commit(&bars->done);
          umma_commit(&bars->empty[at]);
        }
        __syncwarp();
        if (j + 2 < w.tiles) ok = scores(b);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax, queries, results
    const uint32_t lane_addr = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t t_s = tmem + lane_addr, t_o = tmem + lane_addr + C::TM_O;
    uint32_t s_phase = 0;                          // (a bit for each buffer)
    int taken = 0, products = 0;                  // slots of the ring, and products with values, before this list
    bool ok = true;
    auto queries = [&](const Item& w) {
      constexpr int PIECES = D / 8;
      for (int i = tid; i < w.n * PIECES; i += BM) {
        const int x = i / PIECES, c = i - x * PIECES;
        int row, head;
        query(lists, w, x, row, head);
        const uint4 v = row < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(a.q + row * a.q_stride + static_cast<long long>(head) * D) + c);
        *reinterpret_cast<uint4*>(sQ + (c >> 3) * (BM * 128) + x * 128 + (((c & 7) ^ (x & 7)) << 4)) = v;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_full);
    };
    Item w;
    if (u0 < u1) {
      w = locate(lists, a, u0, u1);
      queries(w);
    }
    for (int u = u0; u < u1 && ok;) {
      const bool active = warp * 32 < w.n, mine = tid < w.n;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < w.tiles; ++j) {
        const int b = j & 1;
        if (!mbar_wait_warp(&bars->s_full[b], s_phase >> b & 1, abort_flag)) { if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_WAIT_TMEM_FULL)); ok = false; break; }
        s_phase ^= 1u << b;
        tc_fence_after();
        const int tile = w.keys.tile(w.from + j);
        const bool whole = w.keys.whole(tile);
        if (active) {
          float s[BN];
          {
            uint32_t v[2][32];
            tmem_ld_32x32b_x32(t_s + b * BN, v[0]);
            tmem_ld_32x32b_x32(t_s + b * BN + 32, v[1]);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < BN; ++x) s[x] = __uint_as_float(v[x >> 5][x & 31]) * a.scale_log2;
          }
          if (a.cap_log2 > 0.f) {
            // cap tanh(s / cap) = cap - 2 cap / (1 + e^(2 s / cap)), in the log2 domain
            const float twice = 2.f * LOG2E / a.cap_log2;
#pragma unroll
            for (int x = 0; x < BN; ++x) s[x] = fmaf(-2.f * a.cap_log2, __fdividef(1.f, 1.f + fast_exp2(s[x] * twice)), a.cap_log2);
          }
          if (!whole) {
#pragma unroll
            for (int x = 0; x < BN; ++x) s[x] = w.keys.sees(tile * BN + x) ? s[x] : -INFINITY;
          }
          float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int x = 4; x < BN; x += 4)
#pragma unroll
            for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], s[x + q]);
          const float m_new = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          const bool need = mine && (m_new - m > RESCALE || (m == -INFINITY && m_new > -INFINITY));
          if (__any_sync(FULL, need)) {
            const float by = need && m > -INFINITY ? fast_exp2(m - m_new) : 1.f;
            if (need) { m = m_new; l *= by; }
            if (j > 0) {
              // (the scores of this tile were behind the products before the last ones: those are all that may still be under way)
              if (!mbar_wait_warp(&bars->done, (products + j - 1) & 1, abort_flag)) { if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_WAIT_OTHER)); ok = false; break; }
              tc_fence_after();
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(t_o + c * 16, v);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 16; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * by);
                tmem_st_32x32b_x16(t_o + c * 16, v);
              }
            }
          }
          const float base = m == -INFINITY ? 0.f : m;
          float sum[2] = {0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const float p0 = fast_exp2(s[c * 32 + 2 * x] - base), p1 = fast_exp2(s[c * 32 + 2 * x + 1] - base);
              pk[x] = pack_bf16(p0, p1);
              sum[0] += p0;
              sum[1] += p1;
            }
            tmem_st_32x32b_x16(t_s + b * BN + c * 16, pk);
          }
          l += sum[0] + sum[1];
          tmem_st_wait();
        }
        if (!whole) {
          // values that nobody sees, to zero: they stand in the slot that the j-th value tile of the list has
          const int at = taken + (j + 1 < w.tiles ? 2 + 2 * j : 2 * w.tiles - 1), slot = at % C::RING;
          if (!mbar_wait_warp(&bars->full[slot], (at / C::RING) & 1, abort_flag)) { if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_WAIT_FULL)); ok = false; break; }
          for (int i = tid; i < BN * C::SUB * 8; i += BM) {
            const int x = (i >> 3) % BN;
            if (!w.keys.sees(tile * BN + x)) *reinterpret_cast<uint4*>(ring + slot * C::SLOT + i * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[b]);
      }
      if (!ok) break;
      taken += 2 * w.tiles;
      products += w.tiles;
      u += w.tiles;
      // all of this list's scores are made: the next one's queries may take their place
      const Item now = w;
      if (u < u1) {
        w = locate(lists, a, u, u1);
        queries(w);
      }
      if (!mbar_wait_warp(&bars->done, (products - 1) & 1, abort_flag)) { if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_WAIT_OTHER)); ok = false; break; }
      tc_fence_after();
      if (active) {
        int row = -1, head = 0;
        if (mine) query(lists, now, tid, row, head);
        const long long one = static_cast<long long>(row) * a.heads + head, all = static_cast<long long>(a.rows) * a.heads;
        const bool last = now.slot == -3;
        const long long at = now.slot >= 0 ? 2 * all + static_cast<long long>(now.slot) * BM + tid : now.slot == -1 ? one : all + one;
        float by = 1.f;
        if (last) {
          const float sink = a.sinks != nullptr && row >= 0 ? a.sinks[head] * LOG2E : -INFINITY;
          const float top = fmaxf(m, sink), own = m > -INFINITY ? fast_exp2(m - top) : 0.f;
          const float total = l * own + (sink > -INFINITY ? fast_exp2(sink - top) : 0.f);
          by = total > 0.f || total != total ? own / total : 0.f;
        } else if (row >= 0) {
          a.ml[at] = make_float2(m, l);
        }
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(t_o + c * 32, v);
          tmem_ld_wait();
          if (row >= 0) {
            if (last) {
              store_row_32<false>(a.out + one * D + c * 32, v, by);
            } else {
              store_row_32<false>(a.acc + at * D + c * 32, v, 1.f);
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TM_COLS);
  }
}

// A CTA a (place, key head), a warp a query: the pieces of its group's list and of its row's.
template <int D>
__global__ void __launch_bounds__(128) join_pieces_kernel(const __grid_constant__ Args a) {
  const int place = blockIdx.x, hk = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ratio = a.heads / a.kv_heads, chunks = (ratio + BM - 1) / BM;
  const int* p = a.plan;
  const int per = p[0], prefix_units = p[1];
  p += 2;
  const int own0 = p[place], own_tiles = p[place + 1] - own0;
  p += a.rows + 1;
  const int g = p[place];
  p += a.rows;
  const int at = p[g];
  p += a.groups + 1;
  const int tiles = p[g];
  const int row = a.order[place];
  if (row < 0 || row >= a.rows) return;
  const bool rests = a.lengths[row] <= 0;
  const int begin = max(0, a.first[g]), queries = (min(a.rows, a.first[g + 1]) - begin) * ratio, tall = (queries + BM - 1) / BM;
  const long long all = static_cast<long long>(a.rows) * a.heads;
  constexpr int EACH = D / 32;
  for (int h = warp; h < ratio; h += 4) {
    const int head = hk * ratio + h;
    const long long one = static_cast<long long>(row) * a.heads + head;
    // the two lists: first unit, tiles, lane
    const int x = (place - begin) * ratio + h, c = h / BM;
    const int start[2] = {at + (hk * tall + x / BM) * tiles, prefix_units + own0 * a.kv_heads * chunks + (hk * chunks + c) * own_tiles};
    const int n[2] = {rests ? 0 : tiles, rests ? 0 : own_tiles}, in[2] = {x % BM, h - c * BM};
    if (n[0] == 0 && n[1] > 0 && start[1] / per == (start[1] + n[1] - 1) / per) continue;      // finished
    float top = a.sinks != nullptr ? a.sinks[head] * LOG2E : -INFINITY, sum = top > -INFINITY ? 1.f : 0.f, o[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) o[i] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (n[k] == 0) continue;
      const int c0 = start[k] / per, c1 = (start[k] + n[k] - 1) / per;
      for (int cta = c0; cta <= c1; ++cta) {
        const long long from = c0 == c1 ? k * all + one : 2 * all + (2ll * cta + (cta == c0 ? 1 : 0)) * BM + in[k];
        const float2 ml = a.ml[from];
        float v[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) v[i] = a.acc[from * D + i * 32 + lane];
        if (ml.x == -INFINITY) {                   // (nothing but scores of minus infinity, or none that is a number)
          if (ml.y != ml.y) sum = ml.y;
          continue;
        }
        const float m = fmaxf(top, ml.x), was = top > -INFINITY ? fast_exp2(top - m) : 0.f, is = fast_exp2(ml.x - m);
        sum = sum * was + ml.y * is;
#pragma unroll
        for (int i = 0; i < EACH; ++i) o[i] = o[i] * was + v[i] * is;
        top = m;
      }
    }
    const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) a.out[one * D + i * 32 + lane] = __float2bfloat16(o[i] * by);
  }
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

template <int D>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int ctas, cudaStream_t stream) {
  using C = Cfg<D>;
  constexpr int SMEM = C::Q_BYTES + C::RING * C::SLOT + static_cast<int>(sizeof(Bars) + sizeof(Lists));
  static_assert(C::CTAS * (SMEM + 1024) <= 228 * 1024, "over an SM's shared memory");
  cudaError_t e = cudaFuncSetAttribute(shared_mma_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e != cudaSuccess) return static_cast<int>(e);
  shared_mma_kernel<D><<<ctas, THREADS, SMEM, stream>>>(tk, tv, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return static_cast<int>(e);
  join_pieces_kernel<D><<<dim3(a.rows, a.kv_heads), 128, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace sharedmma
}  // namespace dewb

// CTAs of the first kernel on the current device (two pieces of 128 queries each are kept in scratch).
extern "C" int dewb_shared_mma_ctas(int D) { return dewb::sharedmma::multiprocessors() * (D == 256 ? 1 : 2); }

// As dewb_shared_decode, on the tensor cores: bf16, D 64, 128 or 256, page_size a multiple of 16, up to 512 rows and as many groups, everything 16-byte aligned and q_stride a
// multiple of 8.  acc: (2 rows heads + 256 ctas) D floats; ml: as many pairs; plan: 2 rows + 2 groups + 4 integers.  A CTA takes at least `least` tiles.  Two launches.
extern "C" int dewb_shared_decode_mma(const void* q, long long q_stride, const void* k, const void* v, const int* table, const int* lengths, const int* order, const int* first,
                                      const int* tokens, const float* sinks, float* acc, void* ml, int* plan, void* out, int rows, int heads, int kv_heads, int D, int page_size,
                                      int max_pages, int pages, int groups, int window, int least, int ctas, float scale, float cap, int* err, void* stream_ptr) {
  using namespace dewb::sharedmma;
  if (rows <= 0) return 0;
  const long long most = static_cast<long long>(max_pages) * page_size, chunks = heads > 0 && kv_heads > 0 ? (heads / kv_heads + BM - 1) / BM : 1;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || page_size <= 0 || page_size % 16 != 0 || max_pages <= 0 || pages <= 0 || groups <= 0 || groups > MOST_ROWS ||
      rows > MOST_ROWS || window < 0 || least < 1 || ctas < 1 || most > 0x3fffffffll || static_cast<long long>(pages) * page_size > 0x7fffff00ll || kv_heads > 65535 ||
      (2ll * rows * chunks + groups) * kv_heads * ((most + BN - 1) / BN + 1) > 0x3fffffffll || q_stride % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(acc)) & 15))
    return -3;
  const int box = page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : 16;
  CUtensorMap tk, tv;
  int r;
  const uint64_t cols = static_cast<uint64_t>(kv_heads) * D, tall = static_cast<uint64_t>(pages) * page_size;
  if ((r = dewb::make_tmap_2d(&tk, k, tall, cols, cols, box, 64, 2, true))) return 1000 + r;
  if ((r = dewb::make_tmap_2d(&tv, v, tall, cols, cols, box, 64, 2, true))) return 2000 + r;
  const Args a{reinterpret_cast<const __nv_bfloat16*>(q), q_stride, table, lengths, order, first, tokens, sinks, reinterpret_cast<__nv_bfloat16*>(out), acc,
               reinterpret_cast<float2*>(ml), plan, rows, heads, kv_heads, page_size, box, max_pages, pages, groups, window, least, scale * LOG2E, cap * LOG2E, err};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (D == 64) return launch<64>(tk, tv, a, ctas, stream);
  if (D == 128) return launch<128>(tk, tv, a, ctas, stream);
  if (D == 256) return launch<256>(tk, tv, a, ctas, stream);
  return -3;
}
