// A decode step of rows that share prefixes, on the tensor cores: bf16 queries and pools, heads of 64, 128 or 256, pages of a multiple of 16 tokens.
//
// The work is lists: up to some number of queries (row, head) against a range of keys of one key head.  A group's shared keys (shared_range.cuh) make a list for each key head,
// a row's own keys another.  There are two kinds, each with engines of its own (as many as its share of the work).  All lists of a kind stand behind one another in one sequence
// that its engines share evenly, tile by tile: a list may begin in one engine and end in another.  In front of each list there is room in the sequence for what beginning and
// ending one costs, so that engines with many short lists get fewer tiles.
//
// TALL lists (a group of more than 32 queries on a key head, 128 of them a list): queries are the rows of the products.  Per 64 keys  S = Q K^T  (one of two score buffers in
// tensor memory),  a thread a query makes the weights P over its scores,  O += P V  with P read from tensor memory.
//
// WIDE lists (up to 32 queries: a row's own keys, a small group): keys are the rows, so that few queries make small products and every thread has work.  Per 128 keys
// S^T = K Q^T (16 or 32 columns),  a thread a key makes its weights for all queries,  P^T goes to shared memory,  O^T += V^T P^T (a lane a column of the head).  All queries'
// weights are relative to one maximum a query, which the threads agree on anew only where a score has passed it by 2^8 (one vote a tile); sums of weights stay with the
// threads until the list ends.
//
// An engine is six warps, with rings, barriers and a part of tensor memory of its own:
//   0..3  softmax, results;  tall lists' queries
//   4     TMA: keys and values; finds out what the next list is about, and fetches wide lists' queries
//   5     tensor cores
//
// A CTA an SM, of two engines of one kind (one at heads of 256) whose chains lie beside one another: an SM's share of the memory rate brings 64 keys and values of a head of 128
// in 1400 cycles.  As two CTAs, of either kind as they came, a third of all instruction fetches missed: tall and wide lists' code is more than the SM's instruction cache holds
// (128 rows behind 8192 shared tokens 88 us instead of 65, 61 rows with capped scores 62 instead of 42).
// With four queries as rows of a 128-row product, a wide list's tile took one warp 2300 cycles of scores (four of its lanes had any) and a list of one tile 7100, mostly chain:
// 128 rows in 16 groups of 1000 to 2048 shared tokens 181 us, 128 rows behind 8192 shared tokens 121.
//
// No score needs a mask but at the ends of a list's keys, where it is the same for all queries.  Values there are put to zero in shared memory, since a weight of zero does
// not cancel what is not a number.
//
// A list that is a row's whole attention is finished here.  Otherwise (m, l, sum) of a list, or of the piece of it that an engine had, goes to scratch, and a second kernel joins
// a query's pieces:  o = sum_i 2^(m_i - M) a_i / sum_i 2^(m_i - M) l_i.  Scratch is bounded by queries and engines, whatever the keys' number: an engine holds at most
// two lists in part (its first and its last), the others' queries have a place of their own.  Nothing is counted with atomics: the same call gives the same bits.
#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../common/ptx.cuh"
#include "../common/shared_range.cuh"
#include "../common/tmap.h"

namespace dewb {
namespace sharedmma {

constexpr int BM = 128, BN = 64;                  // tall lists: queries, keys of a tile
constexpr int WK = 128, WN = 32;                  // wide lists: keys of a tile, queries
constexpr int THREADS = 192, TMA_WARP = 4, MMA_WARP = 5;              // of an engine
constexpr int MOST_ROWS = 448;
// tiles that a list takes as long as beyond its own: a tall one, a wide one of a group's, a row's own.  (With 2 for tall ones, 64 rows of 500 keys behind 64 shared ones take 68 us
// instead of 41; with 1 for a group's, 128 rows in 16 groups 100 instead of 90, 256 rows of 256 keys in 32 groups behind 64 tokens 120 instead of 72.)
constexpr int TALL_GAP = 5, SHARED_GAP = 3, WIDE_GAP = 1;
// of a tile (a tall one, one with a cap, a wide one), where engines are dealt: 128 rows behind 8192 tokens take 64 us with 2 : 4 and 75 with 3 : 4, with a cap 82 with 3 : 4, 86
// with 4 : 4 and 97 with 2 : 4
constexpr int TALL_COST = 2, CAPPED_COST = 3, WIDE_COST = 4;
constexpr float RESCALE = 8.f;                    // how far (log2) a query's scores may pass the maximum in use before O is rescaled
constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t FULL = 0xffffffffu;

template <int D>
struct Cfg {
  static constexpr int SUB = D / 64;              // 64-column pieces of a row
  static constexpr int Q_BYTES = BM * D * 2;      // tall: the queries.  wide: two lists' queries and two tiles' weights
  static constexpr int SLOT = BN * D * 2, RING = D == 64 ? 8 : 4, HALF = RING / 2;                // tall: a tile's keys (first half) or values
  static constexpr int W_TILE = WK * D * 2, W_SLOTS = RING / 4;                // wide: the same memory, half for keys and half for values
  static constexpr int W_Q = WN * D * 2, W_P = WN * WK * 2;
  static constexpr int ENGINES = D == 256 ? 1 : 2;                             // a CTA, which has its SM to itself
  static constexpr int HALVES = D == 256 ? 2 : 1; // wide: 128-column pieces of a head
  static constexpr int TM_O = 2 * BN, TM_COLS = D == 256 ? 512 : 256;
  static constexpr int TM_WO = 2 * WN;
  static constexpr int EXTRA = 2 * W_Q + 2 * W_P > Q_BYTES ? 2 * W_Q + 2 * W_P - Q_BYTES : 0;      // (where that is more)
  static constexpr int ENGINE = Q_BYTES + EXTRA + RING * SLOT;                 // bytes
};

struct Ranges {                                   // the keys of a list, [a0, a1) and [b0, b1), counted from `base`, and its tiles of N
  int a0, a1, b0, b1, base;
  template <int N> __device__ __forceinline__ int a_tiles() const { return a1 > a0 ? (a1 + N - 1) / N - a0 / N : 0; }
  template <int N> __device__ __forceinline__ int b_first() const { return a1 > a0 ? max(b0 / N, (a1 + N - 1) / N) : b0 / N; }
  template <int N> __device__ __forceinline__ int tiles() const { return a_tiles<N>() + (b1 > b0 ? max(0, (b1 + N - 1) / N - b_first<N>()) : 0); }
  template <int N> __device__ __forceinline__ int tile(int i) const { const int n = a_tiles<N>(); return i < n ? a0 / N + i : b_first<N>() + i - n; }
  __device__ __forceinline__ bool sees(int key) const { return (key >= a0 && key < a1) || (key >= b0 && key < b1); }
  __device__ __forceinline__ bool meets(int key, int n) const { return (key < a1 && key + n > a0 && a1 > a0) || (key < b1 && key + n > b0 && b1 > b0); }
};

// A list, or the piece of it that an engine has.
struct Item {
  Ranges keys;
  int index, list, lists;                         // group or place, and which of its lists
  bool shared;                                    // of a group
  int start, units;                               // the whole list's first tile, in the sequence, and its tiles
  int from, tiles;                                // of its tiles (tiles 0: the engine's lists are over)
  int place, each, hk, head0, n;                  // first query counted through the places, query heads a row, key head, first query head, queries
  int row;                                        // whose table
};

struct alignas(16) Bars {
  uint64_t list_full[2], list_empty[2];           // what a list is about (wide: and its queries)
  uint64_t full[8], empty[8];                     // slots of the ring: [0, 4) keys, [4, 8) values
  uint64_t q_full, s_full[2], p_full[2];
  uint64_t done[2];                               // of even and odd tiles' products: whoever waits for tile t's knows that tile t - 2's are done, not that t - 1's are
  int abort_flag;
};

struct alignas(16) Own {                          // an engine's
  Bars bars;
  Item item[2];                                   // the list at hand and the next one
  float most[4][WN];                              // wide: largest scores, by warp
  alignas(16) float top[4][WN], by[4][WN];        // (read four at a time) each warp's copy of the maxima in use, and what sums made with older ones are multiplied with
  float sums[4][WN];                              // of weights, by warp
};

// what a CTA knows of all lists (an engine is an engine of the grid's)
struct Lists {
  int tall_units, tall_engines, tall_each, wide_shared_units, wide_units, wide_each;         // (units: tiles and the room in front of lists)
  bool apart;                                     // whether no more engines than CTAs have work
  short first[MOST_ROWS + 2];                     // groups: first place
  short row[MOST_ROWS], group[MOST_ROWS];         // places (row -1: none)
  short through[MOST_ROWS];                       // groups: a row that holds something
  int lo[MOST_ROWS], hi[MOST_ROWS];               // groups: shared keys (hi 0: none)
  int tall[MOST_ROWS + 1], wide[MOST_ROWS + 1];   // groups: units of either kind before
  int own[MOST_ROWS + 1];                         // places: own tiles before
  int len[MOST_ROWS];                             // places
  uint32_t tmem;
  int poisoned;
};

struct Args {
  const __nv_bfloat16* q;
  long long q_stride;
  const int *table, *lengths, *order, *first, *tokens;
  const float* sinks;
  __nv_bfloat16* out;
  float* acc;                                     // [2 rows heads + engines (2 128 + 2 32)][D]
  float2* ml;                                     // [the same]: maximum (log2), sum
  int4* plan;                                     // [rows][2], for the second kernel: see write_plan
  int rows, heads, kv_heads, ratio, chunks, page_size, box, max_pages, pages, groups, window, least;      // (ratio: heads a key head; chunks of 32 of those)
  float scale_log2, cap_log2;
  int* err;
};

// [a0, a1) and [b0, b1) counted from the box that the first of them begins in (so a row's first own tile is full: 64 rows of 500 keys behind 64 shared ones 62 us instead of 86)
__device__ __forceinline__ Ranges ranges(int a0, int a1, int b0, int b1, int box) {
  const int base = (a1 > a0 ? a0 : b0) & -box;     // (boxes are of 16, 32 or 64)
  return a1 > a0 ? Ranges{a0 - base, a1 - base, b0 - base, b1 - base, base} : Ranges{0, 0, b0 - base, b1 - base, base};
}
__device__ __forceinline__ Ranges own_ranges(int len, int window, int lo, int hi, int box) {
  if (len == 0) return Ranges{0, 0, 0, 0, 0};
  const int first = row_first(len, window);
  if (hi == 0) return ranges(first, len, 0, 0, box);
  return ranges(first, max(first, lo), hi, max(hi, len), box);
}

template <typename T>
__device__ __forceinline__ int last_at_most(const T* x, int n, int v) {        // largest i in [0, n) with x[i] <= v (x[0] <= v)
  int lo = 0, hi = n;
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

// A wait that does not end at once, out of line: many places wait, and each launch reads its code anew.
__device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_flag) { return mbar_wait(bar, parity, abort_flag); }
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code, int lane) {
  if (__all_sync(FULL, mbar_try_wait(bar, parity))) return true;
  if (__all_sync(FULL, wait_on(bar, parity, abort_flag))) return true;
  if (lane == 0) atomicCAS(err, 0, code);
  return false;
}

// After a wait that ran out: what is on its way to shared memory gets 20 ms to land before that memory is another's.
__device__ __noinline__ void let_copies_land(volatile int* abort_flag) {
  if (*abort_flag == 0) return;
  const unsigned long long from = globaltimer_ns();
  while (globaltimer_ns() - from < 20000000ull) __nanosleep(1000);
}

__device__ __forceinline__ int group_queries(const Lists& s, const Args& a, int g) { return (s.first[g + 1] - s.first[g]) * a.ratio; }

// The engine's first list, from unit u on, or (!begins) the one behind w's; up to `end`.  One thread.
template <bool TALL>
__device__ __noinline__ void next_list(Item& w, const Lists& s, const Args& a, int u, int end, bool begins) {
  const int* at = TALL ? s.tall : s.wide;
  bool same = false;
  if (begins) {
    w.tiles = 0;
    if (u >= end) return;
    w.shared = TALL || u < s.wide_shared_units;
    w.index = w.shared ? last_at_most(at, a.groups, u) : last_at_most(s.own, a.rows, (u - s.wide_shared_units) / (a.kv_heads * a.chunks));
  } else {
    u = w.start + w.units;                         // (the room in front of the next list)
    w.tiles = 0;
  }
  const int gap = TALL ? TALL_GAP : u < s.wide_shared_units ? SHARED_GAP : WIDE_GAP;
  if (!begins) {
    if (u + gap >= end) return;
    if (++w.list < w.lists) {
      same = true;
      w.start = u + gap;
    } else {
      if (!TALL && w.shared && u >= s.wide_shared_units) {
        w.shared = false;
        w.index = -1;
      }
      if (w.shared) {
#pragma unroll 1
        do ++w.index; while (at[w.index + 1] <= u);
      } else {
#pragma unroll 1
        do ++w.index; while (s.own[w.index + 1] == s.own[w.index]);
      }
    }
  }
  if (!same) {
    if (w.shared) {
      w.keys = ranges(s.lo[w.index], s.hi[w.index], 0, 0, a.box);
      w.lists = a.kv_heads * (TALL ? (group_queries(s, a, w.index) + BM - 1) / BM : 1);
      w.row = s.through[w.index];
      w.start = at[w.index] + gap;
      w.units = w.keys.tiles<TALL ? BN : WK>();
    } else {
      const int g = s.group[w.index];
      w.keys = own_ranges(s.len[w.index], a.window, s.lo[g], s.hi[g], a.box);
      w.lists = a.kv_heads * a.chunks;
      w.row = s.row[w.index];
      w.start = s.wide_shared_units + s.own[w.index] * w.lists + gap;
      w.units = s.own[w.index + 1] - s.own[w.index] - gap;
    }
    w.list = begins ? (u + gap - w.start) / (w.units + gap) : 0;
    w.start += w.list * (w.units + gap);
  }
  if (w.shared) {
    const int queries = group_queries(s, a, w.index), pieces = TALL ? (queries + BM - 1) / BM : 1;
    w.hk = TALL ? w.list / pieces : w.list;
    const int m0 = TALL ? (w.list - w.hk * pieces) * BM : 0;
    w.place = s.first[w.index] * a.ratio + m0;
    w.each = a.ratio;
    w.head0 = w.hk * a.ratio;
    w.n = min(TALL ? BM : WN, queries - m0);
  } else {
    w.hk = a.chunks == 1 ? w.list : w.list / a.chunks;
    const int c = w.list - w.hk * a.chunks;
    w.n = w.each = min(WN, a.ratio - c * WN);
    w.place = w.index * w.n;
    w.head0 = w.hk * a.ratio + c * WN;
  }
  w.from = max(u - w.start, 0);
  w.tiles = max(min(end, w.start + w.units) - max(u, w.start), 0);
}

// row * heads + head of a list's query i, -1 for none
__device__ __forceinline__ int query(const Lists& s, const Args& a, const Item& w, int i) {
  if (i >= w.n) return -1;
  const int x = w.place + i, place = x / w.each, row = s.row[place];
  return row < 0 ? -1 : row * a.heads + w.head0 + x - place * w.each;
}

// A warp's up to 32 queries (lane i holds query()'s answer for number i) to rows of 128 bytes (128-byte swizzle), 64-column pieces `apart` bytes apart; `to`: the first's row,
// on a 1024-byte boundary.  (A loop of copies: it runs once a list, and straight code of 16 loads
// and stores takes 15000 cycles to come from L2 each time.)
template <int D>
__device__ __forceinline__ void fetch_queries(uint8_t* to, int apart, const Args& a, int mine, int n, int lane) {
  constexpr int PIECES = D / 8, ROWS = 32 / PIECES;
  const int row = mine / a.heads, c = lane % PIECES;
  const long long from = mine < 0 ? -1 : row * a.q_stride + static_cast<long long>(mine - row * a.heads) * D;
#pragma unroll 1
  for (int x0 = 0; x0 < n; x0 += ROWS) {
    const int x = x0 + lane / PIECES;
    const long long at = __shfl_sync(FULL, from, x & 31);
    const uint32_t place = smem_u32(to + (c >> 3) * apart + x * 128 + (((c & 7) ^ (x & 7)) << 4));
    const __nv_bfloat16* p = a.q + max(at, 0ll) + c * 8;
    if (x < n) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place), "l"(p), "r"(at < 0 ? 0 : 16) : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  fence_proxy_async();
  __syncwarp();
}

// What the second kernel needs of a place: its group's first unit and tiles (of either kind), its own; its group's first place and queries a key head (0: wide), units a CTA.
// (Nothing for a place that no group holds: group 0's lists, counted from there, would end past the scratch.)
__device__ __forceinline__ void write_plan(const Lists& s, const Args& a) {
  const int lists = a.kv_heads * a.chunks;
#pragma unroll 1
  for (int i = threadIdx.x; i < a.rows; i += blockDim.x) {
    if (s.row[i] < 0) {
      a.plan[2 * i] = a.plan[2 * i + 1] = make_int4(0, 0, 0, 0);
      continue;
    }
    const int g = s.group[i], queries = group_queries(s, a, g);
    const Ranges both = ranges(s.lo[g], s.hi[g], 0, 0, a.box);
    const bool tall = queries > WN;
    a.plan[2 * i] = make_int4(tall ? s.tall[g] : s.wide[g], tall ? both.tiles<BN>() : both.tiles<WK>(), s.wide_shared_units + s.own[i] * lists, max(s.own[i + 1] - s.own[i] - WIDE_GAP, 0));
    a.plan[2 * i + 1] = make_int4(s.first[g], tall ? queries : 0, s.tall_each, s.wide_each);
  }
}

// x[i + 1], 0 <= i < n, to their running sums; x[0] = 0.  One warp.
__device__ __forceinline__ void running_sums(int* x, int n, int lane) {
  const int per = (n + 31) / 32, i0 = min(n, lane * per), i1 = min(n, i0 + per);
  int sum = 0;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) sum += x[i + 1];
  int to = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(FULL, to, o);
    if (lane >= o) to += v;
  }
  int run = to - sum;
  if (lane == 0) x[0] = 0;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) { run += x[i + 1]; x[i + 1] = run; }
}

// All of a CTA's threads.  false: an earlier launch reported an error (read here, beside what else is on its way)
template <int THREADS>
__device__ __forceinline__ bool make_lists(Lists& s, const Args& a, int engines) {
  constexpr int EACH = (MOST_ROWS + THREADS - 1) / THREADS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int most = a.max_pages * a.page_size;
  int* live = s.own;                              // (until the places' tiles are known)
  // rows and lengths are on their way while the groups are looked at
  int row_of[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) row_of[e] = e * THREADS + tid < a.rows ? a.order[e * THREADS + tid] : -1;
  if (tid == THREADS - 1) s.poisoned = *reinterpret_cast<volatile int*>(a.err);
#pragma unroll 1
  for (int g = tid; g <= a.groups; g += THREADS) {
    s.first[g] = static_cast<short>(min(max(a.first[g], 0), a.rows));
    if (g == a.groups) break;
    s.lo[g] = 0;
    s.hi[g] = min(max(a.tokens[g], 0), most);
    live[g] = 0;
    s.through[g] = -1;
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = e * THREADS + tid;
    if (i >= a.rows) break;
    const bool bad = row_of[e] < 0 || row_of[e] >= a.rows;
    s.row[i] = static_cast<short>(bad ? -1 : row_of[e]);
    s.len[i] = bad ? -1 : a.lengths[row_of[e]];
  }
  __syncthreads();
  if (s.poisoned != 0) return false;
#pragma unroll 1
  for (int i0 = warp * 32; i0 < a.rows; i0 += THREADS) {
    const int i = i0 + lane;
    int g = -1, row = -1, len = 0;
    if (i < a.rows) {
      g = last_at_most(s.first, a.groups, i);
      row = s.row[i];
      len = s.len[i];
      bool bad = row < 0 || len > most;
      if (i < s.first[g] || i >= s.first[g + 1]) {
        g = -1;
        bad = true;
      }
      len = g < 0 ? 0 : min(max(len, 0), most);
      if (g < 0) s.row[i] = -1;
      if (bad && blockIdx.x == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
      s.group[i] = static_cast<short>(max(g, 0));
      s.len[i] = len;
    }
    // groups are neighbouring places: lanes of one group answer together
    const unsigned same = __match_any_sync(FULL, len > 0 ? g : -1);
    if (len > 0) {
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
#pragma unroll 1
  for (int g = tid; g < a.groups; g += THREADS) {
    if (blockIdx.x == 0 && s.first[g] > s.first[g + 1]) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
    if (live[g] < 2 || s.lo[g] >= s.hi[g]) s.lo[g] = s.hi[g] = 0;
    const int queries = group_queries(s, a, g);
    const Ranges both = ranges(s.lo[g], s.hi[g], 0, 0, a.box);
    s.tall[g + 1] = s.hi[g] == 0 || queries <= WN ? 0 : a.kv_heads * ((queries + BM - 1) / BM) * (both.tiles<BN>() + TALL_GAP);
    s.wide[g + 1] = s.hi[g] == 0 || queries > WN ? 0 : a.kv_heads * (both.tiles<WK>() + SHARED_GAP);
  }
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < a.rows; i += THREADS) {
    const int n = own_ranges(s.len[i], a.window, s.lo[s.group[i]], s.hi[s.group[i]], a.box).tiles<WK>();
    s.own[i + 1] = n == 0 ? 0 : n + WIDE_GAP;
  }
  __syncthreads();
  if (warp < 3) running_sums(warp == 0 ? s.tall : warp == 1 ? s.wide : s.own, warp < 2 ? a.groups : a.rows, lane);
  __syncthreads();
  if (tid == 0) {
    s.tall_units = s.tall[a.groups];
    s.wide_shared_units = s.wide[a.groups];
    s.wide_units = s.wide_shared_units + s.own[a.rows] * a.kv_heads * a.chunks;
    // engines for either kind by their work
    const long long tall = static_cast<long long>(s.tall_units) * (a.cap_log2 > 0.f ? CAPPED_COST : TALL_COST), wide = static_cast<long long>(s.wide_units) * WIDE_COST;
    int k = tall == 0 ? 0 : wide == 0 ? engines : static_cast<int>((tall * engines + (tall + wide) / 2) / (tall + wide));
    if (tall > 0 && wide > 0) k = min(max(k, 1), engines - 1);
    const int least = a.least + WIDE_GAP;
    s.tall_engines = min(k, (s.tall_units + 2 * least - 1) / (2 * least));
    s.tall_each = s.tall_engines == 0 ? 1 : (s.tall_units + s.tall_engines - 1) / s.tall_engines;
    const int rest = max(1, engines - s.tall_engines);
    s.wide_each = max(least, (s.wide_units + rest - 1) / rest);
    s.apart = s.tall_engines + (s.wide_units + s.wide_each - 1) / s.wide_each <= static_cast<int>(gridDim.x);
  }
  __syncthreads();
  return true;
}

// ---------------------------------------------------------------------------------------------------------- wide lists' softmax
__device__ __forceinline__ bool any_of_128(bool p, int engine) {       // whether p holds for any of an engine's softmax's threads
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"(static_cast<uint32_t>(p)), "r"(1 + engine) : "memory");
  return r != 0;
}
__device__ __forceinline__ void sync_128(int engine) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + engine) : "memory"); }

// largest of a warp's values
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void tmem_ld_x4(uint32_t at, float (&x)[4]) {
  uint32_t v[4];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
}
__device__ __forceinline__ void tmem_st_x4(uint32_t at, const float (&x)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(__float_as_uint(x[0])), "r"(__float_as_uint(x[1])), "r"(__float_as_uint(x[2])),
               "r"(__float_as_uint(x[3])) : "memory");
}
template <int NC>
__device__ __forceinline__ void load_columns(uint32_t at, float (&x)[NC]) {
  if constexpr (NC == 32) {
    uint32_t v[32];
    tmem_ld_32x32b_x32(at, v);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(v[i]);
  } else {
    uint32_t v[16];
    tmem_ld_32x32b_x16(at, v);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < NC; ++i) x[i] = __uint_as_float(v[i]);
  }
}

struct Wide {                                     // what a list's softmax works with
  uint32_t t_s, t_o;                              // tensor memory, this warp's lanes
  uint8_t *weights, *values;                      // shared memory
  Own* own;
  volatile int* abort_flag;
  int tid, warp, lane, engine, at;                // (engine: of the CTA's; at: among those of wide lists)
};

// One wide list of up to NC queries, whose first tile is the CTA's t-th: false after a wait that ran out.  (All warps pass all barriers, whatever went wrong: waits that
// follow one that ran out return at once.)
//
// What runs once a list is written as loops: straight code comes from L2 at some 250 cycles a 128-byte line when a launch first runs it, and all CTAs of a launch are at
// the same line.  (Unrolled over 32 queries, a launch's first maxima took 25000 cycles, and first results 6000.)
template <int D, int NC>
__device__ __forceinline__ bool wide_list(const Wide& x, const Lists& lists, const Args& a, const Item& w, int& t) {
  using C = Cfg<D>;
  Own& own = *x.own;
  Bars* bars = &own.bars;
  const int tid = x.tid, lane = x.lane, warp = x.warp, tiles = w.tiles, n = w.n;
  float *top = own.top[warp], *by = own.by[warp];
  bool ok = true;
  float l[NC];                                    // sums of this thread's keys' weights
#pragma unroll
  for (int q = 0; q < NC; ++q) l[q] = 0.f;
  __syncwarp();
  if (lane < NC) top[lane] = -INFINITY;
  __syncwarp();
#pragma unroll 1
  for (int j = 0; j < tiles; ++j, ++t) {
    const int b = t & 1;
    const bool seen = w.keys.sees(w.keys.tile<WK>(w.from + j) * WK + tid);
    ok = wait(&bars->s_full[b], (t >> 1) & 1, x.abort_flag, a.err, ERR_WAIT_TMEM_FULL, lane) && ok;
    tc_fence_after();
    float s[NC];
    load_columns<NC>(x.t_s + b * WN, s);
#pragma unroll
    for (int q = 0; q < NC; ++q) s[q] *= a.scale_log2;
    if (a.cap_log2 > 0.f) {
      // cap tanh(s / cap) = cap - 2 cap / (1 + e^(2 s / cap)), in the log2 domain
      const float twice = 2.f * LOG2E / a.cap_log2;
#pragma unroll
      for (int q = 0; q < NC; ++q) s[q] = fmaf(-2.f * a.cap_log2, __fdividef(1.f, 1.f + fast_exp2(s[q] * twice)), a.cap_log2);
    }
    bool past = false;
#pragma unroll
    for (int q = 0; q < NC; q += 4) {
      const float4 m = *reinterpret_cast<const float4*>(top + q);
      past = past || (q < n && s[q] > m.x + RESCALE) || (q + 1 < n && s[q + 1] > m.y + RESCALE) || (q + 2 < n && s[q + 2] > m.z + RESCALE) || (q + 3 < n && s[q + 3] > m.w + RESCALE);
    }
    if (j == 0 || any_of_128(past && seen, x.engine)) {
      float mine = -INFINITY;
#pragma unroll
      for (int q = 0; q < NC; ++q) {
        const float most = warp_max(seen ? s[q] : -INFINITY);
        mine = lane == q ? most : mine;
      }
      own.most[warp][lane] = mine;
      sync_128(x.engine);
      if (lane < NC) {
        const float was = top[lane], now = fmaxf(was, fmaxf(fmaxf(own.most[0][lane], own.most[1][lane]), fmaxf(own.most[2][lane], own.most[3][lane])));
        by[lane] = was > -INFINITY && lane < n ? fast_exp2(was - now) : 1.f;
        top[lane] = now;
      }
      __syncwarp();
      if (j > 0) {
#pragma unroll
        for (int q = 0; q < NC; ++q) l[q] *= by[q];
        // (the scores of this tile were behind the products before the last ones: those are all that may still be under way)
        ok = wait(&bars->done[(t - 1) & 1], ((t - 1) >> 1) & 1, x.abort_flag, a.err, ERR_WAIT_OTHER, lane) && ok;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < C::HALVES * WN; c += 4) {
          if ((c & (WN - 1)) >= n) continue;
          float o[4];
          tmem_ld_x4(x.t_o + c, o);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] *= by[(c & (WN - 1)) + i];
          tmem_st_x4(x.t_o + c, o);
        }
        tmem_st_wait();
      }
    }
    // weights: query q's row of 128 keys in two 64-key pieces (128-byte swizzle)
    uint8_t* to = x.weights + b * C::W_P + (tid >> 6) * (WN * 128) + (tid & 7) * 2;
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      const float m = top[q], p = seen ? fast_exp2(s[q] - (m == -INFINITY ? 0.f : m)) : 0.f;
      l[q] += p;
      *reinterpret_cast<__nv_bfloat16*>(to + q * 128 + ((((tid >> 3) & 7) ^ (q & 7)) << 4)) = __float2bfloat16(p);
    }
    if (__ballot_sync(FULL, !seen) != 0) {        // values that nobody sees, to zero (each thread its key's)
      const int slot = t % C::W_SLOTS;
      // (the tile before may still wait for its values in the same slot: its products first)
      if (t > 0) ok = wait(&bars->done[(t - 1) & 1], ((t - 1) >> 1) & 1, x.abort_flag, a.err, ERR_WAIT_OTHER, lane) && ok;
      ok = wait(&bars->full[4 + slot], (t / C::W_SLOTS) & 1, x.abort_flag, a.err, ERR_WAIT_FULL, lane) && ok;
      if (!seen) {
#pragma unroll 1
        for (int p = 0; p < C::SUB; ++p)
#pragma unroll
          for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(x.values + slot * C::W_TILE + p * (WK * 128) + tid * 128 + c * 16) = make_uint4(0, 0, 0, 0);
      }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->p_full[b]);
  }
  // where the results go (lane q: query q's)
  const bool entire = tiles == w.units;
  const bool last = entire && !w.shared && lists.hi[lists.group[w.index]] == 0;
  const int one = query(lists, a, w, lane);
  const long long all = static_cast<long long>(a.rows) * a.heads;
  long long at = last ? one : !entire ? 2 * all + static_cast<long long>(gridDim.x) * (C::ENGINES * 2 * BM) + (2 * x.at + (w.from == 0 ? 1 : 0)) * WN + lane : w.shared ? one : all + one;
  if (one < 0) at = -1;
  // sums over a warp: each exchange halves the queries that a lane is about, until lane i has query i % NC's
#pragma unroll
  for (int h = NC / 2; h > 0; h >>= 1) {
    const bool upper = lane & h;
#pragma unroll
    for (int i = 0; i < h; ++i) {
      const float other = __shfl_xor_sync(FULL, upper ? l[i] : l[i + h], h);
      l[i] = (upper ? l[i + h] : l[i]) + other;
    }
  }
#pragma unroll
  for (int h = NC; h < 32; h <<= 1) l[0] += __shfl_xor_sync(FULL, l[0], h);
  own.sums[warp][lane] = l[0];
  sync_128(x.engine);
  float scale = 1.f;                              // lane q: what query q's result is multiplied with
  if (lane < n) {
    const float m = top[lane], sum = (own.sums[0][lane] + own.sums[1][lane]) + (own.sums[2][lane] + own.sums[3][lane]);
    if (last) {
      const float sink = a.sinks != nullptr ? a.sinks[w.head0 + lane] * LOG2E : -INFINITY;
      const float both = fmaxf(m, sink), part = m > -INFINITY ? fast_exp2(m - both) : 0.f;
      const float total = sum * part + (sink > -INFINITY ? fast_exp2(sink - both) : 0.f);
      scale = sum != sum ? sum : total > 0.f || total != total ? part / total : 0.f;
    } else if (warp == 0 && at >= 0) {
      a.ml[at] = make_float2(m, sum);
    }
  }
  __syncwarp();
  ok = wait(&bars->done[(t - 1) & 1], ((t - 1) >> 1) & 1, x.abort_flag, a.err, ERR_WAIT_OTHER, lane) && ok;
  tc_fence_after();
#pragma unroll 1
  for (int c = 0; c < C::HALVES * WN; c += 4) {
    const int q = c & (WN - 1);
    if (q >= n) continue;
    float o[4];
    tmem_ld_x4(x.t_o + c, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long to = __shfl_sync(FULL, at, q + i);
      const float by = __shfl_sync(FULL, scale, q + i);
      if (q + i < n && to >= 0 && tid < D) {
        const long long place = to * D + (c / WN) * 128 + tid;
        if (last) a.out[place] = __float2bfloat16(o[i] * by);
        else a.acc[place] = o[i];
      }
    }
  }
  tc_fence_before();
  return ok;
}

template <int D>
__global__ void __launch_bounds__(THREADS * Cfg<D>::ENGINES, 1)
shared_mma_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ Args a) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
    return;
  }
  // the softmax's warps of all engines come first: a warp reads the quarter of tensor memory's lanes that its number in the CTA says
  const int number = threadIdx.x >> 5, lane = threadIdx.x & 31, others = number - 4 * C::ENGINES;
  const int engine = others < 0 ? number / 4 : others / 2, warp = others < 0 ? number % 4 : 4 + others % 2, tid = warp * 32 + lane;
  uint8_t *sQ = smem + engine * C::ENGINE, *ring = sQ + C::Q_BYTES + C::EXTRA;
  Own& own = reinterpret_cast<Own*>(smem + C::ENGINES * C::ENGINE)[engine];
  Lists& lists = *reinterpret_cast<Lists*>(reinterpret_cast<Own*>(smem + C::ENGINES * C::ENGINE) + C::ENGINES);
  Bars* bars = &own.bars;
  uint8_t *w_keys = ring, *w_values = ring + C::W_SLOTS * C::W_TILE, *w_weights = sQ + 2 * C::W_Q;
  if (tid == 0) {
    for (int i = 0; i < 8; ++i) { mbar_init(&bars->full[i], 1); mbar_init(&bars->empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], 4);
      mbar_init(&bars->done[i], 1);
      mbar_init(&bars->list_full[i], 1);
      mbar_init(&bars->list_empty[i], 5);         // (the tensor cores' warp, and the softmax's four)
    }
    mbar_init(&bars->q_full, 4);
    bars->abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  griddep_launch();                               // (the second kernel's CTAs come as these end; they wait for all of this grid)
  if (warp == TMA_WARP && lane == 0 && engine == 0) { tma_prefetch_desc(&tk); tma_prefetch_desc(&tv); }
  const int engines = static_cast<int>(gridDim.x) * C::ENGINES;
  if (!make_lists<THREADS * C::ENGINES>(lists, a, engines)) {
    if (blockIdx.x == gridDim.x - 1)              // (the second kernel finds that there is nothing)
      for (int i = threadIdx.x; i < 2 * a.rows; i += blockDim.x) a.plan[i] = make_int4(0, 0, 0, 0);
    return;
  }
  if (warp == MMA_WARP && engine == 0) { tmem_alloc(&lists.tmem, C::ENGINES * C::TM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = lists.tmem + engine * C::TM_COLS;
  volatile int* abort_flag = &bars->abort_flag;
  // this engine's kind, number among those of its kind, and units.  (A CTA's two are of one kind but in one CTA at most: of two kinds, each pushes the other's code out of the SM's
  // instruction cache.  Where there are CTAs enough, only one of each has work)
  const int place = lists.apart ? engine * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) * C::ENGINES + engine;
  const bool tall = place < lists.tall_engines;
  const int at = tall ? place : place - lists.tall_engines;
  const int units = tall ? lists.tall_units : lists.wide_units, per = tall ? lists.tall_each : lists.wide_each;
  const int u0 = static_cast<int>(min(static_cast<long long>(units), static_cast<long long>(at) * per)), u1 = min(units, u0 + per);
  bool ok = true;
  // pool row of the box of tokens that holds `key`, by a row's table
  auto pool_row = [&](int row, int key) -> int {
    const int page = a.table[static_cast<long long>(row) * a.max_pages + key / a.page_size];
    if (page < 0 || page >= a.pages) {            // past the pool's end: zeros
      atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
      return a.pages * a.page_size;
    }
    return page * a.page_size + key % a.page_size;
  };
  // the TMA warp: boxes of rows of one tile, a lane a box, to `to`
  auto load = [&](const CUtensorMap* map, uint8_t* to, int keys, uint64_t* full, int row, unsigned lanes, int hk) {
    if (lane == 0) mbar_expect_tx(full, static_cast<uint32_t>(__popc(lanes)) * a.box * D * 2);
    __syncwarp();
    if (lanes >> lane & 1) {
#pragma unroll
      for (int p = 0; p < C::SUB; ++p) tma_load_2d(to + lane * a.box * 128 + p * (keys * 128), map, full, hk * D + p * 64, row);
    }
    __syncwarp();
  };

  if (tall && warp == TMA_WARP) {
    // K(0) K(1) V(0) K(2) V(1) ...  (t counts the CTA's tiles, over all lists)
    int list = -1, j = 0, tiles = 0, total = 0x3fffffff;
    int row0 = 0, row1 = 0, hk0 = 0, hk1 = 0;     // of the last even and odd tile whose keys were asked for
    unsigned lanes0 = 0, lanes1 = 0;
#pragma unroll 1
    for (int t = 0; ok && t < total + 2; ++t) {
#pragma unroll 1
      for (int what = 0; what < 2 && ok; ++what) {                 // the values of tile t - 2, the keys of tile t
        if (what == 0 ? t < 2 : t >= total) continue;
        if (what == 1) {
          if (j == tiles) {
            ++list;
            ok = wait(&bars->list_empty[list & 1], ((list >> 1) & 1) ^ 1, abort_flag, a.err, ERR_WAIT_EMPTY, lane);
            if (!ok) break;
            if (lane == 0) {
              if (list > 0) own.item[list & 1] = own.item[(list & 1) ^ 1];
              next_list<true>(own.item[list & 1], lists, a, u0, u1, list == 0);
              mbar_arrive(&bars->list_full[list & 1]);
            }
            __syncwarp();
            tiles = own.item[list & 1].tiles;
            j = 0;
            if (tiles == 0) { total = t; continue; }
          }
          const Item& w = own.item[list & 1];
          const int key = w.keys.tile<BN>(w.from + j) * BN + lane * a.box;
          const bool any = lane * a.box < BN && w.keys.meets(key, a.box);
          const int row = any ? pool_row(w.row, w.keys.base + key) : 0;
          const unsigned lanes = __ballot_sync(FULL, any);
          if (t & 1) { row1 = row; lanes1 = lanes; hk1 = w.hk; } else { row0 = row; lanes0 = lanes; hk0 = w.hk; }
          ++j;
        }
        const int nth = what == 1 ? t : t - 2, slot = nth % C::HALF, bar = 4 * (1 - what) + slot;
        ok = wait(&bars->empty[bar], ((nth / C::HALF) & 1) ^ 1, abort_flag, a.err, ERR_WAIT_EMPTY, lane);
        if (!ok) break;
        load(what == 1 ? &tk : &tv, ring + (slot + (what == 1 ? 0 : C::HALF)) * C::SLOT, BN, &bars->full[bar], t & 1 ? row1 : row0, t & 1 ? lanes1 : lanes0, t & 1 ? hk1 : hk0);
      }
    }
  } else if (tall && warp == MMA_WARP) {
    // over the tiles of all lists: S(0) S(1) PV(0) S(2) PV(1) ..., but all of a list's products before the next one's scores, whose queries come when its softmax is done (the warp
    // waits together, one lane issues)
    constexpr uint32_t idesc_qk = make_idesc(BM, BN, 1, 1, 0, 0);
    constexpr uint32_t idesc_pv = make_idesc(BM, D, 1, 1, 0, 1);
    int list = -1, j = 0, tiles = 0, pv = 0;
    uint32_t fresh = 0;                           // (a bit for each buffer, whether its tile is its list's first)
    const uint32_t qa = smem_u32(sQ);
#pragma unroll 1
    for (int t = 0; ok; ++t) {
      const bool begins = j == tiles;
#pragma unroll 1
      for (; pv < (begins ? t : t - 1); ++pv) {   // PV(pv)
        const int b = pv & 1, slot = pv % C::HALF;
        ok = wait(&bars->full[4 + slot], (pv / C::HALF) & 1, abort_flag, a.err, ERR_WAIT_FULL, lane) && wait(&bars->p_full[b], (pv >> 1) & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane);
        if (!ok) break;
        tc_fence_after();
        const uint32_t va = smem_u32(ring + (C::HALF + slot) * C::SLOT);
        const uint32_t add = fresh >> b & 1 ? 0u : 1u;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            umma_bf16_ts(tmem + C::TM_O, tmem + b * BN + kk * 8, make_sdesc_sw128(va + kk * 2048, BN * 128, 1024), idesc_pv, kk > 0 ? 1u : add);
          umma_commit(&bars->done[b]);
          umma_commit(&bars->empty[4 + slot]);
        }
        __syncwarp();
      }
      if (!ok) break;
      const int b = t & 1;
      fresh &= ~(1u << b);
      if (begins) {
        ++list;
        ok = wait(&bars->list_full[list & 1], (list >> 1) & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane);
        if (!ok) break;
        tiles = own.item[list & 1].tiles;
        if (tiles == 0) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->list_empty[list & 1]);
        ok = wait(&bars->q_full, list & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane);
        j = 0;
        fresh |= 1u << b;
      }
      ++j;
      const int slot = t % C::HALF;
      ok = ok && wait(&bars->full[slot], (t / C::HALF) & 1, abort_flag, a.err, ERR_WAIT_FULL, lane);
      if (!ok) break;
      tc_fence_after();
      const uint32_t ka = smem_u32(ring + slot * C::SLOT);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16_ss(tmem + b * BN, make_sdesc_sw128(qa + (kk >> 2) * (BM * 128) + (kk & 3) * 32, 16, 1024),
                       make_sdesc_sw128(ka + (kk >> 2) * (BN * 128) + (kk & 3) * 32, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
        umma_commit(&bars->s_full[b]);
        umma_commit(&bars->empty[slot]);
      }
      __syncwarp();
    }
  } else if (tall) {
    const uint32_t lane_addr = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t t_s = tmem + lane_addr, t_o = tmem + lane_addr + C::TM_O;
    // scores take their scale with the maximum's subtraction, where that orders them and nothing comes between
    const bool plain = a.cap_log2 <= 0.f && a.scale_log2 > 0.f;
    const float factor = plain ? a.scale_log2 : 1.f;
    float* to = nullptr;                          // where the last list's result goes
    bool active = false;
#pragma unroll 1
    for (int t = 0, list = 0;; ++list) {
      // all scores of the lists before are made: the next one's queries may take the place of theirs
      const Item& w = own.item[list & 1];
      ok = wait(&bars->list_full[list & 1], (list >> 1) & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane);
      if (!ok) break;
      const int tiles = w.tiles;
      int one = -1;
      if (tiles > 0) {
        one = query(lists, a, w, tid);
        fetch_queries<D>(sQ + warp * 32 * 128, BM * 128, a, one, min(32, w.n - warp * 32), lane);
        if (lane == 0) mbar_arrive(&bars->q_full);
      }
      if (list > 0) {
        ok = wait(&bars->done[(t - 1) & 1], ((t - 1) >> 1) & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane);
        if (!ok) break;
        tc_fence_after();
        if (active) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(t_o + c * 32, v);
            tmem_ld_wait();
            if (to != nullptr) store_row_32<false>(to + c * 32, v, 1.f);
            __syncwarp();
          }
        }
        tc_fence_before();
      }
      if (tiles == 0) break;
      const bool mine = tid < w.n;
      active = warp * 32 < w.n;
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = 0; j < tiles; ++j, ++t) {
        const int b = t & 1;
        // which of the tile's keys the list sees
        const int key0 = w.keys.tile<BN>(w.from + j) * BN;
        const uint32_t sees[2] = {__ballot_sync(FULL, w.keys.sees(key0 + lane)), __ballot_sync(FULL, w.keys.sees(key0 + 32 + lane))};
        const bool whole = (sees[0] & sees[1]) == FULL;
        ok = wait(&bars->s_full[b], (t >> 1) & 1, abort_flag, a.err, ERR_WAIT_TMEM_FULL, lane);
        if (!ok) break;
        tc_fence_after();
        if (active) {
          float s[BN];
          {
            uint32_t v[2][32];
            tmem_ld_32x32b_x32(t_s + b * BN, v[0]);
            tmem_ld_32x32b_x32(t_s + b * BN + 32, v[1]);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < BN; ++x) s[x] = __uint_as_float(v[x >> 5][x & 31]);
          }
          if (!plain) {
#pragma unroll
            for (int x = 0; x < BN; ++x) s[x] *= a.scale_log2;
            if (a.cap_log2 > 0.f) {
              // cap tanh(s / cap) = cap - 2 cap / (1 + e^(2 s / cap)), in the log2 domain
              const float twice = 2.f * LOG2E / a.cap_log2;
#pragma unroll
              for (int x = 0; x < BN; ++x) s[x] = fmaf(-2.f * a.cap_log2, __fdividef(1.f, 1.f + fast_exp2(s[x] * twice)), a.cap_log2);
            }
          }
          if (!whole) {
#pragma unroll
            for (int x = 0; x < BN; ++x) s[x] = sees[x >> 5] >> (x & 31) & 1 ? s[x] : -INFINITY;
          }
          float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int x = 4; x < BN; x += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q) mx[q] = x + 4 + q < BN ? fmaxf(fmaxf(mx[q], s[x + q]), s[x + 4 + q]) : fmaxf(mx[q], s[x + q]);
          const float m_new = fmaxf(m, factor * fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          const bool need = mine && (m_new - m > RESCALE || (m == -INFINITY && m_new > -INFINITY));
          if (__any_sync(FULL, need)) {
            const float by = need && m > -INFINITY ? fast_exp2(m - m_new) : 1.f;
            if (need) { m = m_new; l *= by; }
            if (j > 0) {
              // (the scores of this tile were behind the products before the last ones: those are all that may still be under way)
              ok = wait(&bars->done[(t - 1) & 1], ((t - 1) >> 1) & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
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
          const uint64_t times = pair_of(factor, factor), less = pair_of(-base, -base);
          uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              float p0, p1;
              unpair(fma2(pair_of(s[c * 32 + 2 * x], s[c * 32 + 2 * x + 1]), times, less), p0, p1);
              p0 = fast_exp2(p0);
              p1 = fast_exp2(p1);
              pk[x] = pack_bf16(p0, p1);
              if (x & 1) sum1 = add2(sum1, pair_of(p0, p1)); else sum0 = add2(sum0, pair_of(p0, p1));
            }
            tmem_st_32x32b_x16(t_s + b * BN + c * 16, pk);
          }
          float p0, p1;
          unpair(add2(sum0, sum1), p0, p1);
          l += p0 + p1;
          tmem_st_wait();
        }
        if (!whole) {
          // values that nobody sees, to zero, in the slot that the t-th value tile has
          const int slot = t % C::HALF;
          ok = wait(&bars->full[4 + slot], (t / C::HALF) & 1, abort_flag, a.err, ERR_WAIT_FULL, lane);
          if (!ok) break;
          const int x = tid >> 1;                 // a key's values by two threads
          if (!((x < 32 ? sees[0] : sees[1]) >> (x & 31) & 1)) {
#pragma unroll 1
            for (int p = 0; p < C::SUB; ++p)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                *reinterpret_cast<uint4*>(ring + (C::HALF + slot) * C::SLOT + p * (BN * 128) + x * 128 + ((tid & 1) * 4 + c) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[b]);
      }
      if (!ok) break;
      // (a piece of a list goes to a place of the CTA's)
      to = nullptr;
      if (one >= 0) {
        const long long where = tiles == w.units ? one : 2ll * a.rows * a.heads + static_cast<long long>(2 * at + (w.from == 0 ? 1 : 0)) * BM + tid;
        a.ml[where] = make_float2(m, l);
        to = a.acc + where * D;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->list_empty[list & 1]);
    }
  } else if (warp == TMA_WARP) {
    // K(0) V(0) K(1) V(1) ...; a tile's pages are looked up while the values of the one before wait for their slot, unless that would wait for an item's room
    int list = -1, j = 0, tiles = 0, row = 0, hk = 0;
    unsigned lanes = 0;
    bool begins = true, more = true;
#pragma unroll 1
    for (int t = -1; ok && more; ++t) {
      const int slot = t % C::W_SLOTS, row_v = row, hk_v = hk;
      const uint32_t phase = ((t / C::W_SLOTS) & 1) ^ 1;
      const unsigned lanes_v = lanes;
      if (t >= 0) {
        ok = wait(&bars->empty[slot], phase, abort_flag, a.err, ERR_WAIT_EMPTY, lane);
        if (!ok) break;
        load(&tk, w_keys + slot * C::W_TILE, WK, &bars->full[slot], row, lanes, hk);
        if (begins) {
          const Item& w = own.item[list & 1];
          fetch_queries<D>(sQ + (list & 1) * C::W_Q, WN * 128, a, query(lists, a, w, lane), w.n, lane);
          if (lane == 0) mbar_arrive(&bars->list_full[list & 1]);
        }
      }
      const int next = list + 1;
      const bool early = j < tiles || __all_sync(FULL, mbar_try_wait(&bars->list_empty[next & 1], ((next >> 1) & 1) ^ 1));
#pragma unroll 1
      for (int what = 0; what < 2 && ok; ++what) {
        if (early != (what == 0)) {               // the values
          if (t < 0) continue;
          ok = wait(&bars->empty[4 + slot], phase, abort_flag, a.err, ERR_WAIT_EMPTY, lane);
          if (ok) load(&tv, w_values + slot * C::W_TILE, WK, &bars->full[4 + slot], row_v, lanes_v, hk_v);
          continue;
        }
        begins = j == tiles;                      // the next tile
        if (begins) {
          list = next;
          ok = wait(&bars->list_empty[list & 1], ((list >> 1) & 1) ^ 1, abort_flag, a.err, ERR_WAIT_EMPTY, lane);
          if (!ok) break;
          if (lane == 0) {
            if (list > 0) own.item[list & 1] = own.item[(list & 1) ^ 1];
            next_list<false>(own.item[list & 1], lists, a, u0, u1, list == 0);
          }
          __syncwarp();
          tiles = own.item[list & 1].tiles;
          j = 0;
          if (tiles == 0) {
            more = false;
            if (lane == 0) mbar_arrive(&bars->list_full[list & 1]);
            continue;
          }
        }
        const Item& w = own.item[list & 1];
        const int key = w.keys.tile<WK>(w.from + j) * WK + lane * a.box;
        const bool any = lane * a.box < WK && w.keys.meets(key, a.box);
        row = any ? pool_row(w.row, w.keys.base + key) : 0;
        lanes = __ballot_sync(FULL, any);
        hk = w.hk;
        ++j;
      }
    }
  } else if (warp == MMA_WARP) {
    // S(0) S(1) PV(0) S(2) PV(1) ..., but a list's last products before the next one's scores
    constexpr uint32_t idesc_s[2] = {make_idesc(WK, 16, 1, 1, 0, 0), make_idesc(WK, 32, 1, 1, 0, 0)};
    constexpr uint32_t idesc_o[2] = {make_idesc(128, 16, 1, 1, 1, 0), make_idesc(128, 32, 1, 1, 1, 0)};
    int list = -1, j = 0, tiles = 0;
    bool more = false, over = false;              // (more: than 16 queries)
    uint32_t flags = 0;                           // bits b: whether the tile in buffer b is its list's first, 2 + b: whether its list has more than 16 queries
#pragma unroll 1
    for (int t = 0; ok && !over; ++t) {
      const bool begins = j == tiles;
#pragma unroll 1
      for (int what = 0; what < 2 && ok; ++what) {
        if (begins == (what == 0)) {              // PV(t - 1)
          if (t == 0) continue;
          const int b = (t - 1) & 1, slot = (t - 1) % C::W_SLOTS;
          ok = wait(&bars->full[4 + slot], ((t - 1) / C::W_SLOTS) & 1, abort_flag, a.err, ERR_WAIT_FULL, lane) &&
               wait(&bars->p_full[b], ((t - 1) >> 1) & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane);
          if (!ok) break;
          tc_fence_after();
          const uint32_t va = smem_u32(w_values + slot * C::W_TILE), pa = smem_u32(w_weights + b * C::W_P);
          const uint32_t idesc = flags >> (2 + b) & 1 ? idesc_o[1] : idesc_o[0], add = flags >> b & 1 ? 0u : 1u;
          if (elect_one()) {
#pragma unroll
            for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
              for (int kk = 0; kk < WK / 16; ++kk)  // (a head of 64 fills half of the rows: the others are of whatever follows)
                umma_bf16_ss(tmem + C::TM_WO + h * WN, make_sdesc_sw128(va + h * 2 * (WK * 128) + kk * 2048, D == 64 ? WK * 64 : WK * 128, 1024),
                             make_sdesc_sw128(pa + (kk >> 2) * (WN * 128) + (kk & 3) * 32, 16, 1024), idesc, kk > 0 ? 1u : add);
            umma_commit(&bars->done[b]);
            umma_commit(&bars->empty[4 + slot]);
          }
          __syncwarp();
          continue;
        }
        if (begins) {
          ++list;
          ok = wait(&bars->list_full[list & 1], (list >> 1) & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane);
          if (!ok) break;
          tiles = own.item[list & 1].tiles;
          more = own.item[list & 1].n > 16;
          j = 0;
          over = tiles == 0;
          if (over) break;
        }
        const int b = t & 1, slot = t % C::W_SLOTS;                // S(t)
        flags = (flags & ~(5u << b)) | ((j == 0 ? 1u : 0u) | (more ? 4u : 0u)) << b;
        ++j;
        ok = wait(&bars->full[slot], (t / C::W_SLOTS) & 1, abort_flag, a.err, ERR_WAIT_FULL, lane);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ka = smem_u32(w_keys + slot * C::W_TILE), qa = smem_u32(sQ + (list & 1) * C::W_Q), idesc = more ? idesc_s[1] : idesc_s[0];
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16_ss(tmem + b * WN, make_sdesc_sw128(ka + (kk >> 2) * (WK * 128) + (kk & 3) * 32, 16, 1024),
                         make_sdesc_sw128(qa + (kk >> 2) * (WN * 128) + (kk & 3) * 32, 16, 1024), idesc, kk > 0 ? 1u : 0u);
          umma_commit(&bars->s_full[b]);
          umma_commit(&bars->empty[slot]);
          if (j == tiles) umma_commit(&bars->list_empty[list & 1]);
        }
        __syncwarp();
      }
    }
  } else {
    const uint32_t lane_addr = static_cast<uint32_t>(warp * 32) << 16;
    const Wide x{tmem + lane_addr, tmem + lane_addr + C::TM_WO, w_weights, w_values, &own, abort_flag, tid, warp, lane, engine, at};
#pragma unroll 1
    for (int t = 0, list = 0;; ++list) {
      const int q = list & 1;
      ok = wait(&bars->list_full[q], (list >> 1) & 1, abort_flag, a.err, ERR_WAIT_OTHER, lane) && ok;
      if (any_of_128(!ok, engine)) break;                 // (all warps or none)
      const Item& w = own.item[q];              // (not a copy: the registers are for scores)
      if (w.tiles == 0) break;
      ok = w.n <= 8 ? wide_list<D, 8>(x, lists, a, w, t) : w.n <= 16 ? wide_list<D, 16>(x, lists, a, w, t) : wide_list<D, 32>(x, lists, a, w, t);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->list_empty[q]);
    }
  }
  if (blockIdx.x == gridDim.x - 1) write_plan(lists, a);
  let_copies_land(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP && engine == 0) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::ENGINES * C::TM_COLS);
  }
}

// A CTA a (place, key head), a warp a query: the pieces of its group's list and of its row's.  Bound by latency: what does not come from the first kernel is read before it ends.
template <int D>
__global__ void __launch_bounds__(128) join_pieces_kernel(const __grid_constant__ Args a, int engines) {
  constexpr int EACH = D / 32;                    // a lane's neighbouring columns
  const int place = blockIdx.x, hk = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = a.order[place];
  const bool there = row >= 0 && row < a.rows, rests = !there || a.lengths[row] <= 0;
  const long long all = static_cast<long long>(a.rows) * a.heads, wide0 = 2 * all + static_cast<long long>(engines) * 2 * BM;
  float sink = a.sinks != nullptr && warp < a.ratio ? a.sinks[hk * a.ratio + warp] * LOG2E : -INFINITY;
  if (hk == 0)                                    // (a row that `order` names twice, and another that it leaves out)
    for (int i = threadIdx.x; i < a.rows; i += blockDim.x)
      if (i != place && a.order[i] == row) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
  griddep_wait();
  if (!there) return;
  const int4 lists = a.plan[2 * place], group = a.plan[2 * place + 1];
  const bool tall = group.y > 0;
#pragma unroll 1
  for (int h = warp; h < a.ratio; h += 4) {
    const int head = hk * a.ratio + h;
    const long long one = static_cast<long long>(row) * a.heads + head;
    if (h > warp && a.sinks != nullptr) sink = a.sinks[head] * LOG2E;
    float top = sink, sum = top > -INFINITY ? 1.f : 0.f, o[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) o[i] = 0.f;
    bool finished = false;
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      const int n = rests ? 0 : k == 0 ? lists.y : lists.w;
      if (n == 0) continue;
      // the list's first tile in its sequence, units an engine, the queries' places in an engine's piece
      int start, per, step;
      long long at;
      if (k == 0) {
        const int x = (place - group.x) * a.ratio + h, pieces = (group.y + BM - 1) / BM;
        start = lists.x + (tall ? (hk * pieces + x / BM) * (n + TALL_GAP) + TALL_GAP : hk * (n + SHARED_GAP) + SHARED_GAP);
        per = tall ? group.z : group.w;
        step = tall ? BM : WN;
        at = tall ? 2 * all + x % BM : wide0 + x;
      } else {
        const int c = h / WN;
        start = lists.z + (hk * a.chunks + c) * (n + WIDE_GAP) + WIDE_GAP;
        per = group.w;
        step = WN;
        at = wide0 + h - c * WN;
      }
      const int c0 = start / per, c1 = (start + n - 1) / per;
      finished = k == 1 && lists.y == 0 && c0 == c1;
      if (finished) break;
#pragma unroll 2
      for (int c = c0; c <= c1; ++c) {
        const long long from = c0 == c1 ? k * all + one : at + (2ll * c + (c == c0 ? 1 : 0)) * step;
        const float2 ml = a.ml[from];
        float v[EACH];
        const float* p = a.acc + from * D + lane * EACH;
        if constexpr (EACH == 2) {
          const float2 x = *reinterpret_cast<const float2*>(p);
          v[0] = x.x; v[1] = x.y;
        } else {
#pragma unroll
          for (int i = 0; i < EACH; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(p + i);
            v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
          }
        }
        // (nothing but scores of minus infinity: nothing to add, unless none was a number)
        const float m = fmaxf(top, ml.x), was = top > -INFINITY ? fast_exp2(top - m) : 0.f, is = ml.x > -INFINITY ? fast_exp2(ml.x - m) : 0.f;
        sum = ml.y != ml.y ? ml.y : sum * was + ml.y * is;
#pragma unroll
        for (int i = 0; i < EACH; ++i) o[i] = o[i] * was + (is > 0.f ? v[i] * is : 0.f);
        top = m;
      }
    }
    if (finished) continue;
    const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    uint32_t w[EACH / 2];
#pragma unroll
    for (int i = 0; i < EACH; i += 2) w[i / 2] = pack_bf16(o[i] * by, o[i + 1] * by);
    __nv_bfloat16* to = a.out + one * D + lane * EACH;
    if constexpr (EACH == 2) *reinterpret_cast<uint32_t*>(to) = w[0];
    else if constexpr (EACH == 4) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
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

static bool room_allowed[3][64];                  // whether a device has been asked for the first kernel's shared memory

template <int D>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int engines, cudaStream_t stream) {
  using C = Cfg<D>;
  static_assert(sizeof(Own) % 16 == 0 && alignof(Own) == 16 && offsetof(Own, top) % 16 == 0 && C::ENGINE % 1024 == 0, "the maxima are read four at a time");
  constexpr int SMEM = C::ENGINES * (C::ENGINE + static_cast<int>(sizeof(Own))) + static_cast<int>(sizeof(Lists));
  static_assert(SMEM <= 227 * 1024, "over an SM's shared memory");
  if (engines % C::ENGINES != 0) return -3;
  constexpr int kind = D == 64 ? 0 : D == 128 ? 1 : 2;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev >= 64 || !room_allowed[kind][dev]) {
    if ((e = cudaFuncSetAttribute(shared_mma_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM)) != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) room_allowed[kind][dev] = true;
  }
  shared_mma_kernel<D><<<engines / C::ENGINES, THREADS * C::ENGINES, SMEM, stream>>>(tk, tv, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows, a.kv_heads);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, join_pieces_kernel<D>, a, engines));
}

}  // namespace sharedmma
}  // namespace dewb

// Engines of the first kernel on the current device.
extern "C" int dewb_shared_mma_engines(int D) { return dewb::sharedmma::multiprocessors() * (D == 256 ? 1 : 2); }

// As dewb_shared_decode, on the tensor cores: bf16, D 64, 128 or 256, page_size a multiple of 16, up to 448 rows and as many groups, everything 16-byte aligned and q_stride a
// multiple of 8.  acc: (2 rows heads + 320 engines) D floats; ml: as many pairs; plan: 8 rows integers on a 16-byte boundary.  An engine takes at least `least` tiles of 128 keys; engines: as dewb_shared_mma_engines has it.  Two launches.
extern "C" int dewb_shared_decode_mma(const void* q, long long q_stride, const void* k, const void* v, const int* table, const int* lengths, const int* order, const int* first,
                                      const int* tokens, const float* sinks, float* acc, void* ml, void* plan, void* out, int rows, int heads, int kv_heads, int D, int page_size,
                                      int max_pages, int pages, int groups, int window, int least, int engines, float scale, float cap, int* err, void* stream_ptr) {
  using namespace dewb::sharedmma;
  if (rows <= 0) return 0;
  const long long most = static_cast<long long>(max_pages) * page_size, chunks = heads > 0 && kv_heads > 0 ? (heads / kv_heads + WN - 1) / WN : 1;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || page_size <= 0 || page_size % 16 != 0 || max_pages <= 0 || pages <= 0 || groups <= 0 || groups > MOST_ROWS ||
      rows > MOST_ROWS || window < 0 || least < 1 || engines < 1 || most > 0x3fffffffll || static_cast<long long>(pages) * page_size > 0x7fffff00ll || kv_heads > 65535 ||
      (2ll * rows * chunks + groups) * kv_heads * ((most + BN - 1) / BN + 1 + TALL_GAP) > 0x3fffffffll || q_stride % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(acc) |
        reinterpret_cast<uintptr_t>(plan)) & 15))
    return -3;
  const int box = page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : 16;
  CUtensorMap tk, tv;
  int r;
  const uint64_t cols = static_cast<uint64_t>(kv_heads) * D, tall = static_cast<uint64_t>(pages) * page_size;
  if ((r = dewb::make_tmap_2d(&tk, k, tall, cols, cols, box, 64, 2, true))) return 1000 + r;
  if ((r = dewb::make_tmap_2d(&tv, v, tall, cols, cols, box, 64, 2, true))) return 2000 + r;
  const Args a{reinterpret_cast<const __nv_bfloat16*>(q), q_stride, table, lengths, order, first, tokens, sinks, reinterpret_cast<__nv_bfloat16*>(out), acc,
               reinterpret_cast<float2*>(ml), reinterpret_cast<int4*>(plan), rows, heads, kv_heads, heads / kv_heads, static_cast<int>(chunks), page_size, box, max_pages, pages, groups, window, least, scale * LOG2E, cap * LOG2E, err};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (D == 64) return launch<64>(tk, tv, a, engines, stream);
  if (D == 128) return launch<128>(tk, tv, a, engines, stream);
  if (D == 256) return launch<256>(tk, tv, a, engines, stream);
  return -3;
}
