// A decode step of rows that share prefixes, for any types and widths: fp32 or bf16 queries, pools in fp32, bf16, int8 or fp8, heads of up to 256.
//
//   o[r, h] = sum_n p_n v_n,   p = softmax of cap(scale q[r, h] . k_n) over the keys that row r sees (a sink joins the denominator)
//
// A group's shared keys (shared_range.cuh) are read once for up to 16 (row, head) queries that share a key head, a row's own keys for its heads.  A softmax over a union of
// key sets is put together from the sets' maxima m, sums l and weighted values a:  o = sum_i 2^(m_i - M) a_i / sum_i 2^(m_i - M) l_i,  M = max m_i.  So each CTA writes
// (m, l, a) of its part of the keys, and a second kernel joins a row's parts.
//
// grid = (place in `order`, key head x sixteens of its query heads, part): parts [0, splits) are of the shared keys, [splits, 2 splits) of the row's own.  A place that does
// not start a tile of the shared queries leaves at once.  Per 32 keys: keys and values to shared memory as fp32, scores with a lane a key, values with a lane every 32nd
// column; a warp whose queries do not exist only fetches.  This is the form for types and widths that the tensor cores' kernel does not take, bound by the chain of a tile's loads,
// scores and values and by what goes through shared memory (128 fp32 rows of 700 to 1000 keys, 8 heads of 64: 350 us, 1.3 TB/s; 24 rows of 500 keys, 6 heads over 2 of 80: 30 us).
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../common/ptx.cuh"
#include "../common/shared_range.cuh"

namespace dewb {
namespace sharedprefix {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int QUERIES = 16, EACH = QUERIES / WARPS;      // a tile's queries, a warp's
constexpr int KEYS = 32;
constexpr int MOST_D = 256;
constexpr uint32_t FULL = 0xffffffffu;

enum : int { POOL_SAME = 0, POOL_INT8 = 1, POOL_FP8 = 2 };   // (POOL_SAME: the queries' type)

struct Args {
  const void *q, *k, *v;
  const float *k_scale, *v_scale, *sinks;
  const int *table, *lengths, *order, *first, *tokens;
  float *part_m, *part_l, *part_acc;                     // [2 splits, rows * heads], [2 splits, rows * heads, D]
  void* out;
  long long q_stride;
  int rows, heads, kv_heads, D, page_size, max_pages, pages, groups, splits, window;
  float scale, cap;
  int* err;
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(int8_t x) { return static_cast<float>(x); }
__device__ __forceinline__ float as_float(__nv_fp8_e4m3 x) { return static_cast<float>(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16(x); }

// the group whose places hold `at`: the last one that begins at it or before (empty ones in front of it are passed over)
__device__ __forceinline__ int group_of(const int* __restrict__ first, int groups, int at) {
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= at) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename TQ, typename TP, bool SCALED>
__global__ void __launch_bounds__(THREADS) shared_prefix_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) float smem[];
  const int D = a.D, wide = D + 1;
  float* sq = smem;                                      // [QUERIES][D]
  float* sk = sq + QUERIES * D;                          // [KEYS][D + 1]
  float* sv = sk + KEYS * wide;                          // [KEYS][D]
  float* sp = sv + KEYS * D;                             // [KEYS][QUERIES]
  __shared__ long long stok[2][KEYS];                    // where keys stand in the pools (-1: nowhere), of this tile and the next one
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ratio = a.heads / a.kv_heads, chunks = (ratio + QUERIES - 1) / QUERIES;
  const int at = blockIdx.x, hk = blockIdx.y / chunks, chunk = blockIdx.y % chunks;
  const int head0 = hk * ratio + chunk * QUERIES, heads = min(QUERIES, ratio - chunk * QUERIES);
  const bool shared = static_cast<int>(blockIdx.z) < a.splits;
  const int split = shared ? blockIdx.z : blockIdx.z - a.splits;
  const int g = group_of(a.first, a.groups, at);
  const int begin = max(0, a.first[g]), end = min(a.rows, a.first[g + 1]);
  if (at < begin || at >= end) {                         // (a place that no group holds: its row is reported, and sees nothing)
    if (tid == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
    const int row = a.order[at];
    if (tid < heads && row >= 0 && row < a.rows) {
      const long long to_part = (static_cast<long long>(blockIdx.z) * a.rows + row) * a.heads + head0 + tid;
      a.part_m[to_part] = -INFINITY;
      a.part_l[to_part] = 0.f;
    }
    return;
  }
  const int together = shared ? max(1, QUERIES / heads) : 1;
  if (shared && (at - begin) % together != 0) return;
  const int n_rows = min(together, end - at), n = n_rows * heads;
  const int most = a.max_pages * a.page_size;
  const SharedRange both = shared_range(a.lengths, a.order, begin, end, a.rows, a.tokens[g], a.window, most, lane);
  const int row0 = a.order[at];
  if (row0 < 0 || row0 >= a.rows) { if (tid == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG)); return; }
  // this part's keys, counted from 0: [first, gap) and, behind `skip` others, the rest
  const int len = row_length(a.lengths, row0, most);
  if (tid == 0 && a.lengths[row0] > most) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
  const int first = shared ? both.lo : row_first(len, a.window);
  const int gap = shared || both.hi == 0 ? 0x7fffffff : both.lo;
  const int skip = shared || both.hi == 0 ? 0 : both.hi - both.lo;
  const int keys = shared ? both.hi - both.lo : max(0, len - first - skip);
  const int per = ((keys + a.splits - 1) / a.splits + KEYS - 1) / KEYS * KEYS;
  const int from = split * per, to = min(keys, from + per);
  // queries of the tile: number i is of row order[at + i / heads], head head0 + i % heads
  auto row_of = [&](int i) { return a.order[at + i / heads]; };
  for (int i = tid; i < QUERIES * D; i += THREADS) {
    const int x = i / D, d = i - x * D;
    const int row = x < n ? row_of(x) : -1;
    sq[i] = row >= 0 && row < a.rows ? as_float(static_cast<const TQ*>(a.q)[row * a.q_stride + static_cast<long long>(head0 + x % heads) * D + d]) : 0.f;
  }
  float m[EACH], l[EACH], acc[EACH][MOST_D / 32];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < MOST_D / 32; ++c) acc[i][c] = 0.f;
  }
  // (the shared pages are read through the first row that holds anything: a resting row's table may say nothing)
  int through = row0;
  if (shared)
    for (int i = begin; i < end; ++i) {
      const int row = a.order[i];
      if (row >= 0 && row < a.rows && a.lengths[row] > 0) { through = row; break; }
    }
  const int* table = a.table + static_cast<long long>(through) * a.max_pages;
  const float scale2 = a.scale * 1.4426950408889634f, cap2 = a.cap * 1.4426950408889634f;
  auto look_up = [&](int k0, int b) {                    // (a thread a key)
    const int x = first + k0 + tid, key = x < gap ? x : x + skip;
    long long tok = -1;
    if (k0 + tid < to) {
      const int page = table[key / a.page_size];
      if (page >= 0 && page < a.pages) tok = static_cast<long long>(page) * a.page_size + key % a.page_size;
      else atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
    }
    stok[b][tid] = tok;
  };
  if (tid < KEYS) look_up(from, 0);
  int b = 0;
  for (int k0 = from; k0 < to; k0 += KEYS, b ^= 1) {
    __syncthreads();
    if (tid < KEYS && k0 + KEYS < to) look_up(k0 + KEYS, b ^ 1);
    // a warp every fourth key, a lane every 32nd column: eight keys' loads are on their way at a time
    for (int d = lane; d < D; d += 32) {
      float kx[KEYS / WARPS], vx[KEYS / WARPS];
#pragma unroll
      for (int e = 0; e < KEYS / WARPS; ++e) {
        const long long tok = stok[b][e * WARPS + warp], x = (tok * a.kv_heads + hk) * D + d;
        kx[e] = tok >= 0 ? as_float(static_cast<const TP*>(a.k)[x]) : 0.f;
        vx[e] = tok >= 0 ? as_float(static_cast<const TP*>(a.v)[x]) : 0.f;
        if (SCALED && tok >= 0) { kx[e] *= a.k_scale[tok * a.kv_heads + hk]; vx[e] *= a.v_scale[tok * a.kv_heads + hk]; }
      }
#pragma unroll
      for (int e = 0; e < KEYS / WARPS; ++e) {
        sk[(e * WARPS + warp) * wide + d] = kx[e];
        sv[(e * WARPS + warp) * D + d] = vx[e];
      }
    }
    __syncthreads();
    if (warp * EACH >= n) continue;                      // (no queries for this warp)
    const bool seen = stok[b][lane] >= 0;
    float s[EACH], weights[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) s[i] = 0.f;
    const float* mine = sq + warp * EACH * D;
    int d = 0;
    if (D % 4 == 0)                                      // (queries four columns at a time)
      for (; d < D; d += 4) {
        float kx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) kx[e] = sk[lane * wide + d + e];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const float4 qx = *reinterpret_cast<const float4*>(mine + i * D + d);
          s[i] = fmaf(qx.w, kx[3], fmaf(qx.z, kx[2], fmaf(qx.y, kx[1], fmaf(qx.x, kx[0], s[i]))));
        }
      }
    for (; d < D; ++d) {
      const float kx = sk[lane * wide + d];
#pragma unroll
      for (int i = 0; i < EACH; ++i) s[i] = fmaf(mine[i * D + d], kx, s[i]);
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      float x = s[i] * scale2;
      if (cap2 > 0.f) x = cap2 * tanhf(x / cap2);
      x = seen ? x : -INFINITY;
      float top = x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
      const float m_new = fmaxf(m[i], top);
      const float by = m[i] == -INFINITY ? 0.f : exp2f(m[i] - m_new);
      const float p = exp2f(x - (m_new == -INFINITY ? 0.f : m_new));       // (a score that is no number is no maximum, and shows in the sum)
      float sum = p;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
      l[i] = l[i] * by + sum;
      m[i] = m_new;
#pragma unroll
      for (int c = 0; c < MOST_D / 32; ++c) acc[i][c] *= by;
      weights[i] = p;
    }
    static_assert(EACH == 4, "a key's weights are one 16-byte word a warp");
    *reinterpret_cast<float4*>(sp + lane * QUERIES + warp * EACH) = make_float4(weights[0], weights[1], weights[2], weights[3]);
    __syncwarp();
    for (int j = 0; j < KEYS; ++j) {
      const float4 word = *reinterpret_cast<const float4*>(sp + j * QUERIES + warp * EACH);
      const float p[EACH] = {word.x, word.y, word.z, word.w};
#pragma unroll
      for (int c = 0; c < MOST_D / 32; ++c) {
        const int d = c * 32 + lane;
        if (d < D) {
          const float vx = sv[j * D + d];
#pragma unroll
          for (int i = 0; i < EACH; ++i) acc[i][c] = fmaf(p[i], vx, acc[i][c]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int x = warp * EACH + i;
    if (x >= n) continue;
    const int row = row_of(x);
    if (row < 0 || row >= a.rows) continue;
    const long long to_part = (static_cast<long long>(blockIdx.z) * a.rows + row) * a.heads + head0 + x % heads;
    // a row that rests is in the tile, and sees none of it
    const bool rests = a.lengths[row] <= 0;
    if (lane == 0) { a.part_m[to_part] = rests ? -INFINITY : m[i]; a.part_l[to_part] = rests ? 0.f : l[i]; }
#pragma unroll
    for (int c = 0; c < MOST_D / 32; ++c)
      if (c * 32 + lane < D) a.part_acc[to_part * D + c * 32 + lane] = acc[i][c];
  }
  // (groups that begin behind their end; asked last, by CTAs that every place has: asked first, 24 rows took 35 us instead of 33)
  if (tid == 0 && blockIdx.y == 0 && split == 0 && !shared)
    for (int i = at; i < a.groups; i += a.rows)
      if (a.first[i] > a.first[i + 1]) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
}

// One CTA a (row, head): its parts joined.
template <typename TQ>
__global__ void __launch_bounds__(64) join_parts_kernel(const __grid_constant__ Args a) {
  const int row = blockIdx.x, head = blockIdx.y;
  if (head == 0) {                                       // (a row that `order` names twice, and another that it leaves out)
    int times = 0;
    for (int i = threadIdx.x; i < a.rows; i += blockDim.x) times += a.order[i] == row;
    if (__syncthreads_count(times > 0) != 1 || __syncthreads_or(times > 1))
      if (threadIdx.x == 0) atomicCAS(a.err, 0, static_cast<int>(ERR_BAD_ARG));
  }
  const long long one = static_cast<long long>(row) * a.heads + head, step = static_cast<long long>(a.rows) * a.heads;
  const float sink = a.sinks != nullptr ? a.sinks[head] * 1.4426950408889634f : -INFINITY;
  float top = sink;
  for (int p = 0; p < 2 * a.splits; ++p) top = fmaxf(top, a.part_m[p * step + one]);
  float sum = sink > -INFINITY ? exp2f(sink - top) : 0.f;
  for (int p = 0; p < 2 * a.splits; ++p) {
    const float m = a.part_m[p * step + one];
    const float l = a.part_l[p * step + one];
    if (m > -INFINITY) sum += l * exp2f(m - top);
    else if (l != l) sum = l;                            // (no score that is a number)
  }
  for (int d = threadIdx.x; d < a.D; d += 64) {
    float x = 0.f;
    for (int p = 0; p < 2 * a.splits; ++p) {
      const float m = a.part_m[p * step + one];
      if (m > -INFINITY) x += a.part_acc[(p * step + one) * a.D + d] * exp2f(m - top);
    }
    put(static_cast<TQ*>(a.out) + one * a.D + d, sum > 0.f || sum != sum ? x / sum : 0.f);
  }
}

template <typename TQ, typename TP, bool SCALED>
int launch(const Args& a, cudaStream_t stream) {
  const int smem = static_cast<int>(sizeof(float)) * (QUERIES * a.D + KEYS * (2 * a.D + 1) + QUERIES * KEYS);
  cudaError_t e = cudaFuncSetAttribute(shared_prefix_kernel<TQ, TP, SCALED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int ratio = a.heads / a.kv_heads;
  const dim3 grid(a.rows, a.kv_heads * ((ratio + QUERIES - 1) / QUERIES), 2 * a.splits);
  shared_prefix_kernel<TQ, TP, SCALED><<<grid, THREADS, smem, stream>>>(a);
  join_parts_kernel<TQ><<<dim3(a.rows, a.heads), 64, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace sharedprefix
}  // namespace dewb

// q [rows, heads, D] (rows q_stride elements apart), pools [pages, page_size, kv_heads, D] (`pool`: 0 of q's type, 1 int8, 2 fp8 e4m3, with fp32 scales [pages, page_size,
// kv_heads]), table int32 [rows, max_pages], lengths int32 [rows]; group g: rows order[first[g], first[g + 1]), whose first tokens[g] keys are the same pages.  part_m,
// part_l: 2 splits x rows x heads floats, part_acc: D times as many.  Two launches.
extern "C" int dewb_shared_decode(const void* q, long long q_stride, const void* k, const void* v, const float* k_scale, const float* v_scale, const int* table,
                                  const int* lengths, const int* order, const int* first, const int* tokens, const float* sinks, float* part_m, float* part_l,
                                  float* part_acc, void* out, int rows, int heads, int kv_heads, int D, int page_size, int max_pages, int pages, int groups, int splits,
                                  int window, float scale, float cap, int fp32, int pool, int* err, void* stream_ptr) {
  using namespace dewb::sharedprefix;
  if (rows <= 0) return 0;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || D <= 0 || D > MOST_D || page_size <= 0 || max_pages <= 0 || pages <= 0 || groups <= 0 || splits < 1 ||
      splits > 1024 || window < 0 || static_cast<long long>(max_pages) * page_size > 0x3fffffffll || heads > 65535 ||
      (pool != POOL_SAME && (k_scale == nullptr || v_scale == nullptr)))
    return -3;
  const Args a{q, k, v, k_scale, v_scale, sinks, table, lengths, order, first, tokens, part_m, part_l, part_acc, out, q_stride, rows, heads, kv_heads, D, page_size,
               max_pages, pages, groups, splits, window, scale, cap, err};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (pool == POOL_SAME) return fp32 ? launch<float, float, false>(a, stream) : launch<__nv_bfloat16, __nv_bfloat16, false>(a, stream);
  if (pool == POOL_INT8) return fp32 ? launch<float, int8_t, true>(a, stream) : launch<__nv_bfloat16, int8_t, true>(a, stream);
  if (pool == POOL_FP8) return fp32 ? launch<float, __nv_fp8_e4m3, true>(a, stream) : launch<__nv_bfloat16, __nv_fp8_e4m3, true>(a, stream);
  return -3;
}
