// Pages of a cache copied to other pages of the same pools, and page tables rewritten: what a fork of a row, or a compaction of the pool, does to the device.
//
//   pool[l, dst[i]] = pool[l, src[i]]   for every pool, layer l and copy i;    table[at[j] + x] = pages[j][x]   for every span j
//
// One launch for all layers and pools (keys, values, scales).  The page numbers are known to the host, which keeps the ledger, so they travel in the kernel's
// parameters: nothing is copied to the device in front of the launch, and no buffer has to outlive it.  No page is both read and written and none is written twice (the
// entry refuses), so the copies need no order among themselves.
//
// Bound by the copy: a page is read once and written as often as it is copied.  A block moves 1024 pieces of 16 bytes, four a thread with all four loads in flight, counted
// through the sources of one layer without regard to where a page ends: pages of 4 KB fill blocks as those of 128 KB do.  Copies of one page that follow one another are a
// run, whose source is loaded once (seven copies each of 16 pages of 128 KB in 16 layers, keys and values: 91 us, loaded once a copy 107).
#include <cstdint>
#include <cstdlib>
#include <cuda_runtime.h>

namespace dewb {
namespace pagemoves {

constexpr int THREADS = 256, EACH = 4, BLOCK = THREADS * EACH;   // pieces a block
constexpr int MOST_POOLS = 32;
constexpr int FEW = 768, MANY = 7680;                           // integers that travel with a launch (a kernel's parameters end at 32764 bytes)

struct Pool {
  void* base;
  long long layer_stride;        // bytes
  int layers, page_bytes;
};

// data: `runs` sources; where runs < copies, runs + 1 places of the runs' first destinations; `copies` destinations; from `tail` on `spans` offsets into the table, spans + 1
// places in what follows, the spans' pages
template <int N>
struct Moves {
  Pool pool[MOST_POOLS];
  int first[MOST_POOLS + 1];     // first block of each pool; the blocks behind the last write the table
  int pools, copies, runs, tail, spans;
  int* table;
  int data[N];
};
static_assert(sizeof(Moves<MANY>) <= 32764, "over what a kernel's parameters may hold");

// widest piece that divides a page and the addresses of a pool
__host__ __device__ inline int piece_bytes(const Pool& p) {
  const unsigned long long all = reinterpret_cast<unsigned long long>(p.base) | static_cast<unsigned long long>(p.layer_stride) | static_cast<unsigned>(p.page_bytes);
  return (all & 15) == 0 ? 16 : (all & 3) == 0 ? 4 : (all & 1) == 0 ? 2 : 1;
}

template <typename T, int N>
__device__ __forceinline__ void copy_block(const Moves<N>& m, const Pool& p, int block) {
  const int per_page = p.page_bytes / static_cast<int>(sizeof(T));
  const long long units = static_cast<long long>(m.runs) * per_page;
  const int per_layer = static_cast<int>((units + BLOCK - 1) / BLOCK);
  const int layer = block / per_layer;
  const long long u0 = static_cast<long long>(block - layer * per_layer) * BLOCK;
  const bool plain = m.runs == m.copies;
  const int *begin = m.data + m.runs, *dst = begin + (plain ? 0 : m.runs + 1);
  T* base = reinterpret_cast<T*>(static_cast<char*>(p.base) + layer * p.layer_stride);
  T v[EACH];
  int run[EACH], at[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const long long u = u0 + i * THREADS + threadIdx.x;
    run[i] = -1;
    if (u >= units) continue;
    run[i] = static_cast<int>(u / per_page);
    at[i] = static_cast<int>(u - static_cast<long long>(run[i]) * per_page);
    v[i] = base[static_cast<long long>(m.data[run[i]]) * per_page + at[i]];
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (run[i] < 0) continue;
    const int end = plain ? run[i] + 1 : begin[run[i] + 1];
    for (int c = plain ? run[i] : begin[run[i]]; c < end; ++c) base[static_cast<long long>(dst[c]) * per_page + at[i]] = v[i];
  }
}

template <int N>
__global__ void __launch_bounds__(THREADS) move_pages_kernel(const __grid_constant__ Moves<N> m) {
  const int block = blockIdx.x;
  if (block >= m.first[m.pools]) {
    const int e = (block - m.first[m.pools]) * THREADS + threadIdx.x;
    const int *at = m.data + m.tail, *begin = at + m.spans, *pages = begin + m.spans + 1;
    if (e >= begin[m.spans]) return;
    int lo = 0, hi = m.spans;                                  // the last span that begins at e or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (begin[mid] <= e) lo = mid; else hi = mid;
    }
    m.table[at[lo] + e - begin[lo]] = pages[e];
    return;
  }
  int i = 0;
  while (block >= m.first[i + 1]) ++i;
  const Pool p = m.pool[i];
  switch (piece_bytes(p)) {
    case 16: copy_block<uint4>(m, p, block - m.first[i]); break;
    case 4: copy_block<uint32_t>(m, p, block - m.first[i]); break;
    case 2: copy_block<uint16_t>(m, p, block - m.first[i]); break;
    default: copy_block<uint8_t>(m, p, block - m.first[i]);
  }
}

// One launch: copies [c0, c1) of the pools [p0, p1), and the next `entries` of the table: `pages`, in span s from its `done`-th entry on and in those behind it.
template <int N>
int launch(const Pool* pools, int p0, int p1, const int* src, const int* dst, int c0, int c1, int* table, int columns, const int* row, const int* first, const int* length,
           const int* pages, int s, int done, int entries, cudaStream_t stream) {
  Moves<N> m;
  m.pools = p1 - p0;
  m.copies = c1 - c0;
  m.runs = 0;
  for (int c = c0; c < c1; ++c) m.runs += c == c0 || src[c] != src[c - 1];
  if (2 * m.runs >= m.copies) m.runs = m.copies;               // (there is room for the runs' places where there are fewer than half as many)
  m.table = table;
  long long blocks = 0;
  for (int i = 0; i < m.pools; ++i) {
    m.pool[i] = pools[p0 + i];
    m.first[i] = static_cast<int>(blocks);
    const long long units = static_cast<long long>(m.runs) * (m.pool[i].page_bytes / piece_bytes(m.pool[i]));
    blocks += (units + BLOCK - 1) / BLOCK * m.pool[i].layers;
    if (blocks > 0x7fff0000ll) return -3;
  }
  m.first[m.pools] = static_cast<int>(blocks);
  int* to = m.data;
  if (m.runs == m.copies) {
    for (int c = c0; c < c1; ++c) *to++ = src[c];
  } else {
    int* begin = to + m.runs;
    for (int c = c0; c < c1; ++c)
      if (c == c0 || src[c] != src[c - 1]) {
        *to++ = src[c];
        *begin++ = c - c0;
      }
    *begin++ = m.copies;
    to = begin;
  }
  for (int c = c0; c < c1; ++c) *to++ = dst[c];
  m.tail = static_cast<int>(to - m.data);
  m.spans = 0;
  for (int e = 0, i = s, d = done; e < entries; ++i, d = 0)
    if (length[i] > d) {
      *to++ = row[i] * columns + first[i] + d;
      e += length[i] - d;
      ++m.spans;
    }
  for (int e = 0, i = s, d = done; e < entries; ++i, d = 0)
    if (length[i] > d) {
      *to++ = e;
      e += length[i] - d;
    }
  *to++ = entries;
  for (int e = 0; e < entries; ++e) *to++ = pages[e];
  blocks += (entries + THREADS - 1) / THREADS;
  if (blocks == 0) return 0;
  move_pages_kernel<N><<<static_cast<int>(blocks), THREADS, 0, stream>>>(m);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace pagemoves
}  // namespace dewb

namespace {
struct Ends { long long from, to; };
int by_from(const void* a, const void* b) {
  const long long x = static_cast<const Ends*>(a)->from, y = static_cast<const Ends*>(b)->from;
  return x < y ? -1 : x > y;
}
}  // namespace

// What is wrong with the copies and spans: 0 nothing, -11 a page outside the pool, -12 a page written twice, -13 a page read and written, -14 an entry outside the table,
// -15 no memory to look, -16 an entry written twice.  Host only.  Span s writes length[s] entries of row[s] from column first[s] on.
extern "C" int dewb_check_moves(const int* src, const int* dst, int copies, int pages_in_pool, const int* row, const int* first, const int* length, const int* pages, int spans,
                                int rows, int columns) {
  if (copies < 0 || spans < 0 || pages_in_pool < 0) return -3;
  unsigned char* seen = static_cast<unsigned char*>(std::calloc(pages_in_pool > 0 ? pages_in_pool : 1, 1));
  if (seen == nullptr) return -15;
  int rc = 0;
  for (int i = 0; i < copies && rc == 0; ++i) {
    if (src[i] < 0 || src[i] >= pages_in_pool || dst[i] < 0 || dst[i] >= pages_in_pool) rc = -11;
    else if (seen[dst[i]]) rc = -12;
    else seen[dst[i]] = 1;
  }
  for (int i = 0; i < copies && rc == 0; ++i)
    if (seen[src[i]]) rc = -13;
  std::free(seen);
  long long n = 0;
  for (int s = 0; s < spans && rc == 0; ++s) {
    if (length[s] < 0 || row[s] < 0 || row[s] >= rows || first[s] < 0 || first[s] > columns - length[s]) { rc = -14; break; }
    for (int e = 0; e < length[s] && rc == 0; ++e)
      if (pages[n + e] < 0 || pages[n + e] >= pages_in_pool) rc = -11;
    n += length[s];
  }
  if (rc != 0 || spans < 2) return rc;
  if (n > 0x7fffffffll) return -3;
  Ends* ends = static_cast<Ends*>(std::malloc(sizeof(Ends) * spans));
  if (ends == nullptr) return -15;
  int used = 0;
  bool sorted = true;
  for (int s = 0; s < spans; ++s) {
    if (length[s] == 0) continue;
    const long long at = static_cast<long long>(row[s]) * columns + first[s];
    ends[used] = {at, at + length[s]};
    sorted = sorted && (used == 0 || ends[used - 1].from <= at);
    ++used;
  }
  if (!sorted) std::qsort(ends, used, sizeof(Ends), by_from);
  for (int i = 1; i < used && rc == 0; ++i)
    if (ends[i].from < ends[i - 1].to) rc = -16;
  std::free(ends);
  return rc;
}

// `pools`: layers x pages_in_pool pages of page_bytes each, one behind another within a layer; `table`: int32 [rows, columns].  All lists are the host's and are read before
// this returns.  One launch for up to 32 pools and what fits the parameters, more where there is more.  `launches` counts them.
extern "C" int dewb_move_pages(const void* pools_ptr, int pools, int pages_in_pool, const int* src, const int* dst, int copies, int* table, int rows, int columns, const int* row,
                               const int* first, const int* length, const int* pages, int spans, int* launches, void* stream_ptr) {
  using namespace dewb::pagemoves;
  *launches = 0;
  const Pool* pool = static_cast<const Pool*>(pools_ptr);
  int rc = static_cast<long long>(rows) * columns > 0x7fffffffll ? -3 : dewb_check_moves(src, dst, copies, pages_in_pool, row, first, length, pages, spans, rows, columns);
  if (rc != 0) return rc;
  for (int i = 0; i < pools; ++i)
    if (pool[i].layers < 0 || pool[i].page_bytes < 0) return -3;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  // the table's entries go with the first launch that has room for them: span s, of which `done` entries are written, comes next, and its pages begin at `named`
  int s = 0, done = 0, p = 0, c = 0;
  long long named = 0;
  bool copying = copies > 0 && pools > 0;
  while (s < spans && length[s] == 0) ++s;
  while (copying || s < spans) {
    int p1 = p, c1 = c, room = MANY - 1;
    if (copying) {
      p1 = pools - p < MOST_POOLS ? pools : p + MOST_POOLS;
      c1 = copies - c < room / 2 ? copies : c + room / 2;
      room -= 2 * (c1 - c);
    }
    const int s0 = s, done0 = done;
    const long long named0 = named;
    while (s < spans && room > 2) {
      const int take = length[s] - done < room - 2 ? length[s] - done : room - 2;
      room -= 2 + take;
      done += take;
      named += take;
      if (done < length[s]) break;
      done = 0;
      do ++s; while (s < spans && length[s] == 0);
    }
    const bool few = MANY - room <= FEW;
    rc = few ? launch<FEW>(pool, p, p1, src, dst, c, c1, table, columns, row, first, length, pages + named0, s0, done0, static_cast<int>(named - named0), stream)
             : launch<MANY>(pool, p, p1, src, dst, c, c1, table, columns, row, first, length, pages + named0, s0, done0, static_cast<int>(named - named0), stream);
    if (rc != 0) return rc;
    ++*launches;
    if (copying) {
      c = c1;
      if (c == copies) {
        p = p1;
        c = 0;
        copying = p < pools;
      }
    }
  }
  return 0;
}
