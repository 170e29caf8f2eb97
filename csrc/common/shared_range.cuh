// Rows of a decode step that share a prefix: which keys are attended to once for a whole group, and which by a row alone.
//
// A row at length len sees the keys [first, len), first = max(0, len - window).  Of a group with two or more rows that hold anything, the keys that ALL of those rows see and
// that lie in the shared pages, [lo, hi) = [max first, min(tokens, min len)), are the group's: no score of them is masked, for any row.  The others, [first, lo) and
// [hi, len), are the row's own.  What a row does not see is thereby never multiplied with anything of its own, whatever stands there.
#pragma once
#include <cuda_runtime.h>

namespace dewb {

struct SharedRange { int lo, hi; };

__device__ __forceinline__ int row_length(const int* __restrict__ lengths, int row, int most) { return min(max(lengths[row], 0), most); }
__device__ __forceinline__ int row_first(int len, int window) { return window > 0 && len > window ? len - window : 0; }

// One warp asks about the rows order[begin, end); every lane gets the answer.  `most`: keys that a row's table has room for.
__device__ __forceinline__ SharedRange shared_range(const int* __restrict__ lengths, const int* __restrict__ order, int begin, int end, int rows, int tokens, int window,
                                                    int most, int lane) {
  int lo = 0, hi = min(max(tokens, 0), most), live = 0;
  for (int i = begin + lane; i < end; i += 32) {
    const int row = order[i];
    const int len = row >= 0 && row < rows ? row_length(lengths, row, most) : 0;
    if (len == 0) continue;
    ++live;
    lo = max(lo, row_first(len, window));
    hi = min(hi, len);
  }
  lo = __reduce_max_sync(0xffffffffu, lo);
  hi = __reduce_min_sync(0xffffffffu, hi);
  live = __reduce_add_sync(0xffffffffu, live);
  return live > 1 && lo < hi ? SharedRange{lo, hi} : SharedRange{0, 0};
}

}  // namespace dewb
