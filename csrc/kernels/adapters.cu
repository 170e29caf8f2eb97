// Low-rank adapters of many requests beside one projection:  y_t += s_i B_i (A_i x_t),  i the adapter of token t (below 0: none).
//
// For any types and sizes: a CTA a (token, part of the width) makes its share of A_i x in fp32, then a CTA a (token, 128 columns) adds the shares and multiplies by B_i.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

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
