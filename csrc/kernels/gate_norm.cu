// The norm behind a gate, for sm_100a:  u = x silu(z),  y = u r w,  r = 1 / sqrt(mean u^2 + eps), over rows of d values; and its gradients
//
//   g = dy w,   du = r g - u r^3 mean(g u),   dx = du silu(z),   dz = du x silu'(z),   dw = sum over rows of dy u r
//
// Bound by memory: a row's values are read once and stay in registers between the sums and the results (`ITEMS` pieces of V values a thread; ITEMS 0, for rows that are longer or lie
// askew, reads them again).  The backward forms r anew from what it reads anyway, in the same reduction as mean(g u), so the forward keeps nothing.  A row belongs to a warp (up to
// 32 V ITEMS values) or to a block of NT threads; in the backward a block walks rows with its columns' dw in registers, and its sums leave as one part, added up in one order by
// weight_sum_kernel.  There values stay as they lie in memory (half the registers in bf16) and the next row is on its way while one is summed.
// 8192 rows of 8192 bf16 values: forward 69 us (5.8 TB/s; with expf and a division, 91: issuing), backward 136 (4.9 TB/s; as fp32 values without the next row ahead, 272).  Two pieces
// a thread: with one (rows of 4096 and 512 threads) the barriers take their share, backward 120 us instead of 83.
// Values are bf16 or fp32 (template T; w either), sums fp32.  Compiled without fast math.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../common/rows.cuh"
#include "../common/special.cuh"

namespace dewb {
namespace gatenorm {

using namespace rows;
using special::gate;

constexpr int THREADS = 256, WARPS = 8;       // of rows that belong to a warp, and of what is read twice

__device__ __forceinline__ void st(float* p, float v) { *p = v; }
__device__ __forceinline__ void st(bf16* p, float v) { *p = __float2bfloat16(v); }

struct Args {
  const void *x, *z, *w, *dy;          // [rows, d]; x, z and dy at strides of their own
  long long x_row, z_row, dy_row, rows;
  int d, w_fp32;
  float eps;
  void *y, *dx, *dz;
  float* parts;                        // [blocks, d]
};

template <int V>
__device__ __forceinline__ void load_w(const Args& p, int c, float (&f)[V], const float*) { load_v<V>(static_cast<const float*>(p.w) + c, f); }
template <int V>
__device__ __forceinline__ void load_w(const Args& p, int c, float (&f)[V], const bf16*) {
  if (p.w_fp32) {
    if constexpr (V == 8) {
      float a[4], b[4];
      load_v<4>(static_cast<const float*>(p.w) + c, a);
      load_v<4>(static_cast<const float*>(p.w) + c + 4, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[4 + i] = b[i]; }
    } else {
      load_v<V>(static_cast<const float*>(p.w) + c, f);
    }
  } else {
    load_v<V>(static_cast<const bf16*>(p.w) + c, f);
  }
}

// The sums of two numbers over a row's threads.
template <bool WARP, int NT>
__device__ __forceinline__ float2 row_sum(float a, float b, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
  if (WARP) return make_float2(a, b);
  __syncthreads();                     // (the row before has been read)
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) { s.x += red[i].x; s.y += red[i].y; }
  return s;
}

template <typename T, int V, int ITEMS, bool WARP, int NT>
__global__ void __launch_bounds__(NT)
gate_norm_kernel(const Args p) {
  __shared__ float2 red[NT / 32];
  constexpr int N = WARP ? 32 : NT;
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  const long long row = WARP ? static_cast<long long>(blockIdx.x) * WARPS + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= p.rows) return;
  const T *x = static_cast<const T*>(p.x) + row * p.x_row, *z = static_cast<const T*>(p.z) + row * p.z_row;
  T* y = static_cast<T*>(p.y) + row * p.d;
  float kept[ITEMS > 0 ? ITEMS : 1][V];
  auto gated = [&](int c, float (&u)[V]) {
    float g[V];
    load_v<V>(x + c, u);
    load_v<V>(z + c, g);
#pragma unroll
    for (int j = 0; j < V; ++j) u[j] *= g[j] * gate<T>(g[j]);
  };
  float ss = 0.f;
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * N + lane) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) kept[i][j] = 0.f;
      if (c < p.d) gated(c, kept[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) ss += kept[i][j] * kept[i][j];
    }
  } else {
    for (int c = lane * V; c < p.d; c += N * V) {
      gated(c, kept[0]);
#pragma unroll
      for (int j = 0; j < V; ++j) ss += kept[0][j] * kept[0][j];
    }
  }
  const float r = 1.f / sqrtf(row_sum<WARP, NT>(ss, 0.f, red).x / p.d + p.eps);
  auto finish = [&](int c, float (&u)[V]) {
    float w[V];
    load_w<V>(p, c, w, static_cast<const T*>(nullptr));
#pragma unroll
    for (int j = 0; j < V; ++j) u[j] *= r * w[j];
    store_v<V>(y + c, u);
  };
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * N + lane) * V;
      if (c < p.d) finish(c, kept[i]);
    }
  } else {
    for (int c = lane * V; c < p.d; c += N * V) {
      gated(c, kept[0]);
      finish(c, kept[0]);
    }
  }
}

// V values as they lie in memory.
template <typename T, int V>
struct Raw {
  static constexpr int WORDS = V * sizeof(T) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    static_assert(WORDS == 4, "pieces of 16 bytes");
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0u; }
  __device__ __forceinline__ float operator[](int j) const {
    return sizeof(T) == 4 ? __uint_as_float(w[j]) : __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
};

// grid: blocks that walk the rows, with dw in registers.
template <typename T, int V, int ITEMS, bool WARP, int NT>
__global__ void __launch_bounds__(NT)
gate_norm_grad_kernel(const Args p) {
  __shared__ float2 red[NT / 32];
  __shared__ float add[WARP ? WARPS : 1][WARP ? 32 * V * ITEMS : 1];
  constexpr int N = WARP ? 32 : NT;
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  const long long step = static_cast<long long>(gridDim.x) * (WARP ? WARPS : 1);
  float* part = p.parts + static_cast<long long>(blockIdx.x) * p.d;
  float dw[ITEMS][V];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = 0.f;
  struct Row { Raw<T, V> x, z, dy; } now[ITEMS], next[ITEMS];
  auto bring = [&](Row (&r)[ITEMS], long long row) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * N + lane) * V;
      if (c < p.d && row < p.rows) {
        r[i].x.load(static_cast<const T*>(p.x) + row * p.x_row + c);
        r[i].z.load(static_cast<const T*>(p.z) + row * p.z_row + c);
        r[i].dy.load(static_cast<const T*>(p.dy) + row * p.dy_row + c);
      } else {
        r[i].x.zero(); r[i].z.zero(); r[i].dy.zero();
      }
    }
  };
  long long row = WARP ? static_cast<long long>(blockIdx.x) * WARPS + (threadIdx.x >> 5) : blockIdx.x;
  bring(next, row);
  for (; row < p.rows; row += step) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) now[i] = next[i];
    bring(next, row + step);
    float ss = 0.f, gu = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * N + lane) * V;
      float w[V];
      if (c < p.d) load_w<V>(p, c, w, static_cast<const T*>(nullptr));
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float z = now[i].z[j], u = now[i].x[j] * z * gate<T>(z);
        ss = fmaf(u, u, ss);
        if (c < p.d) gu = fmaf(now[i].dy[j] * w[j], u, gu);
      }
    }
    const float2 s = row_sum<WARP, NT>(ss, gu, red);
    const float r = 1.f / sqrtf(s.x / p.d + p.eps), back = r * r * r * (s.y / p.d);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * N + lane) * V;
      if (c >= p.d) continue;
      float w[V], ox[V], oz[V];
      load_w<V>(p, c, w, static_cast<const T*>(nullptr));
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = now[i].x[j], z = now[i].z[j], e = now[i].dy[j] * r, sig = gate<T>(z), gate = z * sig, u = x * gate, du = e * w[j] - u * back;
        dw[i][j] = fmaf(e, u, dw[i][j]);
        ox[j] = du * gate;
        oz[j] = du * x * sig * fmaf(z, 1.f - sig, 1.f);
      }
      store_v<V>(static_cast<T*>(p.dx) + row * p.d + c, ox);
      store_v<V>(static_cast<T*>(p.dz) + row * p.d + c, oz);
    }
  }
  if constexpr (WARP) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) add[threadIdx.x >> 5][(i * 32 + lane) * V + j] = dw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < p.d; c += NT) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) s += add[i][c];
      part[c] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if ((i * N + lane) * V < p.d) store_v<V>(part + (i * N + lane) * V, dw[i]);
  }
}

// The same for rows of any length and place, read twice; dw in the block's own part.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
gate_norm_grad_twice_kernel(const Args p) {
  __shared__ float2 red[WARPS];
  float* part = p.parts + static_cast<long long>(blockIdx.x) * p.d;
  for (int c = threadIdx.x * V; c < p.d; c += THREADS * V)
#pragma unroll
    for (int j = 0; j < V; ++j) part[c + j] = 0.f;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T *x = static_cast<const T*>(p.x) + row * p.x_row, *z = static_cast<const T*>(p.z) + row * p.z_row, *dy = static_cast<const T*>(p.dy) + row * p.dy_row;
    float ss = 0.f, gu = 0.f, a[V], b[V], e[V], w[V];
    auto bring = [&](int c) {
      load_v<V>(x + c, a);
      load_v<V>(z + c, b);
      load_v<V>(dy + c, e);
      load_w<V>(p, c, w, static_cast<const T*>(nullptr));
    };
    for (int c = threadIdx.x * V; c < p.d; c += THREADS * V) {
      bring(c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float u = a[j] * b[j] * gate<T>(b[j]);
        ss = fmaf(u, u, ss);
        gu = fmaf(e[j] * w[j], u, gu);
      }
    }
    const float2 s = row_sum<false, THREADS>(ss, gu, red);
    const float r = 1.f / sqrtf(s.x / p.d + p.eps), back = r * r * r * (s.y / p.d);
    for (int c = threadIdx.x * V; c < p.d; c += THREADS * V) {
      float ox[V], oz[V];
      bring(c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float sig = gate<T>(b[j]), gate = b[j] * sig, u = a[j] * gate, du = r * e[j] * w[j] - u * back;
        part[c + j] += e[j] * u * r;
        ox[j] = du * gate;
        oz[j] = du * a[j] * sig * fmaf(b[j], 1.f - sig, 1.f);
      }
      store_v<V>(static_cast<T*>(p.dx) + row * p.d + c, ox);
      store_v<V>(static_cast<T*>(p.dz) + row * p.d + c, oz);
    }
  }
}

// dw[c] = sum of parts[., c]: 32 columns a block, eight slices of the parts.
template <typename W>
__global__ void __launch_bounds__(THREADS)
weight_sum_kernel(const float* __restrict__ parts, int n, int d, W* __restrict__ dw) {
  __shared__ float red[WARPS][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  float s = 0.f;
  if (c < d)
    for (int i = slice; i < n; i += WARPS) s += parts[static_cast<long long>(i) * d + c];
  red[slice][threadIdx.x & 31] = s;
  __syncthreads();
  if (slice == 0 && c < d) {
#pragma unroll
    for (int i = 1; i < WARPS; ++i) s += red[i][threadIdx.x];
    st(dw + c, s);
  }
}

template <typename T, int V, int ITEMS, bool WARP, int NT>
int go(const Args& p, int blocks, cudaStream_t stream) {
  if (p.dy == nullptr) {
    const long long grid = WARP ? (p.rows + WARPS - 1) / WARPS : p.rows;
    if (grid > 0x7fffffffLL) return -3;
    gate_norm_kernel<T, V, ITEMS, WARP, NT><<<static_cast<unsigned>(grid), NT, 0, stream>>>(p);
  } else if constexpr (ITEMS > 0) {
    gate_norm_grad_kernel<T, V, ITEMS, WARP, NT><<<blocks, NT, 0, stream>>>(p);
  } else {
    gate_norm_grad_twice_kernel<T, V><<<blocks, THREADS, 0, stream>>>(p);
  }
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int any(const Args& p, int blocks, cudaStream_t stream) {
  constexpr int V = sizeof(T) == 2 ? 8 : 4;
  const bool whole = p.d % V == 0 && (p.x_row | p.z_row | p.dy_row) % V == 0 && aligned(p.x, 16) && aligned(p.z, 16) && aligned(p.dy, 16) && aligned(p.w, 16);
  if (!whole) return go<T, 1, 0, false, THREADS>(p, blocks, stream);
  if (p.d <= 32 * V) return go<T, V, 1, true, THREADS>(p, blocks, stream);
  if (p.d <= 64 * V) return go<T, V, 2, true, THREADS>(p, blocks, stream);
  if (p.d <= 128 * V) return go<T, V, 1, false, 128>(p, blocks, stream);
  if (p.d <= 256 * V) return go<T, V, 2, false, 128>(p, blocks, stream);
  if (p.d <= 512 * V) return go<T, V, 2, false, 256>(p, blocks, stream);
  if (p.d <= 1024 * V) return go<T, V, 2, false, 512>(p, blocks, stream);
  return go<T, V, 0, false, THREADS>(p, blocks, stream);
}

inline bool ok(const void* x, const void* z, const void* w, long long rows, int d) { return x != nullptr && z != nullptr && w != nullptr && rows > 0 && d > 0; }

}  // namespace gatenorm
}  // namespace dewb

using namespace dewb::gatenorm;

extern "C" int dewb_gate_norm_fwd(const void* x, long long x_row, const void* z, long long z_row, const void* w, void* y, long long rows, int d, float eps, int fp32, int w_fp32, void* stream_ptr) {
  if (!ok(x, z, w, rows, d) || y == nullptr || (fp32 && !w_fp32)) return -3;
  const Args p{x, z, w, nullptr, x_row, z_row, 0, rows, d, w_fp32, eps, y, nullptr, nullptr, nullptr};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  return fp32 ? any<float>(p, 0, stream) : any<bf16>(p, 0, stream);
}

// `blocks`: rows of `parts`.
extern "C" int dewb_gate_norm_bwd(const void* dy, long long dy_row, const void* x, long long x_row, const void* z, long long z_row, const void* w, void* dx, void* dz, void* dw, float* parts,
                                  int blocks, long long rows, int d, float eps, int fp32, int w_fp32, void* stream_ptr) {
  if (!ok(x, z, w, rows, d) || dy == nullptr || dx == nullptr || dz == nullptr || dw == nullptr || parts == nullptr || blocks < 1 || (fp32 && !w_fp32)) return -3;
  const Args p{x, z, w, dy, x_row, z_row, dy_row, rows, d, w_fp32, eps, nullptr, dx, dz, parts};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  const int rc = fp32 ? any<float>(p, blocks, stream) : any<bf16>(p, blocks, stream);
  if (rc != 0) return rc;
  if (w_fp32) weight_sum_kernel<<<(d + 31) / 32, THREADS, 0, stream>>>(parts, blocks, d, static_cast<float*>(dw));
  else weight_sum_kernel<<<(d + 31) / 32, THREADS, 0, stream>>>(parts, blocks, d, static_cast<bf16*>(dw));
  return static_cast<int>(cudaGetLastError());
}
