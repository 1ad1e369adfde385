// Root-mean-square norm of rows, with the residual's addition and an output
// in f32, bf16 or int8 with one scale a row:
//
//   h = x + residual,  y = h * rsqrt(mean(h^2) + eps) * weight,
//   int8: s = max|y| / 127,  q = rint(y / s)  (s = 0 stores zeros).
//
// Bound by HBM: each element is read once and written once.  A row's h stays
// in registers between the sum of squares, the largest magnitude and the
// stores.  Sums are f32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../serve.h"
#include "pdl.cuh"
#include "vec.cuh"

namespace xt {
namespace dev {
namespace {

struct NormDev {
  const void* x;
  const void* residual;
  const void* weight;
  void* y;
  void* sum;
  float* scales;
  int64_t x_stride, residual_stride, y_stride, sum_stride;
  int64_t rows;
  int cols;
  float eps, inv_cols;
  uint8_t weight_elem, y_elem;
};

// Sum (or largest, NaN kept) of ``v`` over the threads of a row: a warp, or
// the whole CTA through ``part`` (one word a warp; two calls use two arrays).
template <bool MAX, bool CTA>
__device__ __forceinline__ float row_reduce(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, w) : v + w;
  }
  if constexpr (CTA) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float w = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? max_nan(v, w) : v + w;
    }
  }
  return v;
}

template <class T, int V>
__device__ __forceinline__ void load_weight(const NormDev& p, int at, float (&w)[V]) {
  if (p.weight_elem == kF32)
    Vec<float, V>::load(static_cast<const float*>(p.weight) + at, w);
  else
    Vec<__nv_bfloat16, V>::load(static_cast<const __nv_bfloat16*>(p.weight) + at, w);
}

template <int V>
__device__ __forceinline__ void store_row(const NormDev& p, int64_t row, int at, const float (&y)[V], float inverse) {
  const int64_t to = row * p.y_stride + at;
  if (p.y_elem == kI8)
    store_i8<V>(static_cast<int8_t*>(p.y) + to, y, inverse);
  else if (p.y_elem == kBF16)
    Vec<__nv_bfloat16, V>::store(static_cast<__nv_bfloat16*>(p.y) + to, y);
  else
    Vec<float, V>::store(static_cast<float*>(p.y) + to, y);
}

// One row in a CTA's registers, or (CTA false) in a warp's: N vectors of V
// elements a thread, every load issued before the first use.
template <class T, int V, int N, bool CTA, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS) rms_norm_rows(const NormDev p) {
  __shared__ float part[2][32];
  const int threads = CTA ? blockDim.x : 32;
  const int me = CTA ? threadIdx.x : threadIdx.x & 31;
  const int64_t row = CTA ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  griddep_launch_dependents();
  griddep_wait();
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  float h[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * threads + me) * V;
    if (at < p.cols) {
      Vec<T, V>::load(x + at, h[i]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) h[i][j] = 0.0f;
    }
  }
  if (p.residual) {
    const T* res = static_cast<const T*>(p.residual) + row * p.residual_stride;
    float r[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * threads + me) * V;
      if (at < p.cols) Vec<T, V>::load(res + at, r[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if ((i * threads + me) * V >= p.cols) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) h[i][j] += r[i][j];
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) ss += h[i][j] * h[i][j];
  if (p.sum) {
    T* sum = static_cast<T*>(p.sum) + row * p.sum_stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * threads + me) * V;
      if (at < p.cols) Vec<T, V>::store(sum + at, h[i]);
    }
  }
  ss = row_reduce<false, CTA>(ss, part[0]);
  const float r = rsqrtf(ss * p.inv_cols + p.eps);
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * threads + me) * V;
    if (at >= p.cols) continue;
    float w[V];
    load_weight<T, V>(p, at, w);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      h[i][j] = h[i][j] * r * w[j];
      top = max_nan(top, fabsf(h[i][j]));
    }
  }
  float inverse = 0.0f;
  if (p.y_elem == kI8) {
    top = row_reduce<true, CTA>(top, part[1]);
    const float scale = quant_scale(top);
    inverse = quant_inverse(scale);
    if (me == 0) p.scales[row] = scale;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * threads + me) * V;
    if (at < p.cols) store_row<V>(p, row, at, h[i], inverse);
  }
}

// Rows too wide for a CTA's registers: three passes over x and the residual,
// the later ones mostly from L2.
template <class T>
__global__ void __launch_bounds__(1024) rms_norm_wide(const NormDev p) {
  __shared__ float part[2][32];
  const int64_t row = blockIdx.x;
  griddep_launch_dependents();
  griddep_wait();
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr;
  // every pass reads its own element before it writes it, so the outputs may be the inputs' own arrays
  auto value = [&](int at) {
    float a[1], b[1] = {0.0f};
    Vec<T, 1>::load(x + at, a);
    if (res) Vec<T, 1>::load(res + at, b);
    return a[0] + b[0];
  };
  float ss = 0.0f;
  for (int at = threadIdx.x; at < p.cols; at += blockDim.x) {
    const float h = value(at);
    ss += h * h;
  }
  ss = row_reduce<false, true>(ss, part[0]);
  const float r = rsqrtf(ss * p.inv_cols + p.eps);
  auto normed = [&](int at) {
    float w[1];
    load_weight<T, 1>(p, at, w);
    return value(at) * r * w[0];
  };
  float inverse = 0.0f;
  if (p.y_elem == kI8) {
    float top = 0.0f;
    for (int at = threadIdx.x; at < p.cols; at += blockDim.x) top = max_nan(top, fabsf(normed(at)));
    top = row_reduce<true, true>(top, part[1]);
    const float scale = quant_scale(top);
    inverse = quant_inverse(scale);
    if (threadIdx.x == 0) p.scales[row] = scale;
  }
  T* sum = p.sum ? static_cast<T*>(p.sum) + row * p.sum_stride : nullptr;
  for (int at = threadIdx.x; at < p.cols; at += blockDim.x) {
    const float h[1] = {value(at)};
    const float y[1] = {normed(at)};
    if (sum) Vec<T, 1>::store(sum + at, h);
    store_row<1>(p, row, at, y, inverse);
  }
}

template <class T, int V>
cudaError_t launch_typed(const NormDev& p, cudaStream_t stream) {
  const int vectors = (p.cols + V - 1) / V;  // V divides cols unless it is 1
  if (vectors <= 128) {
    // narrow rows: a warp each, no barrier
    constexpr int kRows = 8;
    PdlLaunch launch(dim3(static_cast<unsigned>((p.rows + kRows - 1) / kRows)), dim3(32 * kRows), 0, stream);
    return vectors <= 32 ? launch(rms_norm_rows<T, V, 1, false, 256>, p) : launch(rms_norm_rows<T, V, 4, false, 256>, p);
  }
  const dim3 grid(static_cast<unsigned>(p.rows));
  auto go = [&](auto kernel, int n) {
    PdlLaunch launch(grid, dim3(static_cast<unsigned>(((vectors + n - 1) / n + 31) / 32 * 32)), 0, stream);
    return launch(kernel, p);
  };
  if (vectors <= 512) return go(rms_norm_rows<T, V, 2, true, 256>, 2);
  if (vectors <= 1024) return go(rms_norm_rows<T, V, 4, true, 256>, 4);
  if (vectors <= 4096) return go(rms_norm_rows<T, V, 4, true, 1024>, 4);
  PdlLaunch launch(grid, dim3(1024), 0, stream);
  return launch(rms_norm_wide<T>, p);
}

bool multiple(int64_t a, int64_t b) { return a % b == 0; }

}  // namespace

cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
  NormDev p{a.x,        a.residual, a.weight,     a.y,  a.sum, a.scales, a.x_stride, a.residual_stride,
            a.y_stride, a.sum_stride, a.rows, static_cast<int>(a.cols), a.eps, 1.0f / static_cast<float>(a.cols),
            a.weight_elem, a.y_elem};
  // 16-byte vectors of x's type where every row of every array starts on its vector's boundary
  const int v = a.elem == kF32 ? 4 : 8;
  auto fits = [&](const void* ptr, int64_t stride, int bytes) {
    return !ptr || (reinterpret_cast<uintptr_t>(ptr) % (bytes < 16 ? bytes : 16) == 0 && multiple(stride, v));
  };
  const int size = a.elem == kF32 ? 4 : 2;
  const int y_size = a.y_elem == kF32 ? 4 : a.y_elem == kBF16 ? 2 : 1;
  const bool vec = multiple(a.cols, v) && fits(a.x, a.x_stride, v * size) && fits(a.residual, a.residual_stride, v * size) &&
                   fits(a.sum, a.sum_stride, v * size) && fits(a.y, a.y_stride, v * y_size) &&
                   reinterpret_cast<uintptr_t>(a.weight) % 16 == 0;
  if (a.elem == kF32) return vec ? launch_typed<float, 4>(p, stream) : launch_typed<float, 1>(p, stream);
  return vec ? launch_typed<__nv_bfloat16, 8>(p, stream) : launch_typed<__nv_bfloat16, 1>(p, stream);
}

}  // namespace dev
}  // namespace xt
