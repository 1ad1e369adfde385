// Root-mean-square norm of rows, with the residual's addition and an output
// in f32, bf16 or int8 with one scale a row:
//
//   h = x + residual,  y = h * rsqrt(mean(h^2) + eps) * weight,
//   int8: s = max|y| / 127,  q = rint(y / s)  (s = 0 stores zeros).
//
// Bound by HBM: each element is read once and written once.  A row's h stays
// in registers between the sum of squares, the largest magnitude and the
// stores.  Sums are f32.  8192 rows of 4096 bf16 with a residual to int8 take
// 39.8 us, 5910 GB/s of their 235 MB; 8 such rows 2.5 us; 8192 rows of 4095, off
// the vector boundary and so with each weight loaded alone, 70 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstring>

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
  int shift, shift_step;  // SHIFT: elements that row 0 starts behind a vector's boundary, and each row more
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

// Those of V values that fall in a row's [0, cols).
template <class U, int V>
__device__ __forceinline__ void store_some(U* row, int at, int cols, const float (&x)[V], float inverse) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (at + j < 0 || at + j >= cols) continue;
    if constexpr (sizeof(U) == 1) {
      row[at + j] = static_cast<int8_t>(quantize(x[j], inverse));
    } else {
      const float one[1] = {x[j]};
      Vec<U, 1>::store(row + at + j, one);
    }
  }
}

// V elements as they lie in memory.  load_some takes those of [at, at + V) that
// lie in [0, cols), and zeros for the others.
template <class T, int V>
struct Raw {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load_some(const T* row, int at, int cols) {
    T x[V];
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = at + j >= 0 && at + j < cols ? row[at + j] : static_cast<T>(0.0f);
    memcpy(&v, x, sizeof v);
  }
  __device__ __forceinline__ void values(float (&x)[V]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 4) {
        x[i] = __uint_as_float(w[i]);
      } else {
        x[2 * i] = bf16_lo(w[i]);
        x[2 * i + 1] = bf16_hi(w[i]);
      }
    }
  }
};
template <class T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void zero() { v = static_cast<T>(0.0f); }
  __device__ __forceinline__ void load_some(const T*, int, int) {}  // never partial
  __device__ __forceinline__ void values(float (&x)[1]) const { x[0] = static_cast<float>(v); }
};

// A row in a CTA's registers, or (CTA false) in a warp's: N vectors of V
// elements a thread.  SHIFT: rows that start off a vector's boundary, all
// arrays' alike (an odd number of columns); their vectors start on the
// boundary before the row, and the first and last are partial.  Element by
// element, 8192 x 4095 bf16 took 117 us.  A CTA goes on to the row gridDim behind, whose loads are
// under way while this one is reduced, rounded and stored: with a CTA a row
// 8192 x 4096 bf16 took 44.1 us.
template <class T, int V, int N, bool CTA, int MAX_THREADS, int CTAS, bool SHIFT = false>
__global__ void __launch_bounds__(MAX_THREADS, CTAS) rms_norm_rows(const NormDev p) {
  __shared__ float part[2][2][32];
  const int threads = CTA ? blockDim.x : 32;
  const int me = CTA ? threadIdx.x : threadIdx.x & 31;
  const int rows_at_once = CTA ? 1 : blockDim.x >> 5;
  int64_t row = static_cast<int64_t>(blockIdx.x) * rows_at_once + (CTA ? 0 : threadIdx.x >> 5);
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows_at_once;
  griddep_launch_dependents();
  griddep_wait();
  auto shift_of = [&](int64_t at_row) {
    return SHIFT ? static_cast<int>((p.shift + at_row * p.shift_step) % V) : 0;
  };
  auto whole = [&](int at) { return !SHIFT ? at < p.cols : at >= 0 && at + V <= p.cols; };
  auto some = [&](int at) { return SHIFT && at + V > 0 && at < p.cols; };
  Raw<T, V> x[N], res[N];
  auto fetch = [&](int64_t at_row) {
    const T* from = static_cast<const T*>(p.x) + at_row * p.x_stride;
    const T* also = static_cast<const T*>(p.residual) + at_row * p.residual_stride;
    const int shift = shift_of(at_row);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * threads + me) * V - shift;
      x[i].zero();
      res[i].zero();
      if (whole(at)) {
        x[i].load(from + at);
        if (p.residual) res[i].load(also + at);
      } else if (some(at)) {
        x[i].load_some(from, at, p.cols);
        if (p.residual) res[i].load_some(also, at, p.cols);
      }
    }
  };
  if (row < p.rows) fetch(row);
  for (int turn = 0; row < p.rows; row += step, turn ^= 1) {
    const int shift = shift_of(row);
    float h[N][V];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float r[V];
      x[i].values(h[i]);
      res[i].values(r);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] += r[j];
        ss += h[i][j] * h[i][j];
      }
    }
    if (row + step < p.rows) fetch(row + step);
    if (p.sum) {
      T* sum = static_cast<T*>(p.sum) + row * p.sum_stride;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = (i * threads + me) * V - shift;
        if (whole(at))
          Vec<T, V>::store(sum + at, h[i]);
        else if (some(at))
          store_some(sum, at, p.cols, h[i], 0.0f);
      }
    }
    ss = row_reduce<false, CTA>(ss, part[turn][0]);
    const float r = rsqrtf(ss * p.inv_cols + p.eps);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * threads + me) * V - shift;
      if (!whole(at) && !some(at)) continue;
      float w[V];
      if constexpr (SHIFT) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float one[1] = {0.0f};
          if (at + j >= 0 && at + j < p.cols) load_weight<T, 1>(p, at + j, one);
          w[j] = one[0];
        }
      } else {
        load_weight<T, V>(p, at, w);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] = h[i][j] * r * w[j];
        top = max_nan(top, fabsf(h[i][j]));
      }
    }
    float inverse = 0.0f;
    if (p.y_elem == kI8) {
      top = row_reduce<true, CTA>(top, part[turn][1]);
      const float scale = quant_scale(top);
      inverse = quant_inverse(scale);
      if (me == 0) p.scales[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * threads + me) * V - shift;
      if (whole(at)) {
        store_row<V>(p, row, at, h[i], inverse);
      } else if (some(at)) {
        if (p.y_elem == kI8)
          store_some(static_cast<int8_t*>(p.y) + row * p.y_stride, at, p.cols, h[i], inverse);
        else if (p.y_elem == kBF16)
          store_some(static_cast<__nv_bfloat16*>(p.y) + row * p.y_stride, at, p.cols, h[i], inverse);
        else
          store_some(static_cast<float*>(p.y) + row * p.y_stride, at, p.cols, h[i], inverse);
      }
    }
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

template <class T, int V, bool SHIFT = false>
cudaError_t launch_typed(const NormDev& p, cudaStream_t stream) {
  constexpr int kSms = 148;
  // V divides cols unless it is 1; a shifted row may take two vectors more than its elements
  const int vectors = SHIFT ? (p.cols + 2 * V - 2) / V : (p.cols + V - 1) / V;
  // as many CTAs as the SMs hold by the kernel's registers, and no more than there are rows for
  auto go = [&](auto kernel, int regs, int threads, int64_t groups) {
    const int ctas = 65536 / (regs * threads) < 2048 / threads ? 65536 / (regs * threads) : 2048 / threads;
    const int64_t most = static_cast<int64_t>(kSms) * ctas;
    PdlLaunch launch(dim3(static_cast<unsigned>(groups < most ? groups : most)), dim3(static_cast<unsigned>(threads)), 0, stream);
    return launch(kernel, p);
  };
  auto threads_for = [&](int n) { return ((vectors + n - 1) / n + 31) / 32 * 32; };
  // narrow rows: a warp each, no barrier
  const int64_t eights = (p.rows + 7) / 8;
  if (vectors <= 32) return go(rms_norm_rows<T, V, 1, false, 256, 5, SHIFT>, 48, 256, eights);
  if (vectors <= 128) return go(rms_norm_rows<T, V, 4, false, 256, 2, SHIFT>, 128, 256, eights);
  if (vectors <= 512) return go(rms_norm_rows<T, V, 2, true, 256, 4, SHIFT>, 64, threads_for(2), p.rows);
  if (vectors <= 1024) return go(rms_norm_rows<T, V, 2, true, 512, 2, SHIFT>, 64, threads_for(2), p.rows);
  if (vectors <= 4096) return go(rms_norm_rows<T, V, 4, true, 1024, 1, SHIFT>, 64, threads_for(4), p.rows);
  PdlLaunch launch(dim3(static_cast<unsigned>(p.rows)), dim3(1024), 0, stream);
  return launch(rms_norm_wide<T>, p);
}

bool multiple(int64_t a, int64_t b) { return a % b == 0; }

}  // namespace

cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
  NormDev p{a.x,        a.residual, a.weight,     a.y,  a.sum, a.scales, a.x_stride, a.residual_stride,
            a.y_stride, a.sum_stride, a.rows, static_cast<int>(a.cols), a.eps, 1.0f / static_cast<float>(a.cols),
            a.weight_elem, a.y_elem, 0, 0};
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
  // or where every row of every array starts equally far behind one
  auto shift_of = [&](const void* ptr, int bytes) { return static_cast<int>(reinterpret_cast<uintptr_t>(ptr) / bytes % v); };
  p.shift = shift_of(a.x, size);
  p.shift_step = static_cast<int>(a.x_stride % v);
  auto alike = [&](const void* ptr, int64_t stride, int bytes) {
    return !ptr || (shift_of(ptr, bytes) == p.shift && stride % v == p.shift_step);
  };
  const bool shifted = a.x_stride >= 0 && alike(a.residual, a.residual_stride, size) && alike(a.sum, a.sum_stride, size) &&
                       alike(a.y, a.y_stride, y_size);
  if (a.elem == kF32)
    return vec       ? launch_typed<float, 4>(p, stream)
           : shifted ? launch_typed<float, 4, true>(p, stream)
                     : launch_typed<float, 1>(p, stream);
  return vec       ? launch_typed<__nv_bfloat16, 8>(p, stream)
         : shifted ? launch_typed<__nv_bfloat16, 8, true>(p, stream)
                   : launch_typed<__nv_bfloat16, 1>(p, stream);
}

}  // namespace dev
}  // namespace xt
