// Rotary positions over heads, and int8 data read back as values.  Both are
// bound by HBM: each element is read once and written once.  8192 tokens of 32
// f32 heads of 128 take 45.3 us, 5970 GB/s; 67 million int8 values to bf16 33.7
// us, 5980 GB/s; a decode step's 16 tokens 1.9 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../serve.h"
#include "pdl.cuh"
#include "rope.cuh"
#include "vec.cuh"

namespace xt {
namespace dev {
namespace {

constexpr int kThreads = 256;

// A thread turns the same item (two vectors of V elements) of HEADS heads of
// one token, so that it reads the table's cosines and sines once for them all.
// Both vectors are read before either is written: y may be x.
template <class T, class U, int V, int HEADS>
__global__ void __launch_bounds__(kThreads) rope_heads(const RopeArgs a, int items, int groups, int tokens_per_cta) {
  griddep_launch_dependents();
  griddep_wait();
  const int per_token = items * groups;
  const int work = per_token * tokens_per_cta;
  for (int w = threadIdx.x; w < work; w += kThreads) {
    const int64_t token = static_cast<int64_t>(blockIdx.x) * tokens_per_cta + w / per_token;
    if (token >= a.tokens) return;
    const int group = w % per_token / items;
    const RopeSpan span = rope_span<V>(w % items, static_cast<int>(a.rot), a.interleaved);
    float2 cs[V];
    if (span.pair >= 0) {
      const int64_t pos = a.positions[token];
      if (pos >= 0 && pos < a.table_rows) {
        load_turns<V>(a.table + pos * (a.rot / 2) + span.pair, cs);
      } else {
        if (group == 0) atomicCAS(a.error_word, 0u, static_cast<uint32_t>(kErrRopePosition));
#pragma unroll
        for (int j = 0; j < V; ++j) cs[j] = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
      }
      if (a.inverse) {
#pragma unroll
        for (int j = 0; j < V; ++j) cs[j].y = -cs[j].y;
      }
    }
    const T* x = static_cast<const T*>(a.x) + token * a.x_token;
    U* y = static_cast<U*>(a.y) + token * a.y_token;
    float u[HEADS][V], v[HEADS][V];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int64_t head = static_cast<int64_t>(group) * HEADS + i;
      if (head >= a.heads) continue;
      Vec<T, V>::load(x + head * a.x_head + span.first, u[i]);
      Vec<T, V>::load(x + head * a.x_head + span.second, v[i]);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int64_t head = static_cast<int64_t>(group) * HEADS + i;
      if (head >= a.heads) continue;
      if (span.pair >= 0) rope_item<V>(u[i], v[i], cs, a.interleaved);
      Vec<U, V>::store(y + head * a.y_head + span.first, u[i]);
      Vec<U, V>::store(y + head * a.y_head + span.second, v[i]);
    }
  }
}

template <class T, class U, int V>
cudaError_t launch_rope_typed(const RopeArgs& a, cudaStream_t stream) {
  const int items = static_cast<int>(a.dim / (2 * V));
  auto go = [&](auto kernel, int heads) {
    const int groups = static_cast<int>((a.heads + heads - 1) / heads);
    const int per_token = items * groups;
    const int tokens = per_token >= kThreads ? 1 : kThreads / per_token;
    PdlLaunch launch(dim3(static_cast<unsigned>((a.tokens + tokens - 1) / tokens)), dim3(kThreads), 0, stream);
    return launch(kernel, a, items, groups, tokens);
  };
  // four heads a thread once that still leaves every SM its threads, one head below
  const int64_t threads = a.tokens * a.heads * items;
  return threads >= 4 * 148 * 1024 ? go(rope_heads<T, U, V, 4>, 4) : go(rope_heads<T, U, V, 1>, 1);
}

// 16 int8 values as f32 or bf16, one scale.
template <class U>
__device__ __forceinline__ void dequantize_16(const int4& w, float s, U* out) {
  const int words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      y[e] = static_cast<float>(static_cast<int8_t>(words[2 * j + e / 4] >> (8 * (e % 4)))) * s;
    Vec<U, 8>::store(out + 8 * j, y);
  }
}

// Runs of whole 16-byte vectors: two a thread, both loads under way at once.
template <class U>
__global__ void __launch_bounds__(kThreads) dequantize_runs(const int8_t* __restrict__ q, const float* __restrict__ scales,
                                                            U* __restrict__ out, int64_t vectors, int64_t run) {
  griddep_launch_dependents();
  griddep_wait();
  const int4* q4 = reinterpret_cast<const int4*>(q);
  const int64_t run_vectors = run / 16;
  auto scale_of = [&](int64_t i) {
    return scales[(i | run_vectors) >> 32 ? i / run_vectors : static_cast<uint32_t>(i) / static_cast<uint32_t>(run_vectors)];
  };
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (2 * kThreads);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (2 * kThreads) + threadIdx.x; i < vectors; i += stride) {
    const int64_t k = i + kThreads;
    const bool two = k < vectors;
    const int4 a = q4[i], b = two ? q4[k] : make_int4(0, 0, 0, 0);
    const float sa = scale_of(i), sb = two ? scale_of(k) : 0.0f;
    dequantize_16(a, sa, out + 16 * i);
    if (two) dequantize_16(b, sb, out + 16 * k);
  }
}

// Any runs: 16 values a thread, whose scales may change anywhere.
template <class U>
__global__ void __launch_bounds__(kThreads) dequantize_any(const int8_t* __restrict__ q, const float* __restrict__ scales,
                                                           U* __restrict__ out, int64_t n, int64_t run) {
  griddep_launch_dependents();
  griddep_wait();
  const int64_t vectors = (n + 15) / 16;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < vectors;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t at = i * 16;
    int64_t r = (at | run) >> 32 ? at / run : static_cast<uint32_t>(at) / static_cast<uint32_t>(run);
    if (at + 16 <= n) {
      const int4 w = *reinterpret_cast<const int4*>(q + at);
      const int words[4] = {w.x, w.y, w.z, w.w};
      float s = scales[r];
      int64_t left = (r + 1) * run - at;  // elements until the next scale
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (left == 0) {
            s = scales[++r];
            left = run;
          }
          --left;
          y[e] = static_cast<float>(static_cast<int8_t>(words[2 * j + e / 4] >> (8 * (e % 4)))) * s;
        }
        Vec<U, 8>::store(out + at + 8 * j, y);
      }
    } else {
      for (int64_t e = at; e < n; ++e) {
        const float y[1] = {static_cast<float>(q[e]) * scales[e / run]};
        Vec<U, 1>::store(out + e, y);
      }
    }
  }
}

template <class U>
cudaError_t launch_dequantize_typed(const DequantArgs& a, cudaStream_t stream) {
  U* out = static_cast<U*>(a.out);
  const int64_t vectors = (a.n + 15) / 16;
  auto grid = [](int64_t blocks) { return dim3(static_cast<unsigned>(blocks < (1 << 30) ? blocks : (1 << 30))); };
  if (a.run % 16 == 0) {
    PdlLaunch launch(grid((vectors + 2 * kThreads - 1) / (2 * kThreads)), dim3(kThreads), 0, stream);
    return launch(dequantize_runs<U>, a.q, a.scales, out, vectors, a.run);
  }
  PdlLaunch launch(grid((vectors + kThreads - 1) / kThreads), dim3(kThreads), 0, stream);
  return launch(dequantize_any<U>, a.q, a.scales, out, a.n, a.run);
}

}  // namespace

cudaError_t launch_rope(const RopeArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0 || a.heads <= 0) return cudaSuccess;
  const int size = a.elem == kF32 ? 4 : 2, y_size = a.y_elem == kF32 ? 4 : 2;
  // vectors of v elements where both vectors of every item start on one
  auto fits = [&](int v) {
    auto aligned = [&](const void* p, int64_t token, int64_t head, int bytes) {
      return reinterpret_cast<uintptr_t>(p) % (v * bytes) == 0 && token % v == 0 && head % v == 0;
    };
    return a.dim % (2 * v) == 0 && a.rot % (2 * v) == 0 && reinterpret_cast<uintptr_t>(a.table) % 16 == 0 &&
           aligned(a.x, a.x_token, a.x_head, size) && aligned(a.y, a.y_token, a.y_head, y_size);
  };
  using bf16 = __nv_bfloat16;
  if (a.elem == kF32 && a.y_elem == kF32)
    return fits(4) ? launch_rope_typed<float, float, 4>(a, stream) : launch_rope_typed<float, float, 1>(a, stream);
  if (a.elem == kF32)
    return fits(4) ? launch_rope_typed<float, bf16, 4>(a, stream) : launch_rope_typed<float, bf16, 1>(a, stream);
  if (fits(8)) return launch_rope_typed<bf16, bf16, 8>(a, stream);
  return fits(4) ? launch_rope_typed<bf16, bf16, 4>(a, stream) : launch_rope_typed<bf16, bf16, 1>(a, stream);
}

cudaError_t launch_dequantize(const DequantArgs& a, cudaStream_t stream) {
  if (a.n <= 0) return cudaSuccess;
  return a.elem == kF32 ? launch_dequantize_typed<float>(a, stream) : launch_dequantize_typed<__nv_bfloat16>(a, stream);
}

}  // namespace dev
}  // namespace xt
