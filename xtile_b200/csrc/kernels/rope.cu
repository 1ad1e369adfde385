// Rotary positions over heads, and int8 data read back as values.  Both are
// bound by HBM: each element is read once and written once.  8192 tokens of 32
// f32 heads of 128 take 41.5 us, 6520 GB/s (bf16 29.3, 4720 GB/s); 67 million
// int8 values to bf16 31.3 us, 6430 GB/s; a decode step's 16 tokens 2.0 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

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
// Both vectors are read before either is written: y may be x.  The heads come
// before the table's row, whose address waits for the position, and stay packed
// (unpacked at once, 8192 tokens of 32 bf16 heads took 37.0 us, 29.3 so).
template <class T, class U, int V, int HEADS>
__global__ void __launch_bounds__(kThreads) rope_heads(const RopeArgs a, int items, int groups, int tokens_per_cta) {
  // as they lie in memory until a head's turn comes
  using Word = typename std::conditional<V * sizeof(T) == 16, uint4,
                                         typename std::conditional<V * sizeof(T) == 8, uint2, T>::type>::type;
  griddep_launch_dependents();
  griddep_wait();
  const int per_token = items * groups;
  const int work = per_token * tokens_per_cta;
  for (int w = threadIdx.x; w < work; w += kThreads) {
    const int64_t token = static_cast<int64_t>(blockIdx.x) * tokens_per_cta + w / per_token;
    if (token >= a.tokens) return;
    const int group = w % per_token / items;
    const RopeSpan span = rope_span<V>(w % items, static_cast<int>(a.rot), static_cast<int>(a.dim), a.interleaved);
    const T* x = static_cast<const T*>(a.x) + token * a.x_token;
    U* y = static_cast<U*>(a.y) + token * a.y_token;
    Word u[HEADS], v[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int64_t head = static_cast<int64_t>(group) * HEADS + i;
      if (head >= a.heads) continue;
      u[i] = *reinterpret_cast<const Word*>(x + head * a.x_head + span.first);
      v[i] = *reinterpret_cast<const Word*>(x + head * a.x_head + span.second);
    }
    float2 cs[V];
    if (span.pair >= 0) {
      const int64_t pos = a.positions[token];
      if (pos >= 0 && pos < a.table_rows) {
        load_turns<V>(a.table + pos * (a.rot / 2), span, static_cast<int>(a.rot), a.interleaved, cs);
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
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int64_t head = static_cast<int64_t>(group) * HEADS + i;
      if (head >= a.heads) continue;
      float p[V], q[V];
      Vec<T, V>::load(reinterpret_cast<const T*>(&u[i]), p);
      Vec<T, V>::load(reinterpret_cast<const T*>(&v[i]), q);
      if (span.pair >= 0) rope_item<V>(p, q, cs, a.interleaved);
      Vec<U, V>::store(y + head * a.y_head + span.first, p);
      Vec<U, V>::store(y + head * a.y_head + span.second, q);
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

// An item is what makes 16 bytes of values; a thread has ITEMS of them, a CTA's
// width apart and all under way at once, so that a warp reads and writes whole
// lines (16 values a thread at once took 30 us where 25 million f32 ones take
// 21).  ONE: runs are whole items, so an item has one scale.
template <class U, bool ONE>
__global__ void __launch_bounds__(kThreads) dequantize_items(const int8_t* __restrict__ q, const float* __restrict__ scales,
                                                             U* __restrict__ out, int64_t n, int64_t run, FastDiv run_div) {
  constexpr int kValues = 16 / sizeof(U), kItems = 32 / kValues;
  using Word = typename std::conditional<kValues == 4, uint32_t, uint2>::type;
  griddep_launch_dependents();
  griddep_wait();
  const int64_t items = n / kValues;
  auto run_of = [&](int64_t at) { return run_div.d ? static_cast<int64_t>(run_div.quot(static_cast<uint32_t>(at))) : at / run; };
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kItems * kThreads) + threadIdx.x; base < items;
       base += static_cast<int64_t>(gridDim.x) * (kItems * kThreads)) {
    Word w[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int64_t i = base + k * kThreads;
      w[k] = i < items ? reinterpret_cast<const Word*>(q)[i] : Word{};
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int64_t i = base + k * kThreads, at = i * kValues;
      if (i >= items) break;
      const int64_t r = run_of(at);
      const float s = scales[r];
      float y[kValues], next = s;
      int left = kValues;  // values until the next scale
      if (!ONE) {
        left = static_cast<int>(min((r + 1) * run - at, static_cast<int64_t>(kValues)));
        if (left < kValues) next = scales[r + 1];
      }
      const uint32_t* words = reinterpret_cast<const uint32_t*>(&w[k]);
#pragma unroll
      for (int e = 0; e < kValues; ++e) {
        // the byte plus 128 in the mantissa of 2^23: what the conversion unit gives at a quarter of the rate
        const float x = __uint_as_float(__byte_perm(words[e / 4] ^ 0x80808080u, 0x4b000000u, 0x7440u | (e % 4))) - 8388736.0f;
        // runs shorter than an item change more than once in it
        y[e] = x * (ONE || e < left ? s : run >= kValues || e < left + run ? next : scales[run_of(at + e)]);
      }
      Vec<U, kValues>::store(out + at, y);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < n % kValues) {
    const int64_t at = items * kValues + threadIdx.x;
    const float y[1] = {static_cast<float>(q[at]) * scales[run_of(at)]};
    Vec<U, 1>::store(out + at, y);
  }
}

template <class U>
cudaError_t launch_dequantize_typed(const DequantArgs& a, cudaStream_t stream) {
  constexpr int kCtaValues = 32 * kThreads;
  FastDiv run_div{};  // 31-bit numbers, else none
  if (a.n <= INT32_MAX) run_div.set(static_cast<uint32_t>(a.run));
  const int64_t ctas = std::min<int64_t>((a.n + kCtaValues - 1) / kCtaValues, 1 << 30);
  PdlLaunch launch(dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, stream);
  return launch(a.run % (16 / sizeof(U)) == 0 ? dequantize_items<U, true> : dequantize_items<U, false>, a.q, a.scales,
                static_cast<U*>(a.out), a.n, a.run, run_div);
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
