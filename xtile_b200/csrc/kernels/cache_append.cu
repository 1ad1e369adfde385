// New keys (rotated on the way) and values into a paged int8 cache with one
// f32 scale for each block of tokens and head:
//
//   s' = max(s, max|x| / 127)   (s: the block's scale, if it has earlier tokens)
//   q  = rint(x / s');  the earlier tokens' rows become rint(q s / s') if s' > s.
//
// Bound by HBM for prompts (each new element read once, one byte written) and
// by latency for single tokens.  One CTA has one block of one head, of the
// keys or of the values: its new rows stay in registers between the largest
// magnitude and the rounding.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../serve.h"
#include "batch.cuh"
#include "pdl.cuh"
#include "rope.cuh"
#include "vec.cuh"

namespace xt {
namespace dev {
namespace {

// Items (two vectors of V elements) a thread holds in registers; blocks with
// more are read a second time, from L2.
constexpr int kHeld = 4;

// CTAs of a prompt's launch: sequence b's blocks start at slot
// starts[b] / block + 2 b, which leaves room for every block that its tokens
// can touch (at most count / block + 2), so that a slot finds its sequence by
// a search in starts alone.
struct Unit {
  int seq, lo, first, last;  // block's first position; new positions [first, last)
  bool mine;
};

template <class T, int V, int THREADS>
__global__ void __launch_bounds__(THREADS) cache_append_blocks(const AppendArgs a, bool by_token) {
  __shared__ float part[THREADS / 32];
  griddep_launch_dependents();
  griddep_wait();
  const BatchView& bt = a.batch;
  const int block = a.cache.block, page = a.cache.page, dim = a.cache.dim;
  const int slot = blockIdx.x, head = blockIdx.y;
  const bool keys = blockIdx.z == 0;

  const int b = by_token
                    ? last_at_most(bt.seqs, slot, [&](int i) { return static_cast<int64_t>(bt.starts[i]); })
                    : last_at_most(bt.seqs, slot, [&](int i) { return bt.starts[i] / block + 2 * static_cast<int64_t>(i); });
  const Sequence s = load_sequence(bt, page, b);
  const int begin = s.length - s.count;
  if (!s.ok || begin < 0) {
    if (threadIdx.x == 0) atomicCAS(a.error_word, 0u, static_cast<uint32_t>(kErrAppendTable));
    return;
  }
  int lo;
  if (by_token) {
    const int i = slot - s.first;
    if (i < 0 || i >= s.count) return;
    if (i != 0 && (begin + i) % block != 0) return;  // the block's first new token has the CTA
    lo = (begin + i) / block * block;
  } else {
    const int64_t k = slot - (s.first / block + 2 * static_cast<int64_t>(b));
    const int64_t at = (begin / block + k) * block;
    if (s.count == 0 || k < 0 || at >= s.length) return;
    lo = static_cast<int>(at);
  }
  const int first = max(lo, begin), last = min(lo + block, s.length);
  const int into = bt.table[b * bt.table_stride + lo / page];
  if (into < 0 || into >= a.cache.pages) {
    if (threadIdx.x == 0) atomicCAS(a.error_word, 0u, static_cast<uint32_t>(kErrAppendTable));
    return;
  }

  const int rot = keys && a.rope ? static_cast<int>(a.rot) : 0;
  const int64_t token_stride = keys ? a.k_token : a.v_token;
  const T* x = static_cast<const T*>(keys ? a.k : a.v) + head * (keys ? a.k_head : a.v_head) +
               (s.first + first - begin) * token_stride;
  const int items = dim / (2 * V), work = (last - first) * items;

  auto load = [&](int w, float (&u)[V], float (&v)[V]) {
    const int row = w / items;
    const RopeSpan span = rope_span<V>(w % items, rot, a.interleaved);
    Vec<T, V>::load(x + row * token_stride + span.first, u);
    Vec<T, V>::load(x + row * token_stride + span.second, v);
    if (span.pair < 0) return;
    float2 cs[V];
    const int pos = first + row;
    if (pos < a.rope_rows) {
      load_turns<V>(a.rope + static_cast<int64_t>(pos) * (rot / 2) + span.pair, cs);
    } else {
      atomicCAS(a.error_word, 0u, static_cast<uint32_t>(kErrRopePosition));
#pragma unroll
      for (int j = 0; j < V; ++j) cs[j] = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
    }
    rope_item<V>(u, v, cs, a.interleaved);
  };

  float u[kHeld][V], v[kHeld][V];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int w = i * THREADS + threadIdx.x;
    if (w >= work) continue;
    load(w, u[i], v[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) top = max_nan(top, max_nan(fabsf(u[i][j]), fabsf(v[i][j])));
  }
  for (int w = kHeld * THREADS + threadIdx.x; w < work; w += THREADS) {
    float p[V], q[V];
    load(w, p, q);
#pragma unroll
    for (int j = 0; j < V; ++j) top = max_nan(top, max_nan(fabsf(p[j]), fabsf(q[j])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  float* scale_at = (keys ? a.cache.k_scale : a.cache.v_scale) +
                    (static_cast<int64_t>(into) * a.cache.heads + head) * (page / block) + lo % page / block;
  const float was = first > lo ? *scale_at : 0.0f;  // read by every thread before the barrier, written behind it
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) top = max_nan(top, part[i]);
  float scale = quant_scale(top);
  if (first > lo) scale = max_nan(scale, was);
  const float inverse = quant_inverse(scale);

  int8_t* rows = (keys ? a.cache.k : a.cache.v) +
                 ((static_cast<int64_t>(into) * a.cache.heads + head) * page + lo % page) * dim;
  if (scale > was && first > lo) {
    if (threadIdx.x == 0) *scale_at = scale;
    const float ratio = was / scale;
    for (int c = threadIdx.x; c < (first - lo) * (dim / 16); c += THREADS) {
      int4* at = reinterpret_cast<int4*>(rows) + c;
      int4 w = *at;
      int* words = &w.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int old = words[j];
        words[j] = static_cast<int>(pack_i8(quantize(static_cast<float>(static_cast<int8_t>(old)), ratio),
                                            quantize(static_cast<float>(static_cast<int8_t>(old >> 8)), ratio),
                                            quantize(static_cast<float>(static_cast<int8_t>(old >> 16)), ratio),
                                            quantize(static_cast<float>(static_cast<int8_t>(old >> 24)), ratio)));
      }
      *at = w;
    }
  } else if (!(scale == was) || first == lo) {
    if (threadIdx.x == 0) *scale_at = scale;  // a fresh block, or NaN
  }
  auto store = [&](int w, const float (&p)[V], const float (&q)[V]) {
    const RopeSpan span = rope_span<V>(w % items, rot, a.interleaved);
    int8_t* to = rows + static_cast<int64_t>(first - lo + w / items) * dim;
    store_i8<V>(to + span.first, p, inverse);
    store_i8<V>(to + span.second, q, inverse);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int w = i * THREADS + threadIdx.x;
    if (w < work) store(w, u[i], v[i]);
  }
  for (int w = kHeld * THREADS + threadIdx.x; w < work; w += THREADS) {
    float p[V], q[V];
    load(w, p, q);
    store(w, p, q);
  }
}

template <class T, int V>
cudaError_t launch_typed(const AppendArgs& a, cudaStream_t stream) {
  const BatchView& bt = a.batch;
  const int64_t by_block = bt.tokens / a.cache.block + 2 * static_cast<int64_t>(bt.seqs);
  const bool by_token = bt.tokens <= by_block;
  const dim3 grid(static_cast<unsigned>(by_token ? bt.tokens : by_block), static_cast<unsigned>(a.cache.heads), 2);
  const int items = a.cache.block * (a.cache.dim / (2 * V));
  if (items <= kHeld * 128) {
    PdlLaunch launch(grid, dim3(128), 0, stream);
    return launch(cache_append_blocks<T, V, 128>, a, by_token);
  }
  PdlLaunch launch(grid, dim3(512), 0, stream);
  return launch(cache_append_blocks<T, V, 512>, a, by_token);
}

}  // namespace

cudaError_t launch_cache_append(const AppendArgs& a, cudaStream_t stream) {
  if (a.batch.tokens <= 0 || a.batch.seqs <= 0 || a.cache.heads <= 0) return cudaSuccess;
  const int size = a.elem == kF32 ? 4 : 2;
  auto fits = [&](int v) {
    auto aligned = [&](const void* p, int64_t token, int64_t head) {
      return reinterpret_cast<uintptr_t>(p) % (v * size) == 0 && token % v == 0 && head % v == 0;
    };
    return a.cache.dim % (2 * v) == 0 && (!a.rope || (a.rot % (2 * v) == 0 && reinterpret_cast<uintptr_t>(a.rope) % 16 == 0)) &&
           aligned(a.k, a.k_token, a.k_head) && aligned(a.v, a.v_token, a.v_head);
  };
  if (a.elem == kF32) return fits(4) ? launch_typed<float, 4>(a, stream) : launch_typed<float, 1>(a, stream);
  if (fits(8)) return launch_typed<__nv_bfloat16, 8>(a, stream);
  return fits(4) ? launch_typed<__nv_bfloat16, 4>(a, stream) : launch_typed<__nv_bfloat16, 1>(a, stream);
}

}  // namespace dev
}  // namespace xt
