// New keys (rotated on the way) and values into a paged int8 cache with one
// f32 scale for each block of tokens and head:
//
//   s' = max(s, max|x| / 127)   (s: the block's scale, if it has earlier tokens)
//   q  = rint(x / s');  the earlier tokens' rows become rint(q s / s') if s' > s.
//
// Each new element is read once and one byte of it written, but what bounds a
// prompt is instructions: about 20 an element pair for the rotation, the
// largest magnitude and the rounding.  So a unit (one block of one head, of the
// keys or of the values) belongs to as few lanes as hold it in registers
// between the largest magnitude and the rounding, and what finds the block's
// place is done once a warp: 17.5k tokens of 8 heads took 73 us with a CTA of
// four warps a unit.
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

constexpr int kThreads = 256;

struct AppendDev {
  AppendArgs a;
  FastDiv items_div;      // items of a row: dim / (2 V)
  int64_t warps;          // by units of a warp
  int warps_a_slot;
  bool by_token;
};

// Slots of a launch: sequence b's blocks start at slot starts[b] / block + 2 b,
// which leaves room for every block that its tokens can touch (at most count /
// block + 2), so that a slot finds its sequence by a search in starts alone.
// With few tokens each token has a slot (by_token), and the first new token of
// a block does its block's work.
//
// LANES lanes (8, 32, or a CTA's 256) have a unit; a thread holds HELD items
// (two vectors of V elements) of it in registers, and the rest of a longer
// block is read a second time, from L2.
template <class T, int V, int LANES, int HELD>
__global__ void __launch_bounds__(kThreads) cache_append_blocks(const __grid_constant__ AppendDev p) {
  constexpr bool kCta = LANES == kThreads;
  __shared__ float part[kThreads / 32];
  griddep_launch_dependents();
  griddep_wait();
  const AppendArgs& a = p.a;
  const BatchView& bt = a.batch;
  const int block = a.cache.block, page = a.cache.page, dim = a.cache.dim, heads = a.cache.heads;
  const int64_t index = kCta ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (index >= p.warps) return;
  const int64_t slot = index / p.warps_a_slot;
  const int lane = threadIdx.x % LANES;
  // the unit of its slot: keys' heads, then values'
  const int unit = static_cast<int>(index - slot * p.warps_a_slot) * (kCta ? 1 : 32 / LANES) +
                   (kCta ? 0 : (threadIdx.x & 31) / LANES);
  const bool there = unit < 2 * heads;
  const bool keys = unit < heads;
  const int head = keys ? unit : there ? unit - heads : 0;

  const int b = p.by_token
                    ? last_at_most(bt.seqs, slot, [&](int i) { return static_cast<int64_t>(bt.starts[i]); })
                    : last_at_most(bt.seqs, slot, [&](int i) { return bt.starts[i] / block + 2 * static_cast<int64_t>(i); });
  const Sequence s = load_sequence(bt, page, b);
  const int begin = s.length - s.count;
  if (!s.ok || begin < 0) {
    if (lane == 0) atomicCAS(a.error_word, 0u, static_cast<uint32_t>(kErrAppendTable));
    return;
  }
  int lo;
  if (p.by_token) {
    const int64_t i = slot - s.first;
    if (i < 0 || i >= s.count) return;
    const int at = begin + static_cast<int>(i);
    if (i != 0 && at % block != 0) return;  // the block's first new token has the work
    lo = at / block * block;
  } else {
    const int64_t k = slot - (s.first / block + 2 * static_cast<int64_t>(b));
    const int64_t at = (begin / block + k) * block;
    if (s.count == 0 || k < 0 || at >= s.length) return;
    lo = static_cast<int>(at);
  }
  const int first = max(lo, begin), last = min(lo + block, s.length);
  const int into = bt.table[b * bt.table_stride + lo / page];  // checked once the new rows are on their way

  const int rot = keys && a.rope ? static_cast<int>(a.rot) : 0;
  const int64_t token_stride = keys ? a.k_token : a.v_token;
  const T* x = static_cast<const T*>(keys ? a.k : a.v) + head * (keys ? a.k_head : a.v_head) +
               (s.first + first - begin) * token_stride;
  const int items = p.items_div.d, work = there ? (last - first) * items : 0;

  auto load = [&](int w, float (&u)[V], float (&v)[V]) {
    const int row = p.items_div.quot(w);
    const RopeSpan span = rope_span<V>(w - row * items, rot, a.interleaved);
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

  float u[HELD][V], v[HELD][V];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int w = i * LANES + lane;
    if (w >= work) continue;
    load(w, u[i], v[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) top = max_nan(top, max_nan(fabsf(u[i][j]), fabsf(v[i][j])));
  }
  if constexpr (kCta) {
    for (int w = HELD * LANES + lane; w < work; w += LANES) {
      float y[V], z[V];
      load(w, y, z);
#pragma unroll
      for (int j = 0; j < V; ++j) top = max_nan(top, max_nan(fabsf(y[j]), fabsf(z[j])));
    }
  }
#pragma unroll
  for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (into < 0 || into >= a.cache.pages) {
    if (lane == 0) atomicCAS(a.error_word, 0u, static_cast<uint32_t>(kErrAppendTable));
    return;
  }
  float* scale_at = (keys ? a.cache.k_scale : a.cache.v_scale) +
                    (static_cast<int64_t>(into) * heads + head) * (page / block) + lo % page / block;
  // read by every lane of the unit before the barrier, written behind it
  const float was = there && first > lo ? *scale_at : 0.0f;
  if constexpr (kCta) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) top = max_nan(top, part[i]);
  } else {
    __syncwarp();
  }
  if (!there) return;
  float scale = quant_scale(top);
  if (first > lo) scale = max_nan(scale, was);
  const float inverse = quant_inverse(scale);

  int8_t* rows = (keys ? a.cache.k : a.cache.v) + ((static_cast<int64_t>(into) * heads + head) * page + lo % page) * dim;
  if (lane == 0 && (first == lo || !(scale == was))) *scale_at = scale;
  if (scale > was && first > lo) {
    const float ratio = was / scale;
    for (int c = lane; c < (first - lo) * (dim / 16); c += LANES) {
      int4* at = reinterpret_cast<int4*>(rows) + c;
      int4 w = *at;
      w.x = requantize(w.x, ratio), w.y = requantize(w.y, ratio), w.z = requantize(w.z, ratio), w.w = requantize(w.w, ratio);
      *at = w;
    }
  }
  auto store = [&](int w, const float (&y)[V], const float (&z)[V]) {
    const int row = p.items_div.quot(w);
    const RopeSpan span = rope_span<V>(w - row * items, rot, a.interleaved);
    int8_t* to = rows + static_cast<int64_t>(first - lo + row) * dim;
    store_i8<V>(to + span.first, y, inverse);
    store_i8<V>(to + span.second, z, inverse);
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int w = i * LANES + lane;
    if (w < work) store(w, u[i], v[i]);
  }
  if constexpr (kCta) {
    for (int w = HELD * LANES + lane; w < work; w += LANES) {
      float y[V], z[V];
      load(w, y, z);
      store(w, y, z);
    }
  }
}

template <class T, int V>
cudaError_t launch_typed(const AppendArgs& a, cudaStream_t stream) {
  const BatchView& bt = a.batch;
  const int64_t by_block = bt.tokens / a.cache.block + 2 * static_cast<int64_t>(bt.seqs);
  AppendDev p{};
  p.a = a;
  p.by_token = bt.tokens <= by_block;
  const int row = a.cache.dim / (2 * V);
  p.items_div.set(static_cast<uint32_t>(row));
  const int64_t slots = p.by_token ? bt.tokens : by_block;
  auto go = [&](auto kernel, int lanes) {
    const bool cta = lanes == kThreads;
    const int units_a_warp = cta ? 1 : 32 / lanes;
    p.warps_a_slot = (2 * a.cache.heads + units_a_warp - 1) / units_a_warp;
    p.warps = slots * p.warps_a_slot;
    const int64_t ctas = cta ? p.warps : (p.warps + kThreads / 32 - 1) / (kThreads / 32);
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    PdlLaunch launch(dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, stream);
    return launch(kernel, p);
  };
  // the fewest lanes that hold a whole block (4 items a lane: 64 bf16 elements)
  const int64_t items = static_cast<int64_t>(a.cache.block) * row;
  if (items <= 8) return go(cache_append_blocks<T, V, 8, 1>, 8);
  if (items <= 128) return go(cache_append_blocks<T, V, 32, 4>, 32);
  return go(cache_append_blocks<T, V, kThreads, 4>, kThreads);
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
