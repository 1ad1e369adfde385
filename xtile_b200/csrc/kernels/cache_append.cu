// New keys (rotated on the way) and values into a paged int8 cache with one
// f32 scale for each block of tokens and head:
//
//   s' = max(s, max|x| / 127)   (s: the block's scale, if it has earlier tokens)
//   q  = rint(x / s');  the earlier tokens' rows become rint(q s / s') if s' > s.
//
// Each new element is read once (the rest of a block that a CTA's registers do not
// hold, twice) and one byte of it written.  What bounds a prompt is the latency
// of its loads: issue slots are 49% busy and DRAM 29%, and of 7 cycles between
// a warp's issues 2.8 go to global loads, which two CTAs an SM do not cover.  So a unit (one block of one head, of the
// keys or of the values) belongs to as few lanes as hold it in registers
// between the largest magnitude and the rounding, and what finds the block's
// place is done once a warp: 17.1k tokens of 8 heads of 128 bf16
// take 36.0 us (2920 GB/s), and took 73 with a CTA of four warps a unit.  64
// single tokens take 3.7 us where cache and tokens are in L2, 4.8 where they are
// not, and 7.5 where besides every block's scale rises, so that its earlier
// tokens' rows are read and rounded anew.
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
  FastDiv items_div;      // by the items of a row: dim / (2 V)
  FastDiv slot_div;       // by the warps (CTAs) of a slot
  FastDiv block_div, page_div;
  int warps, page_blocks;
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
  if (blockIdx.x == 0) {
    // Every sequence is looked at once: where starts fall the search may miss some,
    // whose tokens are not stored then, and a wrong one without a token has no slot.
    bool wrong = false;
    for (int i = threadIdx.x; i < bt.seqs; i += kThreads) {
      const Sequence t = load_sequence(bt, page, i);
      wrong |= !t.ok || t.length < t.count;
    }
    if (wrong) atomicCAS(a.error_word, 0u, static_cast<uint32_t>(kErrAppendTable));
  }
  const int index = kCta ? blockIdx.x : blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (index >= p.warps) return;
  const int slot = p.slot_div.quot(index);
  const int lane = threadIdx.x % LANES;
  // the unit of its slot: keys' heads, then values'
  const int unit = (index - slot * static_cast<int>(p.slot_div.d)) * (kCta ? 1 : 32 / LANES) +
                   (kCta ? 0 : (threadIdx.x & 31) / LANES);
  const bool there = unit < 2 * heads;
  const bool keys = unit < heads;
  const int head = keys ? unit : there ? unit - heads : 0;

  const int b = p.by_token
                    ? last_at_most(bt.seqs, slot, [&](int i) { return static_cast<int64_t>(bt.starts[i]); })
                    : last_at_most(bt.seqs, slot, [&](int i) { return p.block_div.quot(max(bt.starts[i], 0)) + 2 * static_cast<int64_t>(i); });
  const Sequence s = load_sequence(bt, page, b);
  const int begin = s.length - s.count;
  if (!s.ok || begin < 0) return;  // recorded by the first CTA
  int lo;
  if (p.by_token) {
    const int i = slot - s.first, at = begin + i;
    if (i < 0 || i >= s.count) return;
    lo = p.block_div.quot(at) * block;
    if (i != 0 && at != lo) return;  // the block's first new token has the work
  } else {
    const int64_t k = slot - (p.block_div.quot(s.first) + 2 * static_cast<int64_t>(b));
    const int64_t at = (p.block_div.quot(begin) + k) * block;
    if (s.count == 0 || k < 0 || at >= s.length) return;
    lo = static_cast<int>(at);
  }
  const int first = max(lo, begin), last = min(lo + block, s.length);
  const int page_at = p.page_div.quot(lo), row_at = lo - page_at * page;
  const int into = bt.table[b * bt.table_stride + page_at];  // checked once the new rows are on their way

  const int rot = keys && a.rope ? static_cast<int>(a.rot) : 0;
  const int64_t token_stride = keys ? a.k_token : a.v_token;
  const T* x = static_cast<const T*>(keys ? a.k : a.v) + head * (keys ? a.k_head : a.v_head) +
               (s.first + first - begin) * token_stride;
  const int items = p.items_div.d, new_rows = last - first, work = new_rows * items;

  // Loads come without a branch, from the last item again behind the end, so
  // that all of a thread's are under way before the first is waited for (the
  // keys' in one chain of an item after another made a prompt 55 us).
  struct Item {
    int row;  // at or behind new_rows: none
    RopeSpan span;
  };
  const int row0 = p.items_div.quot(lane), item0 = lane - row0 * items;
  const int row_step = p.items_div.quot(LANES), item_step = LANES - row_step * items;
  auto item_at = [&](int i) {  // item i * LANES + lane
    int row = row0 + i * row_step, at = item0 + i * item_step;
    if (item_step) {
      const int carry = p.items_div.quot(at);
      row += carry;
      at -= carry * items;
    }
    return Item{row, rope_span<V>(at, rot, dim, a.interleaved)};
  };
  auto fetch = [&](const Item& it, float (&u)[V], float (&v)[V]) {
    const T* from = x + min(it.row, new_rows - 1) * token_stride;
    Vec<T, V>::load(from + it.span.first, u);
    Vec<T, V>::load(from + it.span.second, v);
  };
  auto fetch_turns = [&](const Item& it, float2 (&cs)[V]) {
    const int64_t pos = min(static_cast<int64_t>(first + min(it.row, new_rows - 1)), a.rope_rows - 1);
    load_turns<V>(a.rope + pos * (rot / 2), it.span, rot, a.interleaved, cs);
  };
  auto rotate = [&](const Item& it, float (&u)[V], float (&v)[V], const float2 (&cs)[V]) {
    if (it.span.pair >= 0) rope_item<V>(u, v, cs, a.interleaved);
  };
  auto load = [&](const Item& it, float (&u)[V], float (&v)[V]) {
    fetch(it, u, v);
    if (rot) {
      float2 cs[V];
      fetch_turns(it, cs);
      rotate(it, u, v, cs);
    }
  };
  const bool off_table = rot && last > a.rope_rows;  // its scale is NaN, then

  float u[HELD][V], v[HELD][V];
  if (HELD > 1 && work <= LANES) {  // single tokens: one item a lane
    load(item_at(0), u[0], v[0]);
#pragma unroll
    for (int i = 1; i < HELD; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) u[i][j] = v[i][j] = 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < HELD; ++i) fetch(item_at(i), u[i], v[i]);
    if (rot) {
      constexpr int kAtOnce = HELD < 2 ? 1 : 2;  // items whose turns registers hold
#pragma unroll
      for (int i = 0; i < HELD; i += kAtOnce) {
        float2 cs[kAtOnce][V];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) fetch_turns(item_at(i + k), cs[k]);
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) rotate(item_at(i + k), u[i + k], v[i + k], cs[k]);
      }
    }
  }
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < HELD; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) top = max_nan(top, max_nan(fabsf(u[i][j]), fabsf(v[i][j])));
  if constexpr (kCta) {
    for (int i = HELD; i * LANES < work; ++i) {
      float y[V], z[V];
      load(item_at(i), y, z);
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
                    (static_cast<int64_t>(into) * heads + head) * p.page_blocks + p.block_div.quot(row_at);
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
  if (off_table) {
    if (lane == 0) atomicCAS(a.error_word, 0u, static_cast<uint32_t>(kErrRopePosition));
    top = __int_as_float(0x7fc00000);
  }
  float scale = quant_scale(top);
  if (first > lo) scale = max_nan(scale, was);
  const float inverse = quant_inverse(scale);

  int8_t* rows = (keys ? a.cache.k : a.cache.v) + ((static_cast<int64_t>(into) * heads + head) * page + row_at) * dim;
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
  auto store = [&](const Item& it, const float (&y)[V], const float (&z)[V]) {
    if (it.row >= new_rows) return;
    int8_t* to = rows + static_cast<int64_t>(first - lo + it.row) * dim;
    store_i8<V>(to + it.span.first, y, inverse);
    store_i8<V>(to + it.span.second, z, inverse);
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i) store(item_at(i), u[i], v[i]);
  if constexpr (kCta) {
    for (int i = HELD; i * LANES < work; ++i) {
      float y[V], z[V];
      load(item_at(i), y, z);
      store(item_at(i), y, z);
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
  p.block_div.set(static_cast<uint32_t>(a.cache.block));
  p.page_div.set(static_cast<uint32_t>(a.cache.page));
  p.page_blocks = a.cache.page / a.cache.block;
  const int64_t slots = p.by_token ? bt.tokens : by_block;
  auto go = [&](auto kernel, int lanes) {
    const bool cta = lanes == kThreads;
    const int units_a_warp = cta ? 1 : 32 / lanes;
    const int64_t a_slot = (2 * static_cast<int64_t>(a.cache.heads) + units_a_warp - 1) / units_a_warp;
    const int64_t warps = slots * a_slot;
    if (warps > 0x7fffff00) return cudaErrorInvalidValue;
    p.slot_div.set(static_cast<uint32_t>(a_slot));
    p.warps = static_cast<int>(warps);
    const int64_t ctas = cta ? warps : (warps + kThreads / 32 - 1) / (kThreads / 32);
    PdlLaunch launch(dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, stream);
    return launch(kernel, p);
  };
  // the fewest lanes that hold a whole block in 64 registers each; few blocks of
  // more than 128 items are quicker with a CTA each (17.1k tokens of 8 f32 heads
  // of 128: 111 us with 256 lanes a block, 45 with 32; 600 of 2 heads 3.5 and 5.2;
  // they meet near 1000 blocks)
  const int64_t items = static_cast<int64_t>(a.cache.block) * row;
  if (items <= 8) return go(cache_append_blocks<T, V, 8, 1>, 8);
  if (items <= 128) return go(cache_append_blocks<T, V, 32, 4>, 32);
  if constexpr (V == 4) {
    if (items <= 256 && slots * 2 * a.cache.heads >= 1024) return go(cache_append_blocks<T, V, 32, 8>, 32);
  }
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
