// Ragged batches on the device: which sequence a packed row belongs to.
#pragma once

#include <cuda_runtime.h>

#include <type_traits>

#include "../serve.h"

namespace xt {
namespace dev {

// The last b in [0, count) with key(b) <= x, 0 where there is none, for keys
// that never fall.  A whole warp searches, 32 probes at a time.
template <class Key>
__device__ __forceinline__ int last_at_most(int count, int64_t x, Key key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int probe = lo + lane * step;
    const unsigned hits = __ballot_sync(0xffffffffu, probe < hi && key(probe) <= x);
    lo += hits ? (31 - __clz(hits)) * step : 0;
    hi = min(hi, lo + step);
    if (!hits) break;
  }
  return lo;
}

// Sequence b's rows and lengths, checked: ok is false (and nothing of the
// sequence may be touched) where they leave the arrays.
struct Sequence {
  int first;   // its first new token's row
  int count;   // new tokens
  int length;  // tokens in all
  bool ok;
};

__device__ __forceinline__ Sequence check_sequence(const BatchView& batch, int page, int first, int end, int length) {
  Sequence s;
  s.first = first;
  s.length = length;
  s.ok = first >= 0 && end >= first && end <= batch.tokens && length >= 0 &&
         length <= static_cast<int64_t>(batch.table_width) * page;
  s.count = s.ok ? end - first : 0;
  if (!s.ok) s.length = 0;
  return s;
}

__device__ __forceinline__ Sequence load_sequence(const BatchView& batch, int page, int b) {
  return check_sequence(batch, page, batch.starts[b], batch.starts[b + 1], batch.lengths[b]);
}

// The sequence of a slot: the last one with key(start, b) <= slot, for keys that
// never fall where starts do not.  ``fall``: starts fall somewhere, so that the
// search may have found anything and no slot is sure to be visited.  A whole warp
// calls.  Every start is looked at for that, which takes no longer than a search
// alone among up to 256 (attention of 64 sequences of 20 tokens: 7.3 us both
// ways; of 1500 sequences of 60 tokens 11.7 us, and 10.4 with the search alone).
struct Found {
  Sequence seq;
  int b, start;
  bool fall;
};

template <class Key>
__device__ __forceinline__ Found find_sequence(const BatchView& batch, int page, int64_t slot, Key key) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  Found f;
  if (batch.seqs <= 32) {
    const bool there = lane < batch.seqs;
    const int first = there ? batch.starts[lane] : 0, end = there ? batch.starts[lane + 1] : 0;
    const int length = there ? batch.lengths[lane] : 0;
    f.fall = __any_sync(kAll, end < first);
    const unsigned hits = __ballot_sync(kAll, there && key(first, lane) <= slot);
    f.b = hits ? 31 - __clz(hits) : 0;
    f.start = __shfl_sync(kAll, first, f.b);
    f.seq = check_sequence(batch, page, f.start, __shfl_sync(kAll, end, f.b), __shfl_sync(kAll, length, f.b));
    return f;
  }
  // rounds of 32 starts, kAtOnce of them under way together; hits: rounds' counts of keys up to the slot
  int hits = 0;
  bool fall = false;
  auto rounds = [&](auto at_once, auto search) {
    constexpr int kAtOnce = at_once.value;
    for (int base = 0; base < batch.seqs; base += 32 * kAtOnce) {
      int start[kAtOnce + 1];
#pragma unroll
      for (int k = 0; k <= kAtOnce; ++k) start[k] = batch.starts[min(base + 32 * k + lane, batch.seqs)];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int i = base + 32 * k + lane;
        if (search.value && base + 32 * k >= batch.seqs) break;
        fall |= __shfl_sync(kAll, lane == 0 ? start[k + 1] : start[k], (lane + 1) & 31) < start[k];  // the next start
        if (search.value) hits += __popc(__ballot_sync(kAll, i < batch.seqs && key(start[k], i) <= slot));
      }
    }
  };
  if (batch.seqs <= 256) {
    rounds(std::integral_constant<int, 8>{}, std::true_type{});
    f.b = max(hits - 1, 0);
  } else {
    f.b = last_at_most(batch.seqs, slot, [&](int i) { return key(batch.starts[i], i); });
    rounds(std::integral_constant<int, 16>{}, std::false_type{});
  }
  f.fall = __any_sync(kAll, fall);
  f.start = batch.starts[f.b];
  f.seq = load_sequence(batch, page, f.b);
  return f;
}

}  // namespace dev
}  // namespace xt
