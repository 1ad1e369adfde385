// Ragged batches on the device: which sequence a packed row belongs to.
#pragma once

#include <cuda_runtime.h>

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

__device__ __forceinline__ Sequence load_sequence(const BatchView& batch, int page, int b) {
  Sequence s;
  s.first = batch.starts[b];
  const int64_t end = batch.starts[b + 1];
  s.length = batch.lengths[b];
  s.ok = s.first >= 0 && end >= s.first && end <= batch.tokens && s.length >= 0 &&
         s.length <= static_cast<int64_t>(batch.table_width) * page;
  s.count = s.ok ? static_cast<int>(end - s.first) : 0;
  if (!s.ok) s.length = 0;
  return s;
}

}  // namespace dev
}  // namespace xt
