// Attention over the paged int8 cache: for each new token's head
//
//   z_j = scale * ks_j * (q . kq_j)          [z_j = cap * tanh(z_j / cap)]
//   out = sum_j softmax_j(z) * vs_j * vq_j
//
// over the tokens j that the query sees (causal from the end of its sequence,
// and a window if one is set).  A token's reads are 2 dim int8 bytes a kv
// head, so single-token decoding is bound by HBM.
//
// Work is cut into units of kTile tokens of one (sequence, kv head, packed query
// rows) segment; a row is a (new token, head of the group) pair, so the heads
// of a group share the cache's reads.  The units of all segments stand in one
// line, and each warp of a grid that fills the GPU takes an equal run of it:
// ragged lengths, a single long sequence and many short ones all load every SM
// alike.  A warp works alone, without a CTA barrier: it streams its own tiles
// through its own ring in shared memory (TMA boxes of 16 rows where pages hold
// whole tiles, cp.async rows where they do not), runs the two products on
// mma.sync m16n8k16 in f16 and keeps the running reference, sum and output of
// its rows in registers.  Segments that several warps share are joined by a
// second kernel from f32 partial results.  That kernel costs 4.5 us, so small
// calls give each segment to a cluster instead, whose warps split its tokens
// and join in shared memory.
//
// 64 sequences of up to 8192 tokens, 32 query heads over 8 of 128: 124 us, 5420
// GB/s of their 674 MB (graph replay; 126 to 141 as calls among others, by GPU);
// one sequence of 777 tokens 7.5 us.
//
// Tokens (and the output's dims) are the products' m, query rows their n: the
// converted cache bytes are A operands that all of a segment's rows share, and
// a group of up to 8 heads fills one n8 tile.  What a unit costs is mostly the
// conversion of its bytes (five instructions for four key bytes, six for four
// value bytes), not the products.  Keys that entered as the f16 subnormals (byte +
// 128) 2^-24 would take three (64 ragged contexts 122.3 us, 125.7 so), but the
// sums would be rounded at the size of what the 128s add, which is not small
// where a query's large elements meet keys near 0.
//
// int8 values are exact in f16, and so is a bf16 query divided by a power of
// two that brings its row's largest magnitude near 2^10: elements under 2^-27 of
// that lose bits, those under 2^-35 are gone, all at most 2^-35 of it off.  The
// scales of the tokens' blocks stay outside the products: the key's multiplies
// the score in f32, the value's the weight, which is rounded once to f16 (11
// bits) on its way into the second product.
// f32 queries go in as two f16 terms, and so do their weights: 22 bits.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../serve.h"
#include "attend.cuh"
#include "batch.cuh"
#include "pdl.cuh"
#include "sm100.cuh"
#include "vec.cuh"

namespace xt {
namespace dev {
namespace {

constexpr int kTile = 16;  // tokens of a unit: the products' m
constexpr uint32_t kErrUnitWait = 0x307;

// How one instance of the kernel is laid out.  DP: dims, padded; NR: n8 tiles
// of query rows.
template <int DP, bool F32, int NR>
struct Shape {
  static constexpr int kRows = 8 * NR;  // query rows of a segment
  static constexpr int kWarps = DP <= 128 ? 4 : 2;
  static constexpr bool kHeavy = F32 || NR == 4 || DP > 128;
  // CTAs an SM, by the registers of a row and dim
  static constexpr int kCtas = DP > 128 ? (F32 && NR > 1 ? 2 : 3) : F32 || DP * NR > 128 ? 2 : NR == 2 ? 3 : 4;
  static constexpr int kMatrix = kTile * DP;             // a stage holds keys and values
  static constexpr bool kQueryInSmem = kHeavy;           // else its fragments stay in registers
  static constexpr int kQueryBytes = kQueryInSmem ? (DP / 16) * NR * 256 * (F32 ? 2 : 1) : 0;
  // shared memory of a CTA: 1 KB is the system's, 1 KB alignment, 256 bytes barriers
  static constexpr int kSpare = 227 * 1024 / kCtas - 2 * 1024 - 256;
  static constexpr int kFit = (kSpare / kWarps - kQueryBytes) / (2 * kMatrix);
  static constexpr int kStages = kFit < 4 ? kFit : 4;
  static_assert(kStages >= 3, "a warp's ring holds three stages at least");
  static constexpr int kWarpBytes = kStages * 2 * kMatrix + kQueryBytes;
  static_assert(kWarpBytes % 1024 == 0, "a ring starts on a swizzle atom");
  static constexpr int kBytes = kWarps * kWarpBytes + 256 + 1024;
  static_assert(kRows * DP * 4 + kRows * 16 <= kWarpBytes, "a warp's partial result fits its ring");
};

// How tiles come: rows by cp.async or boxes by TMA, units shared out over the
// grid; or rows by cp.async, a cluster a segment.
enum class Form { kRows, kBoxes, kCluster };

// The units of sequence b: kv heads x row tiles x token tiles [lo, hi).
struct Segments {
  Sequence seq;
  int row_tiles, lo, hi;
  __device__ __forceinline__ int64_t units(int heads) const {
    return static_cast<int64_t>(heads) * row_tiles * (hi - lo);
  }
};

template <int ROWS>
__device__ __forceinline__ Segments segments_of_sequence(const AttendDev& p, const Sequence& seq) {
  Segments g;
  g.seq = seq;
  if (!g.seq.ok) atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
  g.row_tiles = static_cast<int>((static_cast<int64_t>(g.seq.count) * p.group + ROWS - 1) / ROWS);
  const int64_t first_seen = p.a.window > 0 ? static_cast<int64_t>(g.seq.length) - g.seq.count - p.a.window + 1 : 0;
  g.lo = first_seen > 0 ? static_cast<int>(first_seen) / kTile : 0;
  g.hi = (g.seq.length + kTile - 1) / kTile;
  if (g.lo > g.hi) g.lo = g.hi;
  return g;
}

template <int ROWS>
__device__ __forceinline__ Segments load_segments(const AttendDev& p, int b) {
  return segments_of_sequence<ROWS>(p, load_sequence(p.a.batch, p.a.cache.page, b));
}

// a / b of positive values; 64-bit division took a third of a microsecond.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Units that each worker takes.
__device__ __forceinline__ int64_t units_each(const AttendDev& p, int64_t total) {
  return max(divide(total + p.workers - 1, p.workers), static_cast<int64_t>(p.least));
}

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Units of all sequences, and of those before ``b``; -1 where starts fall, and no
// sequence is sure of its rows.  A whole warp calls.
template <int ROWS>
__device__ __forceinline__ int64_t count_units(const AttendDev& p, int b, int64_t* before) {
  int64_t total = 0, front = 0;
  bool fall = false;
  for (int i = threadIdx.x & 31; i < p.a.batch.seqs; i += 32) {
    const int64_t u = load_segments<ROWS>(p, i).units(p.a.cache.heads);
    total += u;
    if (i < b) front += u;
    fall |= p.a.batch.starts[i + 1] < p.a.batch.starts[i];
  }
  *before = warp_sum64(front);
  return __any_sync(0xffffffffu, fall) ? -1 : warp_sum64(total);
}

// A place in the line of units.
template <int ROWS>
struct Cursor {
  Segments seg;
  int b, head, row_tile, tile;

  __device__ __forceinline__ void seek(const AttendDev& p, int64_t u) {
    const int lane = threadIdx.x & 31, heads = p.a.cache.heads;
    int64_t front = 0;
    b = 0;
    for (int base = 0; base < p.a.batch.seqs; base += 32) {
      const int i = base + lane;
      const int64_t mine = i < p.a.batch.seqs ? load_segments<ROWS>(p, i).units(heads) : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t w = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += w;
      }
      const unsigned behind = __ballot_sync(0xffffffffu, front + upto > u);
      if (behind) {
        const int l = __ffs(behind) - 1;
        b = base + l;
        front += __shfl_sync(0xffffffffu, upto - mine, l);
        break;
      }
      front += __shfl_sync(0xffffffffu, upto, 31);
    }
    seg = load_segments<ROWS>(p, b);
    const int tiles = seg.hi - seg.lo;
    const int64_t at = u - front, line = divide(at, tiles);
    tile = seg.lo + static_cast<int>(at - line * tiles);
    head = static_cast<int>(divide(line, seg.row_tiles));
    row_tile = static_cast<int>(line - static_cast<int64_t>(head) * seg.row_tiles);
  }

  // The next unit; there must be one.  True if it is of the same segment.
  __device__ __forceinline__ bool advance(const AttendDev& p) {
    if (++tile < seg.hi) return true;
    tile = seg.lo;
    if (++row_tile < seg.row_tiles) return false;
    row_tile = 0;
    if (++head < p.a.cache.heads) return false;
    head = 0;
    do {
      ++b;
      seg = load_segments<ROWS>(p, b);
    } while (seg.units(1) == 0 && b + 1 < p.a.batch.seqs);
    tile = seg.lo;
    return false;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// Arrives on ``bar`` once the calling lane's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(sm100::smem_addr(bar)) : "memory");
}

// c += a b for 16 x 16 f16 a, 16 x 8 f16 b, f32 c.
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}

// The transpose of an 8 x 8 matrix of 16-bit elements, a row's pairs over a quad.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// What two values leave after their rounding to f16, as f16.
__device__ __forceinline__ uint32_t rest_half2(float lo, float hi, uint32_t rounded) {
  const float2 r = unpack_half2(rounded);
  return pack_half2(lo - r.x, hi - r.y);
}

// Shared-memory places of 16-byte chunk ``c`` of a tile's token ``row``: TMA's
// swizzle of 128-byte rows (two halves of 16 rows at 256 dims) or 64-byte rows.
template <int DP>
__device__ __forceinline__ uint32_t place(int row, int c) {
  if constexpr (DP == 64) return row * 64 + ((c ^ (row >> 1 & 3)) << 4);
  return (c >> 3) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}

// The token of a tile that row r (of 8) of the score product stands for; row
// r + 8 is the one 8 behind it.  With that order the eight lanes of each
// quarter of a 16-byte read meet eight different bank groups, both where keys
// are read (chunks t .. of rows 2 q and 2 q + 1) and values (chunk 2 q or 2 q + 1
// of rows 0, 2, 4, 6 or 1, 3, 5, 7).
template <int DP>
__device__ __forceinline__ int token_of_row(int r) {
  return DP == 64 ? r ^ (r >> 1 & 1) : r ^ ((r & 1) << 2);
}

__device__ __forceinline__ void lds128(uint32_t (&w)[4], uint32_t at) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
}

template <int DP, bool F32, int NR, Form FORM>
__global__ void __launch_bounds__(Shape<DP, F32, NR>::kWarps * 32, Shape<DP, F32, NR>::kCtas)
    attend_units(const __grid_constant__ AttendDev p, const __grid_constant__ CUtensorMap key_map,
                 const __grid_constant__ CUtensorMap value_map) {
  using S = Shape<DP, F32, NR>;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  constexpr bool TMA = FORM == Form::kBoxes, kCluster = FORM == Form::kCluster;
  constexpr int kRows = S::kRows, kStages = S::kStages;
  constexpr int kSteps = DP / 16;    // k16 steps of the score product
  constexpr int kOut = DP / 16;      // m16 tiles of the output
  constexpr int kSpan = DP >= 128 ? 16 : 8;  // consecutive dims that a lane reads of a value row
  constexpr int kBox = DP < 128 ? DP : 128;  // bytes of a row in a TMA box
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + warp * S::kWarpBytes;
  const uint32_t ring_addr = sm100::smem_addr(ring);
  uint2* query = reinterpret_cast<uint2*>(ring + kStages * 2 * S::kMatrix);
  const int warps = kCluster ? blockDim.x >> 5 : S::kWarps;
  uint64_t* landed = reinterpret_cast<uint64_t*>(smem + warps * S::kWarpBytes) + warp * kStages;  // a stage's data
  int* abort_flag = reinterpret_cast<int*>(smem + warps * S::kWarpBytes + 128) + warp;
  const CacheView& cache = p.a.cache;
  const int dim = cache.dim;

  if (!TMA && dim < DP) {
    // chunks behind dim are never loaded by cp.async; they stay zero
    for (int i = lane; i < kStages * 2 * S::kMatrix / 16; i += 32)
      reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
  }
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) sm100::mbar_init(&landed[i], TMA ? 1 : 32);
    *abort_flag = 0;
    sm100::fence_barrier_init();
  }
  __syncwarp();
  griddep_wait();
  // behind the wait: what the join reads before its own wait is final, then
  griddep_launch_dependents();

  Cursor<kRows> at;
  int64_t worker = 0;
  int left;  // units to do
  if constexpr (kCluster) {
    const int rank = blockIdx.x % p.cluster, index = blockIdx.x / p.cluster, slot = index / cache.heads;
    auto base = [&](int start, int i) { return first_slot(start, i, p.group, kRows); };
    const Found found = find_sequence(p.a.batch, cache.page, slot, base);
    at.b = found.b;
    at.head = index - slot * cache.heads;
    at.seg = segments_of_sequence<kRows>(p, found.seq);
    const int64_t row_tile = slot - base(found.start, found.b);
    // the cluster's CTAs return together
    if (found.fall) {
      refuse_batch<T>(p);
      return;
    }
    if (!at.seg.seq.ok) {
      if (row_tile == 0 && rank == 0) refuse_sequence<T>(p, at.b, at.head, threadIdx.x, blockDim.x);
      return;
    }
    if (row_tile < 0 || row_tile >= at.seg.row_tiles) return;
    at.row_tile = static_cast<int>(row_tile);
    const int64_t tiles = at.seg.hi - at.seg.lo, of = p.cluster * warps, mine = rank * warps + warp;
    at.tile = at.seg.lo + static_cast<int>(divide(tiles * mine, of));
    left = at.seg.lo + static_cast<int>(divide(tiles * (mine + 1), of)) - at.tile;
  } else {
    int64_t unused;
    const int64_t total = count_units<kRows>(p, 0, &unused);
    const int64_t per = units_each(p, total);
    worker = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
    const int64_t begin = worker * per;
    if (begin >= total) return;
    left = static_cast<int>(total - begin < per ? total - begin : per);
    at.seek(p, begin);
  }
  int to_issue = left;
  Cursor<kRows> ahead = at;

  // --- loading.  By TMA a tile is one run of rows of a page: the next page is
  // looked up as soon as the one at hand is entered.  Else lane l looks up the
  // page of token l % 16 of the tile to come.  Lane l holds the scale of that
  // token's keys (lanes 0 to 15) or values of each tile under way.
  const float* my_scales = lane < kTile ? cache.k_scale : cache.v_scale;
  float scale[kStages - 1];  // oldest first
  int page_id = 0, page_row = 0, next_id = 0, page_index = 0;
  auto table_at = [&](int index) {
    return index * cache.page < ahead.seg.seq.length ? p.a.batch.table[ahead.b * p.a.batch.table_stride + index] : 0;
  };
  auto look_up = [&](bool same_segment) {
    if constexpr (TMA) {
      if (same_segment) {
        page_row += kTile;
        if (page_row < cache.page) return;
        page_row = 0;
        ++page_index;
        page_id = next_id;
      } else {
        page_index = p.page_div.quot(ahead.tile * kTile);
        page_row = ahead.tile * kTile - page_index * cache.page;
        page_id = table_at(page_index);
      }
      next_id = table_at(page_index + 1);
    } else {
      const int token = ahead.tile * kTile + lane % kTile;
      const int index = p.page_div.quot(token);
      page_row = token - index * cache.page;
      page_id = token < ahead.seg.seq.length ? table_at(index) : 0;
    }
  };
  auto issue = [&](int stage) {
    float s = 0.0f;
    if (to_issue > 0) {
      const int there = ahead.seg.seq.length - ahead.tile * kTile;  // tokens of the tile: 16 of them, or fewer
      const bool bad = static_cast<uint32_t>(page_id) >= static_cast<uint32_t>(cache.pages);
      const int line = (bad ? 0 : page_id) * cache.heads + ahead.head;
      const int row = page_row + (TMA ? lane % kTile : 0);
      const uint64_t scale_at = static_cast<uint64_t>(static_cast<uint32_t>(line)) * static_cast<uint32_t>(p.blocks) +
                                p.block_div.quot(row);
      if (lane % kTile < there) {
        s = bad ? __int_as_float(0x7fc00000) : my_scales[scale_at];
        // a page outside the cache: recorded, and NaN for whoever attends to it
        if (bad) atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
      }
      // Rows behind the sequence's end are whatever the page or the ring holds:
      // finite int8, and their weight is 0.  So are a bad page's, with NaN.
      if constexpr (TMA) {
        if (sm100::elect_sync()) {
          if (bad) {
            sm100::mbar_arrive(&landed[stage]);
          } else {
            sm100::mbar_arrive_expect_tx(&landed[stage], 2 * S::kMatrix);
            unsigned char* to = ring + stage * 2 * S::kMatrix;
#pragma unroll
            for (int h = 0; h < DP / kBox; ++h) {
              sm100::tma_load_2d(to + h * kTile * kBox, &key_map, &landed[stage], h * kBox, line * cache.page + page_row);
              sm100::tma_load_2d(to + S::kMatrix + h * kTile * kBox, &value_map, &landed[stage], h * kBox,
                                 line * cache.page + page_row);
            }
          }
        }
        __syncwarp();
      } else {
        constexpr int kChunks = DP / 16;  // 16-byte chunks of a token
        constexpr int kRowsAtOnce = 32 / kChunks;
        const int my_chunk = lane % kChunks, my_row = lane / kChunks;
        const uint32_t base = ring_addr + stage * 2 * S::kMatrix;
        const int64_t row_at = static_cast<int64_t>(line) * cache.page + page_row;
        const unsigned rows_there = __ballot_sync(0xffffffffu, lane % kTile < there && !bad);
#pragma unroll
        for (int i = 0; i < kTile / kRowsAtOnce; ++i) {
          const int r = i * kRowsAtOnce + my_row;
          const int64_t from = __shfl_sync(0xffffffffu, row_at, r) * dim + my_chunk * 16;
          if (my_chunk * 16 < dim && (rows_there >> r & 1)) {
            cp_async16(base + place<DP>(r, my_chunk), cache.k + from);
            cp_async16(base + S::kMatrix + place<DP>(r, my_chunk), cache.v + from);
          }
        }
        cp_async_arrive(&landed[stage]);
      }
      if (--to_issue > 0) look_up(ahead.advance(p));
    }
    return s;
  };
  if (to_issue > 0) look_up(false);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) scale[i] = issue(i);

  // --- the segment at hand
  uint2 qf[S::kQueryInSmem ? 1 : NR][S::kQueryInSmem ? 1 : kSteps];
  float o[kOut][NR][4];
  // rows 2 t and 2 t + 1 of each n8 tile: reference of the exponents, sum of
  // the weights, factor of the score in the exponent (1 behind a cap, whose own
  // factor is capped_scale), position of the query
  float ref[NR][2], sum[NR][2], row_scale[NR][2], capped_scale[NR][2];
  int row_pos[NR][2];
  int pos_min = 0, pos_max = 0;
  int value_exp = 0;                     // the weights carry vs 2^(10 - value_exp); set by the first token seen
  bool value_set = false, whole = true;  // whole: the segment's first unit is this worker's
  const float cap = p.a.softcap;
  const bool negative = p.a.scale < 0.0f;

  auto row_of = [&](int r, int* token) {  // packed row r of the row tile: its new token and query head, or -1
    const int packed = at.row_tile * kRows + r;
    const int i = p.group_div.quot(packed);
    *token = i;
    return i < at.seg.seq.count ? at.head * p.group + packed - i * p.group : -1;
  };

  auto start_segment = [&] {
    whole = at.tile == at.seg.lo;
    value_set = false;
    value_exp = 0;
    const int before = at.seg.seq.length - at.seg.seq.count;
    pos_min = before + p.group_div.quot(at.row_tile * kRows);
    pos_max = before + min(static_cast<int>(p.group_div.quot(at.row_tile * kRows + kRows - 1)), at.seg.seq.count - 1);
    if constexpr (S::kQueryInSmem) __syncwarp();
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int i = 0; i < kOut; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][nr][j] = 0.0f;
      // the lane's part of row g: four dims of each step
      float q[kSteps][4], top = 0.0f;
      int i;
      const int head = row_of(8 * nr + g, &i);
      const T* from = static_cast<const T*>(p.a.q) + static_cast<int64_t>(at.seg.seq.first + i) * p.a.q_token +
                      static_cast<int64_t>(head) * p.a.q_head;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int d = 64 * (s / 4) + 16 * t + 4 * (s % 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) q[s][e] = 0.0f;
        if (head >= 0 && d < dim) Vec<T, 4>::load(from + d, q[s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(q[s][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row times 2^(10 - exponent of its largest magnitude), and the scale's sign
      const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 11), 254);
      const float up = __uint_as_float(static_cast<uint32_t>(264 - e) << 23 | (negative ? 0x80000000u : 0u));
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int x = 0; x < 4; ++x) q[s][x] *= up;
        const uint2 f = make_uint2(pack_half2(q[s][0], q[s][1]), pack_half2(q[s][2], q[s][3]));
        if constexpr (S::kQueryInSmem)
          query[(nr * kSteps + s) * 32 + lane] = f;  // read back by this lane alone
        else
          qf[nr][s] = f;
        if constexpr (F32)
          query[((NR + nr) * kSteps + s) * 32 + lane] =
              make_uint2(rest_half2(q[s][0], q[s][1], f.x), rest_half2(q[s][2], q[s][3], f.y));
      }
      const float down = __uint_as_float(static_cast<uint32_t>(e - 10) << 23) * fabsf(p.a.scale) * (cap > 0.0f ? 1.0f / cap : kLog2e);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        capped_scale[nr][c] = __shfl_sync(0xffffffffu, down, (2 * t + c) * 4);
        row_scale[nr][c] = cap > 0.0f ? 1.0f : capped_scale[nr][c];
        row_pos[nr][c] = before + static_cast<int>(p.group_div.quot(at.row_tile * kRows + 8 * nr + 2 * t + c));
        ref[nr][c] = kNone;
        sum[nr][c] = 0.0f;
      }
    }
  };

  auto finish_segment = [&](bool last_unit) {
    const float up = __uint_as_float(static_cast<uint32_t>(value_exp + 117) << 23);
    const bool done = whole && last_unit;
    const int64_t slot = worker * 2 + (whole ? 1 : 0);
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s = sum[nr][c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const int row = 8 * nr + 2 * t + c;
        int i;
        const int head = row_of(row, &i);
        if (head < 0) continue;
        const float by = done ? (s > 0.0f || s != s ? up / s : 0.0f) : up;
        T* to = static_cast<T*>(p.a.out) + static_cast<int64_t>(at.seg.seq.first + i) * p.a.out_token +
                static_cast<int64_t>(head) * p.a.out_head;
        float* part = p.part + (slot * kRows + row) * dim;
#pragma unroll
        for (int x = 0; x < kOut * 2; x += 4) {
          // m16 tile i's rows g and g + 8 stand for two neighbouring dims of the lane's span
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = o[(x + e) / 2][nr][2 * ((x + e) % 2) + c] * by;
          const int d = x / kSpan * 8 * kSpan + g * kSpan + x % kSpan;
          if (d >= dim) continue;
          if (done)
            Vec<T, 4>::store(to + d, y);
          else
            *reinterpret_cast<float4*>(part + d) = make_float4(y[0], y[1], y[2], y[3]);
        }
        if (!done && g == 0) p.part_ml[slot * kRows + row] = make_float2(ref[nr][c], s);
      }
  };

  start_segment();
  // what the lane reads of a tile: keys of tokens (row g) and 8 behind, values
  // of tokens (rows 2 t and 2 t + 1) and 8 behind
  const int key_row = token_of_row<DP>(g);
  const uint32_t key_at = place<DP>(key_row, t);
  const uint32_t value_at[2] = {place<DP>(token_of_row<DP>(2 * t), DP == 64 ? g >> 1 : g) + (DP == 64 ? (g & 1) * 8 : 0),
                                place<DP>(token_of_row<DP>(2 * t + 1), DP == 64 ? g >> 1 : g) + (DP == 64 ? (g & 1) * 8 : 0)};
  constexpr int kEight = 8 * kBox;  // eight rows on
  const sm100::Abort ab{abort_flag, p.a.error_word, sm100::wait_limit_or_default(p.a.wait_limit_cycles)};
  int stage = 0;
  uint32_t phase = 0;
  while (!kCluster || left > 0) {
    if (!__all_sync(0xffffffffu, bounded_wait(&landed[stage], phase, ab, kErrUnitWait))) break;
    __syncwarp();  // every lane has read the stage before this one
    const float scales = scale[0];
#pragma unroll
    for (int i = 0; i < kStages - 2; ++i) scale[i] = scale[i + 1];
    scale[kStages - 2] = issue(stage == 0 ? kStages - 1 : stage - 1);
    const uint32_t keys = ring_addr + stage * 2 * S::kMatrix;
    const uint32_t values = keys + S::kMatrix;

    // --- scores: rows g and g + 8 of the tile's tokens
    float z[NR][4];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int e = 0; e < 4; ++e) z[nr][e] = 0.0f;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      uint32_t u[4], w[4];
      float part[NR][4] = {};  // f32: a fresh sum for 64 dims, added in f32, as the tensor cores' own sums round toward zero
      const uint32_t from = keys + (key_at ^ ((j & 1) << 6)) + (j >> 1) * kTile * 128;
      lds128(u, from);
      lds128(w, from + kEight);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t x = u[s] ^ 0x80808080u, y = w[s] ^ 0x80808080u;
        const int step = 4 * j + s;
        const uint32_t a0 = bytes_to_half2<kLow>(x), a2 = bytes_to_half2<kHigh>(x);
        const uint32_t a1 = bytes_to_half2<kLow>(y), a3 = bytes_to_half2<kHigh>(y);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
          if constexpr (F32) {
            mma_16816(part[nr], a0, a1, a2, a3, query[((NR + nr) * kSteps + step) * 32 + lane]);
            mma_16816(part[nr], a0, a1, a2, a3, query[(nr * kSteps + step) * 32 + lane]);
          } else if constexpr (S::kQueryInSmem) {
            mma_16816(z[nr], a0, a1, a2, a3, query[(nr * kSteps + step) * 32 + lane]);
          } else {
            mma_16816(z[nr], a0, a1, a2, a3, qf[nr][step]);
          }
        }
      }
      if constexpr (F32) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int e = 0; e < 4; ++e) z[nr][e] += part[nr][e];
      }
    }

    // --- weights: z becomes the score over the row's factor (with a cap: the
    // capped score in the exponent's unit), y its exponent
    const int token0 = at.tile * kTile;
    // every row sees all of the tile's tokens
    const bool open = token0 + kTile - 1 <= pos_min && (p.a.window == 0 || token0 > pos_max - p.a.window);
    const float ks[2] = {__shfl_sync(0xffffffffu, scales, key_row), __shfl_sync(0xffffffffu, scales, key_row + 8)};
    const float vs[2] = {__shfl_sync(0xffffffffu, scales, key_row + 16), __shfl_sync(0xffffffffu, scales, key_row + 24)};
    float y[NR][4];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int e = 0; e < 4; ++e) z[nr][e] *= ks[e >> 1];
    if (cap > 0.0f) {
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = z[nr][e] * capped_scale[nr][e & 1];
          z[nr][e] = (F32 ? tanhf(x) : tanh_fast(x)) * (cap * kLog2e);
        }
    }
    auto exponents = [&] {
      float top = -INFINITY;
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[nr][e] = fmaf(z[nr][e], row_scale[nr][e & 1], -ref[nr][e & 1]);
          if (!open) {
            const int j = token0 + key_row + 8 * (e >> 1), pos = row_pos[nr][e & 1];
            if (j > pos || (p.a.window > 0 && j <= pos - p.a.window)) y[nr][e] = -INFINITY;
          }
          top = fmaxf(top, y[nr][e]);
        }
      return top;
    };
    const float top = exponents();
    float shift = __uint_as_float(static_cast<uint32_t>(137 - value_exp) << 23);
    // The reference of a row's exponents follows its maximum only when that has
    // risen by more than 2^4, and the values' scales enter the weights as
    // multiples of a power of two that the first scales seen set and that
    // changes only where a weight could leave f16's range: most units leave
    // the output as it is.  2^10 of room below the largest weights keeps f16's
    // subnormals (2^-24 apart) at 2^-34 of them.
    if (__any_sync(0xffffffffu, top > 4.0f || fmaxf(vs[0], vs[1]) * shift > 2048.0f || !value_set)) {
      int e = 0;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float seen = -INFINITY;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) seen = fmaxf(seen, fmaxf(y[nr][2 * r], y[nr][2 * r + 1]));
        const int b = static_cast<int>(__float_as_uint(vs[r]) >> 23 & 255);
        if (seen > -INFINITY && b < 255) e = max(e, b);
      }
      e = __reduce_max_sync(0xffffffffu, e);
      float fall = 1.0f;
      if (e > 0) {
        e = min(max(e, 11), 250) - 127;
        if (!value_set) {
          value_exp = e;
        } else if (e > value_exp) {
          fall = __uint_as_float(static_cast<uint32_t>(max(127 + value_exp - e, 0)) << 23);
          value_exp = e;
        }
        value_set = true;
        shift = __uint_as_float(static_cast<uint32_t>(137 - value_exp) << 23);
      }
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float rise = fmaxf(y[nr][c], y[nr][c + 2]);
          float best = -INFINITY;
          if (y[nr][c] > -INFINITY) best = fmaxf(best, z[nr][c] * row_scale[nr][c]);
          if (y[nr][c + 2] > -INFINITY) best = fmaxf(best, z[nr][c + 2] * row_scale[nr][c]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            rise = fmaxf(rise, __shfl_xor_sync(0xffffffffu, rise, x));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, x));
          }
          float f = 1.0f;
          if (rise > 0.0f) {
            f = exp2_fast(ref[nr][c] - best);
            ref[nr][c] = best;
          }
          sum[nr][c] *= f;
          f *= fall;
#pragma unroll
          for (int i = 0; i < kOut; ++i) {
            o[i][nr][c] *= f;
            o[i][nr][c + 2] *= f;
          }
        }
      exponents();
    }
    uint2 wf[NR], wl[F32 ? NR : 1];
    const float v0 = vs[0] * shift, v1 = vs[1] * shift;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float weight = exp2_fast(y[nr][e]);
        sum[nr][e & 1] += weight;
        w[e] = weight * (e < 2 ? v0 : v1);
        // a token that is not seen may have any scale
        if (!open && y[nr][e] == -INFINITY) w[e] = 0.0f;
      }
      const uint32_t a = pack_half2(w[0], w[1]), b = pack_half2(w[2], w[3]);
      wf[nr] = make_uint2(transpose_8x8(a), transpose_8x8(b));
      if constexpr (F32)
        wl[nr] = make_uint2(transpose_8x8(rest_half2(w[0], w[1], a)), transpose_8x8(rest_half2(w[2], w[3], b)));
    }

    // --- output
    constexpr int kWords = kSpan / 4;  // words of a token that one read brings
#pragma unroll
    for (int h = 0; h < DP / (8 * kSpan); ++h) {
      uint32_t v[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t from = values + value_at[i & 1] + (i >> 1) * kEight + h * kTile * 128;
        if constexpr (DP >= 128)
          lds128(v[i], from);
        else
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[i][0]), "=r"(v[i][1]) : "r"(from));
      }
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // bytes 2 half and 2 half + 1 of two tokens, side by side
          const uint32_t a = __byte_perm(v[0][k], v[1][k], half ? 0x7362u : 0x5140u) ^ 0x80808080u;
          const uint32_t b = __byte_perm(v[2][k], v[3][k], half ? 0x7362u : 0x5140u) ^ 0x80808080u;
          const uint32_t a0 = bytes_to_half2<kLow>(a), a1 = bytes_to_half2<kHigh>(a);
          const uint32_t a2 = bytes_to_half2<kLow>(b), a3 = bytes_to_half2<kHigh>(b);
          const int i = h * kSpan / 2 + 2 * k + half;
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) {
            if constexpr (F32) {
              // a fresh sum for the tile, added in f32: the tensor cores' own sums round toward zero
              float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_16816(c, a0, a1, a2, a3, wl[nr]);
              mma_16816(c, a0, a1, a2, a3, wf[nr]);
#pragma unroll
              for (int x = 0; x < 4; ++x) o[i][nr][x] += c[x];
            } else {
              mma_16816(o[i][nr], a0, a1, a2, a3, wf[nr]);
            }
          }
        }
      }
    }
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }

    --left;
    if constexpr (kCluster) {
      ++at.tile;
      continue;
    }
    const bool last_unit = at.tile + 1 == at.seg.hi;
    if (last_unit || left == 0) {
      finish_segment(last_unit);
      if (left == 0) return;
      at.advance(p);
      start_segment();
    } else {
      ++at.tile;
    }
  }
  if (left > 0) {
    // a wait gave up: what is under way lands before the memory goes ...
    for (int i = 0; i < kStages - 1 && left - to_issue > i; ++i) {
      sm100::mbar_wait_drain(&landed[stage], phase, 500000000ull);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    // ... and the rows of all units that were left are NaN
    auto spoil = [&] {
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) sum[nr][0] = sum[nr][1] = __int_as_float(0x7fc00000);
    };
    spoil();
    if constexpr (!kCluster) {
      while (true) {
        const int here = min(left, at.seg.hi - at.tile);
        at.tile += here - 1;  // the last of them
        left -= here;
        finish_segment(at.tile + 1 == at.seg.hi);
        if (left == 0) return;
        at.advance(p);
        whole = true;
        spoil();
      }
    }
  }
  if constexpr (kCluster) {
    if (p.cluster * warps == 1) {
      finish_segment(true);
      return;
    }
    // --- the warps' results, over their rings: [rows][dim], then (reference, sum) of each row
    __syncwarp();
    const float up = __uint_as_float(static_cast<uint32_t>(value_exp + 117) << 23);
    auto part_of = [&](int w) { return reinterpret_cast<float*>(smem + w * S::kWarpBytes); };
    auto sums_of = [&](int w) { return reinterpret_cast<float2*>(part_of(w) + kRows * DP); };
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s = sum[nr][c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const int row = 8 * nr + 2 * t + c;
#pragma unroll
        for (int x = 0; x < kOut * 2; x += 4) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = o[(x + e) / 2][nr][2 * ((x + e) % 2) + c] * up;
          const int d = x / kSpan * 8 * kSpan + g * kSpan + x % kSpan;
          *reinterpret_cast<float4*>(part_of(warp) + row * DP + d) = make_float4(y[0], y[1], y[2], y[3]);
        }
        if (g == 0) sums_of(warp)[row] = make_float2(ref[nr][c], s);
      }
    __syncthreads();
    // --- the CTA's, four dims a thread, over warp 0's (its sums behind them)
    auto join = [&](auto count) {
      constexpr int kWarps = count.value, kThreads = kWarps * 32, kItems = kRows * DP / 4;
      float2* cta_sums = sums_of(0) + kRows;
      for (int item = threadIdx.x; item < kItems; item += kThreads) {
        const int row = item / (DP / 4), d = item % (DP / 4) * 4;
        float2 ml[kWarps];
        float top = kNone;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          ml[w] = sums_of(w)[row];
          top = fmaxf(top, ml[w].x);
        }
        float s = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float by = exp2_fast(ml[w].x - top);
          const float4 v = *reinterpret_cast<const float4*>(part_of(w) + row * DP + d);
          s += ml[w].y * by;
          y[0] += v.x * by, y[1] += v.y * by, y[2] += v.z * by, y[3] += v.w * by;
        }
        *reinterpret_cast<float4*>(part_of(0) + row * DP + d) = make_float4(y[0], y[1], y[2], y[3]);
        if (d == 0) cta_sums[row] = make_float2(top, s);
      }
      // --- the cluster's: each CTA has a share of the items
      if (p.cluster > 1)
        sm100::cluster_sync();
      else
        __syncthreads();
      const int rank = blockIdx.x % p.cluster;
      for (int item = rank * kThreads + threadIdx.x; item < kItems; item += p.cluster * kThreads) {
        const int row = item / (DP / 4), d = item % (DP / 4) * 4;
        int i;
        const int head = row_of(row, &i);
        if (head < 0 || d >= dim) continue;
        float top = kNone;
        for (int c = 0; c < p.cluster; ++c) top = fmaxf(top, cluster_load2(cta_sums + row, c).x);
        float s = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = 0; c < p.cluster; ++c) {
          const float2 ml = cluster_load2(cta_sums + row, c);
          const float4 v = cluster_load4(part_of(0) + row * DP + d, c);
          const float by = exp2_fast(ml.x - top);
          s += ml.y * by;
          y[0] += v.x * by, y[1] += v.y * by, y[2] += v.z * by, y[3] += v.w * by;
        }
        const float over = s > 0.0f || s != s ? 1.0f / s : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= over;
        Vec<T, 4>::store(static_cast<T*>(p.a.out) + static_cast<int64_t>(at.seg.seq.first + i) * p.a.out_token +
                             static_cast<int64_t>(head) * p.a.out_head + d, y);
      }
    };
    if (warps == S::kWarps)
      join(std::integral_constant<int, S::kWarps>{});
    else
      join(std::integral_constant<int, 2>{});
    if (p.cluster > 1) sm100::cluster_sync();  // no CTA goes while another reads its memory
  }
}

// Joins the partial results of the segments that several workers had.  WARPS
// warps have one (new token, query head): each takes every WARPS-th partial.
template <class T, int DP, int ROWS, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) attend_join(const __grid_constant__ AttendDev p) {
  constexpr int kPer = DP / 32;  // dims a lane
  __shared__ float shared_o[WARPS == 1 ? 1 : WARPS][WARPS == 1 ? 1 : DP];
  __shared__ float2 shared_ml[WARPS];
  // The batch's tables were final before attend_units let this grid start, so
  // they are read before the wait for its results.  Every thread waits, also
  // those with nothing to join: what follows this grid counts on attend_units
  // being done.
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t index = WARPS == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + warp : blockIdx.x;
  if (index >= static_cast<int64_t>(p.a.batch.tokens) * p.a.q_heads) {
    griddep_wait();
    return;
  }
  const int token = static_cast<int>(static_cast<uint32_t>(index) / static_cast<uint32_t>(p.a.q_heads));
  const int q_head = static_cast<int>(index) - token * p.a.q_heads;
  const int b = last_at_most(p.a.batch.seqs, token, [&](int i) { return static_cast<int64_t>(p.a.batch.starts[i]); });
  const Segments seg = load_segments<ROWS>(p, b);
  const int i = token - seg.seq.first, tiles = seg.hi - seg.lo;
  const int head = p.group_div.quot(q_head);
  const int packed = i * p.group + q_head - head * p.group;
  int64_t first = 0, last = 0, front;
  const int64_t total = count_units<ROWS>(p, b, &front);
  const bool sure = total >= 0;
  const bool mine_to_join = sure && seg.seq.ok && i >= 0 && i < seg.seq.count && tiles > 0;
  if (mine_to_join) {
    const int64_t per = units_each(p, total);
    const int64_t u0 = front + (static_cast<int64_t>(head) * seg.row_tiles + packed / ROWS) * tiles;
    first = divide(u0, per), last = divide(u0 + tiles - 1, per);
  }
  griddep_wait();
  T* out = static_cast<T*>(p.a.out) + static_cast<int64_t>(token) * p.a.out_token + static_cast<int64_t>(q_head) * p.a.out_head;
  if (!mine_to_join) {
    if (sure && seg.seq.ok && (i < 0 || i >= seg.seq.count)) return;  // a row of no sequence
    // no token at all: 0; a wrong table: recorded, and NaN
    const float v[1] = {sure && seg.seq.ok ? 0.0f : __int_as_float(0x7fc00000)};
    for (int d = lane; d < p.a.cache.dim; d += 32) Vec<T, 1>::store(out + d, v);
    return;
  }
  if (first == last) return;  // one worker had it all, and has written it
  const int row = packed % ROWS, dim = p.a.cache.dim;
  auto slot_of = [&](int64_t c) { return (c * 2 + (c == first ? 1 : 0)) * ROWS + row; };

  float ref = -INFINITY, sum = 0.0f, y[kPer];
#pragma unroll
  for (int d = 0; d < kPer; ++d) y[d] = 0.0f;
  const bool mine = lane * kPer < dim;
  for (int64_t base = first + (WARPS == 1 ? 0 : warp); base <= last; base += 32 * WARPS) {
    // 32 partials: lane l has the reference and sum of one
    const int64_t c = base + lane * WARPS;
    const float2 ml = c <= last ? p.part_ml[slot_of(c)] : make_float2(-INFINITY, 0.0f);
    float top = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float now = fmaxf(ref, top), safe = now == -INFINITY ? 0.0f : now;
    const float f = exp2f(ref - safe);
    const float weight = exp2f(ml.x - safe);
    float s = c <= last ? ml.y * weight : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    sum = sum * f + s;
    ref = now;
#pragma unroll
    for (int d = 0; d < kPer; ++d) y[d] *= f;
    const int64_t left = (last - base) / WARPS + 1;
    const int count = left < 32 ? static_cast<int>(left) : 32;
#pragma unroll 4
    for (int k = 0; k < count; ++k) {
      const float by = __shfl_sync(0xffffffffu, weight, k);
      const float* from = p.part + slot_of(base + k * WARPS) * dim + lane * kPer;
      if (!mine) continue;
#pragma unroll
      for (int d = 0; d < kPer; d += 2) {
        const float2 v = *reinterpret_cast<const float2*>(from + d);
        y[d] += v.x * by;
        y[d + 1] += v.y * by;
      }
    }
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int d = 0; d < kPer; ++d) shared_o[warp][lane * kPer + d] = y[d];
    if (lane == 0) shared_ml[warp] = make_float2(ref, sum);
    __syncthreads();
    if (warp != 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, shared_ml[w].x);
    const float safe = top == -INFINITY ? 0.0f : top;
    sum = 0.0f;
#pragma unroll
    for (int d = 0; d < kPer; ++d) y[d] = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float by = exp2f(shared_ml[w].x - safe);
      sum += shared_ml[w].y * by;
#pragma unroll
      for (int d = 0; d < kPer; ++d) y[d] += shared_o[w][lane * kPer + d] * by;
    }
  }
  if (!mine) return;
  const float by = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int d = 0; d < kPer; ++d) {
    const float v[1] = {y[d] * by};
    Vec<T, 1>::store(out + lane * kPer + d, v);
  }
}

int sm_count() {
  static std::atomic<int> known[kMaxDevices];
  int device = 0, sms = 148;
  cudaGetDevice(&device);
  const bool keep = device >= 0 && device < kMaxDevices;
  if (keep && known[device]) return known[device];
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (keep) known[device] = sms;
  return sms;
}

// A tensor map of ``lines`` rows of ``dim`` bytes whose boxes are 16 rows of up
// to 128 bytes, swizzled as place() has it; bytes behind dim read as zeros.
bool cache_map(CUtensorMap* map, const void* base, int dim, uint64_t lines, int padded) {
  typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  auto encode = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
  if (!encode) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(dim), lines};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(dim)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(padded < 128 ? padded : 128), kTile};
  const cuuint32_t step[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, padded < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, bool F32, int NR>
cudaError_t launch_shape(AttendDev& p, cudaStream_t stream, size_t* bytes) {
  using S = Shape<DP, F32, NR>;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  const int sms = sm_count(), dim = p.a.cache.dim, resident = sms * S::kCtas;
  static std::atomic<bool> allowed[3][kMaxDevices];
  const int64_t longest = longest_seen(p, kTile), tiles = (longest + kTile - 1) / kTile, segments = segments_of(p, S::kRows);
  // A cluster a segment where the whole is small (1.3 units a nanosecond make
  // 16384 of them 12 us, of which an uneven share loses less than the join) and no
  // warp of a cluster has many units beyond an even share, at 0.7 us each (1.1 over
  // 128 dims): one sequence of 4000 tokens and two kv heads takes 13.0 us in
  // clusters and 14.4 shared out, of 8000 19.7 and 16.2, of 64000 112 and 34.
  const int64_t even = segments * tiles / (static_cast<int64_t>(resident) * S::kWarps);
  if (segments * tiles <= 16384 && tiles <= ((DP <= 128 ? 12 : 5) + even) * 8 * S::kWarps) {
    if (bytes) {
      *bytes = 0;
      return cudaSuccess;
    }
    auto kernel = attend_units<DP, F32, NR, Form::kCluster>;
    const cudaError_t e = allow_smem(kernel, S::kBytes, allowed[2]);
    if (e != cudaSuccess) return e;
    const int64_t slots = first_slot(p.a.batch.tokens, p.a.batch.seqs, p.group, S::kRows) * p.a.cache.heads;
    auto launch = [&](int warps, int cluster) {
      return PdlLaunch(dim3(static_cast<unsigned>(slots * cluster)), dim3(warps * 32),
                       S::kBytes - (S::kWarps - warps) * S::kWarpBytes, stream, cluster);
    };
    // A segment's warps: as many as it has tiles and the GPU has room for, so
    // that many short segments stand side by side, each with a warp (50 sequences
    // of 5 new tokens, 56 f32 heads and 28 tokens: 30.7 us with four warps for
    // each segment, 10.8 with one).  A cluster's SMs are neighbours: how many fit
    // is less than their CTAs would.
    static std::atomic<int> fitting[2][kMaxDevices];  // 8 and 4 CTAs a cluster
    auto fit = [&](int cluster) {
      if (cluster <= 2) return resident / cluster;
      return clusters_at_once(kernel, launch(S::kWarps, cluster), fitting[cluster == 4]);
    };
    int warps = S::kWarps;
    p.cluster = 8;
    while (p.cluster > 1 && (p.cluster * warps > tiles || segments > fit(p.cluster))) p.cluster /= 2;
    // alone, a CTA has fewer warps only where there is no room: one without a tile still helps with the join
    if (tiles == 1) warps = 1;
    while (p.cluster == 1 && warps > 1 && segments * warps > resident * S::kWarps) warps /= 2;
    return launch(warps, p.cluster)(kernel, p, CUtensorMap{}, CUtensorMap{});
  }
  p.workers = static_cast<int64_t>(resident) * S::kWarps;
  const int64_t rows = static_cast<int64_t>(p.a.batch.tokens) * p.a.q_heads;
  // a row's partials are spread over eight warps where the rows alone would not fill the GPU
  const int join_warps = rows <= 4 * sms ? 8 : 1;
  // A worker's unit takes 0.7 us and a partial result 0.3 us of its row's warps in
  // the join: few segments get as many units a worker as make the sum least (64000
  // tokens of two kv heads: 55 us with a worker for each four units, 34 so).  No more
  // than 16: the sequences may be shorter than their table allows.
  p.least = std::clamp(static_cast<int>(std::sqrt(0.43f * tiles / join_warps)), 1, 16);
  if (bytes) {
    *bytes = static_cast<size_t>(p.workers) * 2 * S::kRows * (dim + 2) * sizeof(float);
    return cudaSuccess;
  }
  p.part = static_cast<float*>(p.a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part + p.workers * 2 * S::kRows * dim);
  // Boxes of a tile's rows by TMA where pages hold whole tiles (a box's row is a
  // 32-bit coordinate) and the sequences may be long enough: encoding the maps
  // costs 5 us on the host, and TMA wins 12 us of 134 at 670 MB.
  CUtensorMap maps[2] = {};
  const uint64_t lines = static_cast<uint64_t>(p.a.cache.pages) * p.a.cache.heads * p.a.cache.page;
  const bool tma = p.a.cache.page % kTile == 0 && lines <= 0x7fffffff &&
                   longest * p.a.batch.seqs * p.a.cache.heads * dim >= (64 << 20);
  if (tma && (!cache_map(&maps[0], p.a.cache.k, dim, lines, DP) || !cache_map(&maps[1], p.a.cache.v, dim, lines, DP)))
    return cudaErrorInvalidValue;
  auto kernel = tma ? attend_units<DP, F32, NR, Form::kBoxes> : attend_units<DP, F32, NR, Form::kRows>;
  cudaError_t e = allow_smem(kernel, S::kBytes, allowed[tma]);
  if (e != cudaSuccess) return e;
  PdlLaunch launch(dim3(static_cast<unsigned>(resident)), dim3(S::kWarps * 32), S::kBytes, stream);
  e = launch(kernel, p, maps[0], maps[1]);
  if (e != cudaSuccess) return e;
  if (join_warps == 8) {
    PdlLaunch join(dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream);
    return join(attend_join<T, DP, S::kRows, 8>, p);
  }
  PdlLaunch join(dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream);
  return join(attend_join<T, DP, S::kRows, 1>, p);
}

// Whether the tcgen05 kernel for many query rows runs the call, and the CTAs
// that share a segment's tokens in it, by what the two kernels would take as far
// as the host knows (us; fitted to 1 to 89 sequences of 1024 to 65536 tokens,
// 4 to 512 of them new, within a third of what was measured):
//   that one    6.5, 6.5 a wave of CTAs (7.5 where clusters join), and 2.2 or 2.7
//               a tile of 128 tokens with 64 or 128 dims and up to 128 rows, 2.8
//               or 3.4 with up to 256
//   this one    4 to 20, and 1.7 or 3.0 for a million (row, token) pairs
// 16384 rows of one sequence and 4096 tokens: 240 here, 79 there; 256 rows 25 and
// 24; 64 sequences of 32 rows, 8 heads and up to 1024 tokens 85 and 112.
bool for_prompt(AttendDev& p) {
  const int64_t rows = static_cast<int64_t>(new_tokens(p)) * p.group;
  const bool vectors = reinterpret_cast<uintptr_t>(p.a.q) % 16 == 0 && reinterpret_cast<uintptr_t>(p.a.out) % 16 == 0 &&
                       p.a.q_token % 8 == 0 && p.a.q_head % 8 == 0 && p.a.out_token % 8 == 0 && p.a.out_head % 8 == 0;
  if (p.a.elem != kBF16 || p.a.cache.dim > 128 || !vectors || rows <= 16) return false;
  const bool small = p.a.cache.dim <= 64;
  const int64_t longest = longest_seen(p, 128), tiles = (longest + 127) / 128, segments = segments_of(p, 256);
  if (tiles == 0) return false;  // no page at all
  const float tile_us = small ? (rows <= 128 ? 2.2f : 2.8f) : rows <= 128 ? 2.7f : 3.4f;
  float best = 0.0f;
  for (int cluster = 1; cluster <= 8 && cluster <= tiles; cluster *= 2) {
    const int64_t at_once = cluster == 1 ? sm_count() : prompt_clusters(cluster);
    if (at_once == 0) break;
    // ragged or many segments fill each other's gaps
    float waves = std::max(static_cast<float>(segments) / at_once, 1.0f);
    if (p.a.batch.seqs == 1 && waves < 2.0f) waves = std::ceil(waves);
    const float us = 6.5f + waves * (tile_us * ((tiles + cluster - 1) / cluster) + (cluster > 1 ? 7.5f : 6.5f));
    if (cluster > 1 && us >= best) continue;
    best = us;
    p.cluster = cluster;
  }
  const float pairs = static_cast<float>(segments_of(p, 32)) * 32e-6f * longest;
  return best < 4.0f + std::min(16.0f, longest / 160.0f) + (small ? 1.7f : 3.0f) * pairs;
}

// Query rows of a segment: 8, 16 or 32, by the rows that a sequence's new
// tokens and the group make.  Registers hold 16 at dims over 128 and in f32.
// Where the GPU has a warp for each unit of fewer rows (2368 of them run at
// once at best), sharing units would only leave warps idle: 21 new tokens of 4
// heads behind a window of 5 took 11.8 us with 32 rows and 5.6 with 8.
template <int DP, bool F32>
cudaError_t launch_rows_for(AttendDev& p, cudaStream_t stream, size_t* bytes) {
  const int64_t rows = static_cast<int64_t>(new_tokens(p)) * p.group;
  const int64_t tiles = (longest_seen(p, kTile) + kTile - 1) / kTile;
  auto spread = [&](int fewer) { return segments_of(p, fewer) * tiles <= 16 * sm_count(); };
  if (rows <= 8 || spread(8)) return launch_shape<DP, F32, 1>(p, stream, bytes);
  if constexpr (DP <= 128 && !F32) {
    if (rows > 16 && !spread(16)) return launch_shape<DP, F32, 4>(p, stream, bytes);
  }
  return launch_shape<DP, F32, 2>(p, stream, bytes);
}

// Launches, or tells the size of the workspace where ``bytes`` is given.
cudaError_t launch_any(const AttendArgs& a, cudaStream_t stream, size_t* bytes) {
  AttendDev p{};
  p.a = a;
  p.group = a.q_heads / a.cache.heads;
  p.blocks = a.cache.page / a.cache.block;
  p.page_div.set(static_cast<uint32_t>(a.cache.page));
  p.block_div.set(static_cast<uint32_t>(a.cache.block));
  p.group_div.set(static_cast<uint32_t>(p.group));
  const int dim = a.cache.dim;
  if (for_prompt(p)) {
    if (!bytes) return launch_attend_prompt(p, stream);
    *bytes = 0;
    return cudaSuccess;
  }
  if (a.elem == kF32)
    return dim <= 64    ? launch_rows_for<64, true>(p, stream, bytes)
           : dim <= 128 ? launch_rows_for<128, true>(p, stream, bytes)
                        : launch_rows_for<256, true>(p, stream, bytes);
  return dim <= 64    ? launch_rows_for<64, false>(p, stream, bytes)
         : dim <= 128 ? launch_rows_for<128, false>(p, stream, bytes)
                      : launch_rows_for<256, false>(p, stream, bytes);
}

}  // namespace

size_t attend_workspace_bytes(const AttendArgs& a) {
  if (a.batch.tokens <= 0 || a.batch.seqs <= 0) return 0;
  size_t bytes = 0;
  launch_any(a, nullptr, &bytes);
  return bytes;
}

cudaError_t launch_cache_attention(const AttendArgs& a, cudaStream_t stream) {
  if (a.batch.tokens <= 0 || a.batch.seqs <= 0 || a.q_heads <= 0) return cudaSuccess;
  return launch_any(a, stream, nullptr);
}

}  // namespace dev
}  // namespace xt
