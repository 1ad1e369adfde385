// Attention over the paged int8 cache: for each new token's head
//
//   z_j = scale * ks_j * (q . kq_j)          [z_j = cap * tanh(z_j / cap)]
//   out = sum_j softmax_j(z) * vs_j * vq_j
//
// over the tokens j that the query sees (causal from the end of its sequence,
// and a window if one is set).  A token's reads are 2 dim int8 bytes a kv
// head, so single-token decoding is bound by HBM.
//
// Work is cut into units of 16 tokens of one (sequence, kv head, 16 packed
// query rows) segment; a row is a (new token, head of the group) pair, so the
// heads of a group share the cache's reads.  The units of all segments stand
// in one line, and each warp of a grid that fills the GPU takes an equal run
// of it: ragged lengths, a single long sequence and many short ones all load
// every SM alike.  A warp works alone, without a CTA barrier: it streams its
// own tiles with cp.async through its own ring in shared memory, runs the two
// products on mma.sync m16n8k16 in f16 and keeps the running maximum, sum and
// output of its rows in registers.  Segments that several warps share are
// joined by a second kernel from f32 partial results.
//
// int8 values are exact in f16, and so is a bf16 query divided by a power of
// two that brings its row's largest magnitude near 2^10 (elements under 2^-35
// of that lose bits).  The scales of the tokens' blocks stay outside the
// products: the key's multiplies the score in f32, the value's the weight,
// which is rounded once to f16 (11 bits) on its way into the second product.
// f32 queries go in as two f16 terms, and so do their weights: 22 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../serve.h"
#include "batch.cuh"
#include "pdl.cuh"
#include "vec.cuh"

namespace xt {
namespace dev {
namespace {

constexpr int kTile = 16;  // tokens of a unit, and query rows of a segment
constexpr float kLog2e = 1.4426950408889634f;

template <int DP, bool F32>
struct Shape {
  static constexpr int kWarps = DP <= 128 ? 4 : 2;
  static constexpr int kStages = DP <= 64 ? 8 : DP <= 128 ? 4 : 3;
  static constexpr int kCtas = F32 ? 2 : 3;                       // CTAs an SM
  static constexpr int kStageBytes = 2 * kTile * DP + 2 * kTile * 4;  // keys, values, their scales
  static constexpr bool kQueryInSmem = F32 || DP > 128;           // else its fragments stay in registers
  static constexpr int kQueryBytes = kQueryInSmem ? (DP / 16) * 512 * (F32 ? 2 : 1) : 0;
  static constexpr int kWarpBytes = kStages * kStageBytes + kQueryBytes;
};

struct AttendDev {
  AttendArgs a;
  FastDiv page_div, block_div, group_div;
  int group;
  float* part;     // [workers][2][16][dim] partial outputs
  float2* part_ml; // [workers][2][16] (reference, sum)
  int64_t workers;
};

// The units of sequence b: kv heads x row tiles x token tiles [lo, hi).
struct Segments {
  Sequence seq;
  int row_tiles, lo, hi;
  __device__ __forceinline__ int64_t units(int heads) const {
    return static_cast<int64_t>(heads) * row_tiles * (hi - lo);
  }
};

__device__ __forceinline__ Segments load_segments(const AttendDev& p, int b) {
  Segments g;
  g.seq = load_sequence(p.a.batch, p.a.cache.page, b);
  if (!g.seq.ok) atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
  g.row_tiles = static_cast<int>((static_cast<int64_t>(g.seq.count) * p.group + kTile - 1) / kTile);
  const int64_t first_seen = p.a.window > 0 ? static_cast<int64_t>(g.seq.length) - g.seq.count - p.a.window + 1 : 0;
  g.lo = first_seen > 0 ? static_cast<int>(first_seen) / kTile : 0;
  g.hi = (g.seq.length + kTile - 1) / kTile;
  if (g.lo > g.hi) g.lo = g.hi;
  return g;
}

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Units of all sequences, and of those before ``b``.  A whole warp calls.
__device__ __forceinline__ int64_t count_units(const AttendDev& p, int b, int64_t* before) {
  int64_t total = 0, front = 0;
  for (int i = threadIdx.x & 31; i < p.a.batch.seqs; i += 32) {
    const int64_t u = load_segments(p, i).units(p.a.cache.heads);
    total += u;
    if (i < b) front += u;
  }
  *before = warp_sum64(front);
  return warp_sum64(total);
}

// A place in the line of units.
struct Cursor {
  Segments seg;
  int b, head, row_tile, tile;

  __device__ __forceinline__ void seek(const AttendDev& p, int64_t u) {
    const int lane = threadIdx.x & 31, heads = p.a.cache.heads;
    int64_t front = 0;
    b = 0;
    for (int base = 0; base < p.a.batch.seqs; base += 32) {
      const int i = base + lane;
      const int64_t mine = i < p.a.batch.seqs ? load_segments(p, i).units(heads) : 0;
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
    seg = load_segments(p, b);
    const int tiles = seg.hi - seg.lo;
    const int64_t at = u - front, line = at / tiles;
    tile = seg.lo + static_cast<int>(at - line * tiles);
    head = static_cast<int>(line / seg.row_tiles);
    row_tile = static_cast<int>(line - static_cast<int64_t>(head) * seg.row_tiles);
  }

  // The next unit; there must be one.
  __device__ __forceinline__ void advance(const AttendDev& p) {
    if (++tile < seg.hi) return;
    tile = seg.lo;
    if (++row_tile < seg.row_tiles) return;
    row_tile = 0;
    if (++head < p.a.cache.heads) return;
    head = 0;
    do {
      ++b;
      seg = load_segments(p, b);
    } while (seg.units(1) == 0 && b + 1 < p.a.batch.seqs);
    tile = seg.lo;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// 4 bytes, or 4 zero bytes where ``bytes`` is 0.
__device__ __forceinline__ void cp_async4(uint32_t to, const void* from, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// c += a b for 16 x 16 f16 a, 16 x 8 f16 b, f32 c.
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// Two biased bytes (int8 + 128), picked by ``sel`` from w, as f16 values: the
// byte lands in the mantissa of 1024, and 1152 is taken off again, exactly.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t biased) {
  const uint32_t h = __byte_perm(biased, 0x64646464u, SEL);
  const uint32_t off = 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr uint32_t kLow = 0x4140u, kHigh = 0x4342u;  // bytes 0, 1 and bytes 2, 3

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What two values leave after their rounding to f16, as f16.
__device__ __forceinline__ uint32_t rest_half2(float lo, float hi, uint32_t rounded) {
  const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
  return pack_half2(lo - r.x, hi - r.y);
}

// Shared-memory places of 16-byte chunk ``c`` of a tile's token ``row``,
// permuted so that the eight lanes of each quarter of a warp-wide 16-byte read
// meet eight different bank groups: key reads take chunk 4 j + t of tokens g
// (two tokens a quarter), value reads chunk g of tokens 2 t.
template <int DP>
__device__ __forceinline__ uint32_t key_place(int row, int c) {
  return row * DP + ((DP >= 128 ? c ^ ((row & 1) << 2) : c) << 4);
}
template <int DP>
__device__ __forceinline__ uint32_t value_place(int row, int c) {
  return row * DP + ((DP >= 128 ? c ^ (((row >> 1) & 3) << 1) : c ^ (((row >> 1) & 1) << 1)) << 4);
}

template <int DP, bool F32>
__global__ void __launch_bounds__(Shape<DP, F32>::kWarps * 32, Shape<DP, F32>::kCtas)
    attend_units(const __grid_constant__ AttendDev p) {
  using S = Shape<DP, F32>;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  constexpr int kSteps = DP / 16;    // k16 steps of the score product
  constexpr int kOut = DP / 8;       // n8 tiles of the output
  constexpr int kChunks = DP / 16;   // 16-byte chunks of a token
  constexpr int kRowsAtOnce = 32 / kChunks;
  extern __shared__ __align__(128) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + warp * S::kWarpBytes;
  const uint32_t ring_addr = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  uint4* query = reinterpret_cast<uint4*>(ring + S::kStages * S::kStageBytes);
  const CacheView& cache = p.a.cache;
  const int dim = cache.dim;

  // chunks behind dim are never loaded; they stay zero
  if (dim < DP) {
    for (int i = lane; i < S::kStages * S::kStageBytes / 16; i += 32)
      reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  griddep_launch_dependents();
  griddep_wait();

  int64_t unused;
  const int64_t total = count_units(p, 0, &unused);
  const int64_t per = (total + p.workers - 1) / p.workers;
  const int64_t worker = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
  const int64_t begin = worker * per, end = begin + per < total ? begin + per : total;
  if (begin >= end) return;

  Cursor at;
  at.seek(p, begin);
  Cursor ahead = at;
  int64_t to_issue = end - begin;

  // --- loading: lane l & 15 looks up the page of token l of the tile to come
  int page_id = 0, page_row = 0;
  bool token_there = false;
  auto look_up = [&] {
    const int token = ahead.tile * kTile + (lane & 15);
    token_there = token < ahead.seg.seq.length;
    const int index = p.page_div.quot(token);
    page_row = token - index * cache.page;
    page_id = token_there ? p.a.batch.table[ahead.b * p.a.batch.table_stride + index] : 0;
  };
  auto issue = [&](int stage) {
    if (to_issue > 0) {
      const uint32_t base = ring_addr + stage * S::kStageBytes;
      const bool bad = page_id < 0 || page_id >= cache.pages;
      const bool there = token_there && !bad;
      const int64_t line = static_cast<int64_t>(bad ? 0 : page_id) * cache.heads + ahead.head;
      const int64_t row_at = line * cache.page + page_row;
      const int64_t scale_at = line * (cache.page / cache.block) + p.block_div.quot(page_row);
      const uint32_t scale_to = base + 2 * kTile * DP + lane * 4;
      if (token_there && bad) {
        // a page outside the cache: recorded, and NaN for whoever attends to it
        atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(scale_to), "r"(0x7fc00000u) : "memory");
      } else {
        cp_async4(scale_to, (lane < kTile ? cache.k_scale : cache.v_scale) + (there ? scale_at : 0), there ? 4 : 0);
      }
      const unsigned rows_there = __ballot_sync(0xffffffffu, there);
      const int chunk = lane % kChunks;
#pragma unroll
      for (int i = 0; i < kTile / kRowsAtOnce; ++i) {
        const int row = i * kRowsAtOnce + lane / kChunks;
        const int64_t from = __shfl_sync(0xffffffffu, row_at, row) * dim + chunk * 16;
        if (chunk * 16 >= dim) continue;
        // rows behind the sequence's end are left as they are: finite int8, and their weight is 0
        if (!(rows_there >> row & 1)) continue;
        cp_async16(base + key_place<DP>(row, chunk), cache.k + from);
        cp_async16(base + kTile * DP + value_place<DP>(row, chunk), cache.v + from);
      }
      if (--to_issue > 0) {
        ahead.advance(p);
        look_up();
      }
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue(i);

  // --- the segment at hand
  uint4 qf[S::kQueryInSmem ? 1 : kSteps];
  float o[kOut][4];
  float ref[2], sum[2], row_scale[2];   // rows g and g + 8: reference of the exponents, sum of the weights
  int row_pos[2];                       // positions of their queries
  int value_exp = 0;                    // the weights carry vs 2^(10 - value_exp); set by the first token seen
  bool value_set = false, whole = true; // whole: the segment's first unit is this worker's
  const float cap = p.a.softcap;

  auto row_of = [&](int r, int* token) {  // packed row r of the row tile: its new token and query head, or -1
    const int packed = at.row_tile * kTile + r;
    const int i = p.group_div.quot(packed);
    *token = i;
    return i < at.seg.seq.count ? at.head * p.group + packed - i * p.group : -1;
  };

  auto start_segment = [&] {
    whole = at.tile == at.seg.lo;
    value_set = false;
    value_exp = 0;
#pragma unroll
    for (int i = 0; i < kOut; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    float q[2][kSteps][4];
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      int i;
      const int head = row_of(g + 8 * r, &i);
      row_pos[r] = head < 0 ? -1 : at.seg.seq.length - at.seg.seq.count + i;
      const T* from = static_cast<const T*>(p.a.q) + static_cast<int64_t>(at.seg.seq.first + i) * p.a.q_token +
                      static_cast<int64_t>(head) * p.a.q_head;
      top[r] = 0.0f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int d = 64 * (s / 4) + 16 * t + 4 * (s % 4);  // the lane's four dims of this step
#pragma unroll
        for (int e = 0; e < 4; ++e) q[r][s][e] = 0.0f;
        if (head >= 0 && d < dim) Vec<T, 4>::load(from + d, q[r][s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) top[r] = fmaxf(top[r], fabsf(q[r][s][e]));
      }
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      // the row times 2^(10 - exponent of its largest magnitude)
      const int e = min(max(static_cast<int>(__float_as_uint(top[r]) >> 23), 11), 243);
      const float up = __uint_as_float(static_cast<uint32_t>(264 - e) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(e - 10) << 23);
      row_scale[r] = down * p.a.scale * (cap > 0.0f ? 1.0f / cap : kLog2e);
      ref[r] = -INFINITY;
      sum[r] = 0.0f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) q[r][s][e2] *= up;
    }
    if constexpr (S::kQueryInSmem) __syncwarp();
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint4 f = make_uint4(pack_half2(q[0][s][0], q[0][s][1]), pack_half2(q[1][s][0], q[1][s][1]),
                                 pack_half2(q[0][s][2], q[0][s][3]), pack_half2(q[1][s][2], q[1][s][3]));
      if constexpr (S::kQueryInSmem) {
        query[s * 32 + lane] = f;  // read back by this lane alone
        if constexpr (F32)
          query[(kSteps + s) * 32 + lane] =
              make_uint4(rest_half2(q[0][s][0], q[0][s][1], f.x), rest_half2(q[1][s][0], q[1][s][1], f.y),
                         rest_half2(q[0][s][2], q[0][s][3], f.z), rest_half2(q[1][s][2], q[1][s][3], f.w));
      } else {
        qf[s] = f;
      }
    }
  };

  auto finish_segment = [&](bool last_unit) {
    const float up = __uint_as_float(static_cast<uint32_t>(value_exp + 117) << 23);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      int i;
      const int head = row_of(g + 8 * r, &i);
      if (head < 0) continue;
      constexpr int kSpan = DP >= 128 ? 32 : 16;  // consecutive dims that the lane holds of a row
      const bool done = whole && last_unit;
      const float by = done ? (sum[r] > 0.0f || sum[r] != sum[r] ? up / sum[r] : 0.0f) : up;
      const int64_t slot = worker * 2 + (whole ? 1 : 0);
      T* to = static_cast<T*>(p.a.out) + static_cast<int64_t>(at.seg.seq.first + i) * p.a.out_token +
              static_cast<int64_t>(head) * p.a.out_head;
      float* part = p.part + (slot * kTile + g + 8 * r) * dim;
#pragma unroll
      for (int h = 0; h < kOut * 2 / kSpan; ++h) {
        // C columns 2 t and 2 t + 1 of n-tile i stand for dims (2 t) kSpan / 2 + i and (2 t + 1) kSpan / 2 + i
#pragma unroll
        for (int d = 0; d < kSpan; d += 4) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int x = d + e, nt = h * (kSpan / 2) + x % (kSpan / 2);
            y[e] = o[nt][2 * r + x / (kSpan / 2)] * by;
          }
          const int dim_at = h * 4 * kSpan + t * kSpan + d;
          if (dim_at >= dim) continue;
          if (done)
            Vec<T, 4>::store(to + dim_at, y);
          else
            *reinterpret_cast<float4*>(part + dim_at) = make_float4(y[0], y[1], y[2], y[3]);
        }
      }
      if (!done && t == 0) p.part_ml[slot * kTile + g + 8 * r] = make_float2(ref[r], sum[r]);
    }
  };

  start_segment();
  int stage = 0;
  for (int64_t u = begin; u < end; ++u) {
    cp_async_wait<S::kStages - 2>();
    __syncwarp();
    issue(stage == 0 ? S::kStages - 1 : stage - 1);
    const uint32_t keys = ring_addr + stage * S::kStageBytes;
    const uint32_t values = keys + kTile * DP;
    const float* scales = reinterpret_cast<const float*>(ring + stage * S::kStageBytes + 2 * kTile * DP);

    // --- scores: two n8 tiles of tokens
    float z[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[n][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < DP / 64; ++j) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(keys + key_place<DP>(8 * n + g, 4 * j + t)));
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t biased = w[s] ^ 0x80808080u;
          const uint32_t b0 = bytes_to_half2<kLow>(biased), b1 = bytes_to_half2<kHigh>(biased);
          const int step = 4 * j + s;
          if constexpr (S::kQueryInSmem) {
            mma_16816(z[n], query[step * 32 + lane], b0, b1);
            if constexpr (F32) mma_16816(z[n], query[(kSteps + step) * 32 + lane], b0, b1);
          } else {
            mma_16816(z[n], qf[step], b0, b1);
          }
        }
      }
    }

    // --- weights
    const int token0 = at.tile * kTile;
    float vs[2][2];
    float top[2] = {-INFINITY, -INFINITY};
    bool some = false;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const float2 ks = *reinterpret_cast<const float2*>(scales + 8 * n + 2 * t);
      const float2 v = *reinterpret_cast<const float2*>(scales + kTile + 8 * n + 2 * t);
      vs[n][0] = v.x, vs[n][1] = v.y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = z[n][e] * ((e & 1) ? ks.y : ks.x) * row_scale[e >> 1];
        if (cap > 0.0f) x = tanhf(x) * (cap * kLog2e);
        const int j = token0 + 8 * n + 2 * t + (e & 1), pos = row_pos[e >> 1];
        const bool seen = j <= pos && (p.a.window == 0 || j > pos - p.a.window);
        z[n][e] = seen ? x : -INFINITY;
        some |= seen;
        top[e >> 1] = fmaxf(top[e >> 1], z[n][e]);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
    }
    // The reference of a row's exponents follows its maximum only when that has
    // risen by more than 2^4, so that most units leave the output as it is.
    const bool rise = top[0] > ref[0] + 4.0f || top[1] > ref[1] + 4.0f;
    if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float now = fmaxf(ref[r], top[r]);
        const float f = now == -INFINITY ? 1.0f : exp2f(ref[r] - now);
        ref[r] = now;
        sum[r] *= f;
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
          o[i][2 * r] *= f;
          o[i][2 * r + 1] *= f;
        }
      }
    }
    // The values' scales enter the weights as multiples of a power of two that
    // the first scale seen sets, and that changes only where a weight would
    // leave f16's range.  2^10 of room below the largest weights keeps f16's
    // subnormals (2^-24 apart) at 2^-34 of them.
    auto exponent_of_scales = [&] {
      int e = 0;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const bool seen = z[n][c] != -INFINITY || z[n][c + 2] != -INFINITY;
          const int b = static_cast<int>(__float_as_uint(vs[n][c]) >> 23 & 255);
          if (seen && b < 255) e = max(e, b);
        }
      return __reduce_max_sync(0xffffffffu, e);
    };
    if (!value_set && __any_sync(0xffffffffu, some)) {
      const int e = exponent_of_scales();
      value_set = e > 0;
      value_exp = e > 0 ? min(max(e, 11), 250) - 127 : 0;
    }
    float shift = __uint_as_float(static_cast<uint32_t>(137 - value_exp) << 23);
    float w[2][4];
    bool large = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float base = ref[r] == -INFINITY ? 0.0f : ref[r];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float x = z[n][2 * r + c];
          const float e = exp2f(x - base);
          sum[r] += e;
          w[n][2 * r + c] = x == -INFINITY ? 0.0f : e * (vs[n][c] * shift);
          large |= w[n][2 * r + c] > 60000.0f;
        }
    }
    if (__any_sync(0xffffffffu, large)) {
      const int e = min(max(exponent_of_scales(), 11), 250) - 127;
      if (e > value_exp) {
        const float f = __uint_as_float(static_cast<uint32_t>(max(127 + value_exp - e, 0)) << 23);
        value_exp = e;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) w[n][c] *= f;
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[i][c] *= f;
      }
    }
    uint4 wf, wl;
    wf = make_uint4(pack_half2(w[0][0], w[0][1]), pack_half2(w[0][2], w[0][3]), pack_half2(w[1][0], w[1][1]),
                    pack_half2(w[1][2], w[1][3]));
    if constexpr (F32)
      wl = make_uint4(rest_half2(w[0][0], w[0][1], wf.x), rest_half2(w[0][2], w[0][3], wf.y),
                      rest_half2(w[1][0], w[1][1], wf.z), rest_half2(w[1][2], w[1][3], wf.w));

    // --- output: the lane's tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
    constexpr int kWords = DP >= 128 ? 4 : 2;  // words of a token that one read brings
#pragma unroll
    for (int h = 0; h < DP / (32 * kWords); ++h) {
      uint32_t v[4][kWords];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 2 * t + (i & 1) + 8 * (i >> 1);
        if constexpr (DP >= 128) {
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v[i][0]), "=r"(v[i][1]), "=r"(v[i][kWords - 2]), "=r"(v[i][kWords - 1])
                       : "r"(values + value_place<DP>(row, 8 * h + g)));
        } else {
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                       : "=r"(v[i][0]), "=r"(v[i][1])
                       : "r"(values + value_place<DP>(row, g >> 1) + (g & 1) * 8));
        }
#pragma unroll
        for (int k = 0; k < kWords; ++k) v[i][k] ^= 0x80808080u;
      }
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // bytes 2 half and 2 half + 1 of two tokens, side by side
          const uint32_t a = __byte_perm(v[0][k], v[1][k], half ? 0x7362u : 0x5140u);
          const uint32_t b = __byte_perm(v[2][k], v[3][k], half ? 0x7362u : 0x5140u);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int nt = h * 4 * kWords + 4 * k + 2 * half + e;
            const uint32_t b0 = e ? bytes_to_half2<kHigh>(a) : bytes_to_half2<kLow>(a);
            const uint32_t b1 = e ? bytes_to_half2<kHigh>(b) : bytes_to_half2<kLow>(b);
            if constexpr (F32) {
              // a fresh sum for the unit, added in f32: the tensor cores' own sums round toward zero
              float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_16816(c, wl, b0, b1);
              mma_16816(c, wf, b0, b1);
#pragma unroll
              for (int x = 0; x < 4; ++x) o[nt][x] += c[x];
            } else {
              mma_16816(o[nt], wf, b0, b1);
            }
          }
        }
      }
    }
    stage = stage == S::kStages - 1 ? 0 : stage + 1;

    const bool last_unit = at.tile + 1 == at.seg.hi;
    if (last_unit || u + 1 == end) {
      finish_segment(last_unit);
      if (u + 1 < end) {
        at.advance(p);
        start_segment();
      }
    } else {
      ++at.tile;
    }
  }
  cp_async_wait<0>();
}

// Joins the partial results of the segments that several workers had.  WARPS
// warps have one (new token, query head): each takes every WARPS-th partial.
template <class T, int DP, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) attend_join(const __grid_constant__ AttendDev p) {
  constexpr int kPer = DP / 32;  // dims a lane
  __shared__ float shared_o[WARPS == 1 ? 1 : WARPS][WARPS == 1 ? 1 : DP];
  __shared__ float2 shared_ml[WARPS];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t index = WARPS == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + warp : blockIdx.x;
  if (index >= static_cast<int64_t>(p.a.batch.tokens) * p.a.q_heads) return;
  const int token = static_cast<int>(index / p.a.q_heads), q_head = static_cast<int>(index % p.a.q_heads);
  const int b = last_at_most(p.a.batch.seqs, token, [&](int i) { return static_cast<int64_t>(p.a.batch.starts[i]); });
  const Segments seg = load_segments(p, b);
  const int i = token - seg.seq.first;
  T* out = static_cast<T*>(p.a.out) + static_cast<int64_t>(token) * p.a.out_token + static_cast<int64_t>(q_head) * p.a.out_head;
  if (!seg.seq.ok) {
    // its table is wrong: recorded, and its rows are NaN
    for (int d = lane; d < p.a.cache.dim; d += 32) {
      const float nan[1] = {__int_as_float(0x7fc00000)};
      Vec<T, 1>::store(out + d, nan);
    }
    return;
  }
  if (i < 0 || i >= seg.seq.count) return;  // a row of no sequence
  int64_t front;
  const int64_t total = count_units(p, b, &front);
  const int64_t per = (total + p.workers - 1) / p.workers;
  const int head = q_head / p.group;
  const int packed = i * p.group + q_head % p.group;
  const int tiles = seg.hi - seg.lo;
  if (tiles == 0) {
    for (int d = lane; d < p.a.cache.dim; d += 32) {
      const float zero[1] = {0.0f};
      Vec<T, 1>::store(out + d, zero);
    }
    return;
  }
  const int64_t u0 = front + (static_cast<int64_t>(head) * seg.row_tiles + packed / kTile) * tiles;
  const int64_t first = u0 / per, last = (u0 + tiles - 1) / per;
  if (first == last) return;  // one worker had it all, and has written it
  const int row = packed % kTile, dim = p.a.cache.dim;
  auto slot_of = [&](int64_t c) { return (c * 2 + (c == first ? 1 : 0)) * kTile + row; };

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

template <int DP, bool F32>
int64_t worker_count(int sms) {
  using S = Shape<DP, F32>;
  return static_cast<int64_t>(sms) * S::kCtas * S::kWarps;
}

constexpr int kMaxDevices = 64;

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

// Grants ``kernel`` its shared memory, once a device.
template <class K>
cudaError_t allow_smem(K kernel, int bytes, std::atomic<bool> (&done)[kMaxDevices]) {
  int device = 0;
  cudaGetDevice(&device);
  const bool keep = device >= 0 && device < kMaxDevices;
  if (keep && done[device]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && keep) done[device] = true;
  return e;
}

template <int DP, bool F32>
cudaError_t launch_shape(AttendDev& p, cudaStream_t stream) {
  using S = Shape<DP, F32>;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  const int sms = sm_count();
  p.workers = worker_count<DP, F32>(sms);
  p.part = static_cast<float*>(p.a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part + p.workers * 2 * kTile * p.a.cache.dim);
  constexpr int kSmem = S::kWarps * S::kWarpBytes;
  static_assert(kSmem * S::kCtas <= 227 * 1024, "the CTAs of an SM share 227 KB");
  static std::atomic<bool> allowed[kMaxDevices];
  cudaError_t e = allow_smem(attend_units<DP, F32>, kSmem, allowed);
  if (e != cudaSuccess) return e;
  PdlLaunch launch(dim3(static_cast<unsigned>(sms * S::kCtas)), dim3(S::kWarps * 32), kSmem, stream);
  e = launch(attend_units<DP, F32>, p);
  if (e != cudaSuccess) return e;
  const int64_t rows = static_cast<int64_t>(p.a.batch.tokens) * p.a.q_heads;
  // a row's partials are spread over eight warps where the rows alone would not fill the GPU
  if (rows <= 4 * sms) {
    PdlLaunch join(dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream);
    return join(attend_join<T, DP, 8>, p);
  }
  PdlLaunch join(dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream);
  return join(attend_join<T, DP, 1>, p);
}

}  // namespace

size_t attend_workspace_bytes(int dim, int, int, int, int, int, uint8_t elem) {
  const int sms = sm_count();
  const bool f32 = elem == kF32;
  const int64_t workers = dim <= 64    ? (f32 ? worker_count<64, true>(sms) : worker_count<64, false>(sms))
                          : dim <= 128 ? (f32 ? worker_count<128, true>(sms) : worker_count<128, false>(sms))
                                       : (f32 ? worker_count<256, true>(sms) : worker_count<256, false>(sms));
  return static_cast<size_t>(workers) * 2 * kTile * (dim + 2) * sizeof(float);
}

cudaError_t launch_cache_attention(const AttendArgs& a, cudaStream_t stream) {
  if (a.batch.tokens <= 0 || a.batch.seqs <= 0 || a.q_heads <= 0) return cudaSuccess;
  AttendDev p{};
  p.a = a;
  p.group = a.q_heads / a.cache.heads;
  p.page_div.set(static_cast<uint32_t>(a.cache.page));
  p.block_div.set(static_cast<uint32_t>(a.cache.block));
  p.group_div.set(static_cast<uint32_t>(p.group));
  const int dim = a.cache.dim;
  if (a.elem == kF32)
    return dim <= 64 ? launch_shape<64, true>(p, stream)
                     : dim <= 128 ? launch_shape<128, true>(p, stream) : launch_shape<256, true>(p, stream);
  return dim <= 64 ? launch_shape<64, false>(p, stream)
                   : dim <= 128 ? launch_shape<128, false>(p, stream) : launch_shape<256, false>(p, stream);
}

}  // namespace dev
}  // namespace xt
