// Attention over the paged int8 cache for prompts: many query rows a sequence,
// bound by the tensor cores, where attend.cu's split by tokens is bound by the
// conversion of the cache's bytes.  The mathematics and the roundings are the
// same (attend.cu).  Two chunks of 2048 new tokens behind 2048, 32 query heads
// over 8 of 128: 259 us, 532 TFLOP/s.  A query tile's token tile takes 4000 to
// 4500 cycles of its SM, as if the two query tiles' softmaxes ran one after the
// other, and about 1050 of products: the tensor pipe is busy 26% of the time, the
// issue slots 47%; warps wait for their loads from TMEM and shared memory.
//
// One CTA has 256 packed query rows (new token, head of the group) of one kv
// head, as two tiles of 128, and walks over the cache in tiles of 128 tokens:
//
//   warps 0-3, 4-7   softmax of query tile 0 and 1, one row a thread: scores
//                    from TMEM, weights as f16 back to TMEM over the scores'
//                    columns; they also divide and store the result.  Warps 0
//                    and 4 issue their tile's tcgen05.mma: S = Q K^T (both in
//                    shared memory) and O += P V (P in TMEM, V read N-major)
//   warps 8-11, 12-15  load the int8 rows of the keys and of the values and
//                    turn them into f16 in shared memory (128-byte swizzle,
//                    two stages); one such group for both was the bottleneck
//
// Where there are few segments a cluster of up to eight CTAs has each: they share
// out its token tiles, leave their f32 sums in shared memory and join a share of
// the rows each (16384 rows of one sequence and 4096 tokens: 124 us alone, 79 in
// clusters of two; 2048 rows 122 and 32).
//
// Registers go where the rows are: 168 a softmax thread, 88 a converting one.
// While one query tile's softmax runs, the tensor cores work for the other.
// The scores of the next token tile go to the same columns as the weights that
// the product before it reads: the MMAs of one thread execute in order.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <type_traits>

#include "attend.cuh"
#include "batch.cuh"
#include "pdl.cuh"
#include "sm100.cuh"
#include "vec.cuh"

namespace xt {
namespace dev {
namespace {

using namespace sm100;

constexpr int kTokens = 128;  // tokens of a tile
constexpr int kTileRows = 128, kRows = 2 * kTileRows;
constexpr int kThreads = 16 * 32;
constexpr int kSoftmaxRegs = 168, kConvertRegs = 88;  // 256 threads each: the 64 K registers of the launch at 128
constexpr int kScaleSlots = 4;
enum : uint32_t { kErrSoftmaxWait = 0x304, kErrConvertWait = 0x305 };

template <int DP>
struct Layout {
  static constexpr int kHalf = 128 * 128;            // 128 rows of 128 bytes: 64 dims
  static constexpr int kMatrix = DP / 64 * kHalf;    // 128 rows of DP f16
  static constexpr int kQuery = 0;                   // two tiles
  static constexpr int kKeys = 2 * kMatrix;          // two stages
  static constexpr int kValues = 4 * kMatrix;        // two stages
  static constexpr int kScales = 6 * kMatrix;        // kScaleSlots x (128 keys', 128 values')
  static constexpr int kBars = kScales + kScaleSlots * 2 * kTokens * 4;
  static constexpr int kBytes = kBars + 256 + 1024;  // barriers and the like, alignment
};

struct Bars {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], o_full[2], drain[2];
  uint64_t scales_full[kScaleSlots];
  float most[kScaleSlots][4];  // largest value scale of a tile, a converting warp each
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Bars) <= 256 + 64, "the barriers' room");

// ---- packed f32 arithmetic: two values an instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Four f32 values at a shared-memory address, as two pairs.
__device__ __forceinline__ void lds_pairs(uint64_t (&v)[2], uint32_t at) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v[0]), "=l"(v[1]) : "r"(at));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Waits for a phase as mbar_wait does; a whole warp calls.  The limit is
// looked at once in 256 polls, each of which the hardware may suspend; a limit of
// the caller's own (not the default) with every poll, none of which it suspends.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, const Abort& ab, uint32_t code) {
  const uint32_t at = smem_addr(bar);
  const uint32_t own = ab.limit < kWaitLimitCycles;
  uint64_t t0 = 0;
  while (true) {
#pragma unroll 1
    for (int poll = own ? 255 : 0; poll < 256; ++poll) {
      uint32_t ok;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 q, %3, 0;\n\t"
          "@q mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "@!q mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(at), "r"(parity), "r"(own)
          : "memory");
      if (__any_sync(0xffffffffu, ok)) return true;  // the phase is over for every lane, then
    }
    if (__any_sync(0xffffffffu, *ab.flag != 0)) return false;
    const uint64_t now = clock64();
    bool late = false;
    if (t0 == 0)
      t0 = now;
    else
      late = now - t0 > ab.limit;
    if (__any_sync(0xffffffffu, late)) {
      *ab.flag = 1;
      atomicCAS(ab.error_word, 0u, code);
      return false;
    }
  }
}

// D[tmem] (+)= A[tmem] * B[smem], f16 inputs, f32 accumulate.
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One CTA's work: 256 packed rows from ``row0`` of a sequence's kv head, over
// token tiles [lo, hi).
struct Work {
  Sequence seq;
  const int32_t* table;  // its pages
  int head, row0, rows;  // rows that there are
  int lo, hi;
};

template <int DP, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) attend_prompt(const __grid_constant__ AttendDev p, int slots) {
  using L = Layout<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars& bars = *reinterpret_cast<Bars*>(smem + L::kBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const CacheView& cache = p.a.cache;
  const int dim = cache.dim, rank = static_cast<int>(blockIdx.x) % p.cluster;

  griddep_launch_dependents();
  griddep_wait();

  // --- which rows.  The last slots, which see the most tokens, come first.
  Work work;
  {
    const int index_of = static_cast<int>(blockIdx.x) / p.cluster;
    const int slot = slots - 1 - index_of / cache.heads;
    work.head = index_of % cache.heads;
    auto base = [&](int start, int i) { return first_slot(start, i, p.group, kRows); };
    const Found found = find_sequence(p.a.batch, cache.page, slot, base);
    const int b = found.b;
    work.seq = found.seq;
    work.table = p.a.batch.table + b * p.a.batch.table_stride;
    const int64_t index = slot - base(found.start, b);
    if (found.fall) {
      refuse_batch<__nv_bfloat16>(p);
      return;
    }
    if (!work.seq.ok) {
      if (threadIdx.x == 0) atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
      if (index == 0) refuse_sequence<__nv_bfloat16>(p, b, work.head, threadIdx.x, kThreads);
      return;
    }
    const int64_t row0 = index * kRows, all = static_cast<int64_t>(work.seq.count) * p.group;
    if (index < 0 || row0 >= all) return;
    work.row0 = static_cast<int>(row0);
    work.rows = static_cast<int>(min(all - row0, static_cast<int64_t>(kRows)));
    const int before = work.seq.length - work.seq.count;
    const int pos_first = before + p.group_div.quot(work.row0);
    const int pos_last = before + p.group_div.quot(work.row0 + work.rows - 1);
    // 64 bits: with more new tokens than tokens the first position is negative
    const int64_t seen_from = p.a.window > 0 ? static_cast<int64_t>(pos_first) - p.a.window + 1 : 0;
    work.lo = seen_from > 0 ? static_cast<int>(seen_from) / kTokens : 0;
    work.hi = pos_last < 0 ? work.lo : max(pos_last / kTokens + 1, work.lo);
    // a cluster's CTAs share them out (and returned together above)
    const int all_tiles = work.hi - work.lo, first = all_tiles * rank / p.cluster;
    work.hi = work.lo + all_tiles * (rank + 1) / p.cluster;
    work.lo += first;
  }
  const int tiles = work.hi - work.lo;
  const int queries = work.rows > kTileRows ? 2 : 1;  // query tiles that have rows

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], 128);
      mbar_init(&bars.k_empty[i], queries);
      mbar_init(&bars.v_full[i], 128);
      mbar_init(&bars.v_empty[i], queries);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.drain[i], 1);
    }
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(&bars.scales_full[i], 256);
    bars.abort = 0;
    fence_barrier_init();
  }
  if (warp == 15) {
    tmem_alloc(&bars.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  const Abort ab{&bars.abort, p.a.error_word, wait_limit_or_default(p.a.wait_limit_cycles)};
  // TMEM columns: scores and weights of the two query tiles, then outputs
  auto score_at = [&](int w) { return tmem + w * 128; };
  auto out_at = [&](int w) { return tmem + 256 + w * 128; };

  // Where a cluster shares the tokens: a query tile's f32 sums in the rooms of the
  // keys (tile 0) and of the values (tile 1), and in its own room each row's
  // (exponent of the sums, sum of the weights)
  auto part_at = [&](int row, int chunk) {  // four dims
    return reinterpret_cast<float*>(smem + L::kKeys + (row >> 7) * 2 * L::kMatrix + (row & 127) * DP * 4 + ((chunk ^ (row & 7)) << 4));
  };
  auto part_sum = [&](int row) { return reinterpret_cast<float2*>(smem + L::kQuery + (row >> 7) * L::kMatrix) + (row & 127); };

  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int w = warp >> 2;
    if (w < queries) {
      const int local = w * kTileRows + (threadIdx.x & 127);  // the thread's row; its TMEM lane modulo 128
      const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21;      // lane offset 32 * (warp & 3)
      const int packed = work.row0 + local;
      const int i = p.group_div.quot(packed);
      const int pos = work.seq.length - work.seq.count + i;
      const float cap = p.a.softcap;

      // --- the query rows as f16 times 2^(10 - exponent of the row's largest
      // magnitude).  DP / 8 lanes have a row, 16 bytes each: asynchronous copies
      // to where the row's f16 will be, turned there.  The loops here and at the
      // end stay short: they run once a CTA, and straight code that is not in the
      // instruction cache took 12 cycles an instruction (9000 for this part).
      constexpr int kRowLanes = DP / 8, kWarpRows = 32 / kRowLanes, kSteps = 32 / kWarpRows;
      const int part = lane % kRowLanes, sub = lane / kRowLanes;
      const int warp_row = w * kTileRows + (warp & 3) * 32;  // the warp's first row
      // the lane's part of the warp's rows, kWarpRows apart
      struct Rows {
        int at, token, head;  // packed row (of the CTA), its new token and head of the group
      };
      const bool part_there = part * 8 < dim;
      auto first_row = [&] {
        const int at = warp_row + sub, token = p.group_div.quot(work.row0 + at);
        return Rows{at, token, work.row0 + at - token * p.group};
      };
      auto next_row = [&](Rows& row) {
        row.at += kWarpRows;
        row.head += kWarpRows;
        if (row.head < p.group) return;
        const int tokens = p.group >= kWarpRows ? 1 : p.group_div.quot(row.head);
        row.token += tokens;
        row.head -= tokens * p.group;
      };
      auto offset = [&](const Rows& row, int64_t token_stride, int64_t head_stride) {
        return static_cast<int64_t>(work.seq.first + row.token) * token_stride +
               static_cast<int64_t>(work.head * p.group + row.head) * head_stride + part * 8;
      };
      const uint32_t base = smem_addr(smem);
      float row_scale = 0.0f;
      {
        auto place = [&](int x) {
          const int r = (warp & 3) * 32 + x * kWarpRows + sub;
          return base + L::kQuery + w * L::kMatrix + part / 8 * L::kHalf + r * 128 + (((part & 7) ^ (r & 7)) << 4);
        };
        Rows row = first_row();
#pragma unroll 2
        for (int x = 0; x < kSteps; ++x) {
          const bool there = row.at < work.rows && part_there;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place(x)),
                       "l"(static_cast<const __nv_bfloat16*>(p.a.q) + (there ? offset(row, p.a.q_token, p.a.q_head) : 0)),
                       "r"(there ? 16 : 0)
                       : "memory");
          next_row(row);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");  // each lane reads back what it copied itself
#pragma unroll 4
        for (int x = 0; x < kSteps; ++x) {
          uint32_t v[4];
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(place(x)));
          float top = 0.0f;
#pragma unroll
          for (int y = 0; y < 4; ++y) top = max3(top, fabsf(bf16_lo(v[y])), fabsf(bf16_hi(v[y])));
#pragma unroll
          for (int o = kRowLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 11), 254);
          const float up = __uint_as_float(static_cast<uint32_t>(264 - e) << 23 | (p.a.scale < 0.0f ? 0x80000000u : 0u));
          const float down = __uint_as_float(static_cast<uint32_t>(e - 10) << 23) * fabsf(p.a.scale) *
                             (CAP ? 1.0f / cap : kLog2e);
          // to the thread that has the row
          const float mine = __shfl_sync(0xffffffffu, down, lane % kWarpRows * kRowLanes);
          if (lane / kWarpRows == x) row_scale = mine;
          uint32_t h[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) h[y] = pack_half2(bf16_lo(v[y]) * up, bf16_hi(v[y]) * up);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(place(x)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3])
                       : "memory");
        }
        fence_proxy_async_smem();
      }

      // --- the tile's products, issued by its first warp
      constexpr uint32_t kScoreDesc = instr_desc(1, 0, 0, 0, 0, 128, kTokens);
      constexpr uint32_t kOutDesc = instr_desc(1, 0, 0, 0, 1, 128, DP);
      auto score = [&](int j) {  // S = Q K^T of token tile j; false: a wait gave up
        if (!wait_phase(&bars.k_full[j & 1], (j >> 1) & 1, ab, kErrSoftmaxWait)) return false;
        tc_fence_after();
        if (elect_sync()) {
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            const uint64_t q = smem_desc_sw128(base + L::kQuery + w * L::kMatrix + k / 4 * L::kHalf, 16, 1024) + (k & 3) * 2;
            const uint64_t c =
                smem_desc_sw128(base + L::kKeys + (j & 1) * L::kMatrix + k / 4 * L::kHalf, 16, 1024) + (k & 3) * 2;
            umma_bf16(score_at(w), q, c, kScoreDesc, k != 0);
          }
          umma_commit(&bars.s_full[w]);
          umma_commit(&bars.k_empty[j & 1]);
        }
        __syncwarp();
        return true;
      };
      auto output = [&](int j) {  // O += P V of token tile j
        if (!wait_phase(&bars.v_full[j & 1], (j >> 1) & 1, ab, kErrSoftmaxWait)) return false;
        tc_fence_after();
        if (elect_sync()) {
          const uint64_t c = smem_desc_sw128(base + L::kValues + (j & 1) * L::kMatrix, L::kHalf, 1024);
#pragma unroll
          for (int k = 0; k < kTokens / 16; ++k)
            umma_f16_ts(out_at(w), score_at(w) + k * 8, c + k * 128, kOutDesc, (j | k) != 0);
          umma_commit(&bars.v_empty[j & 1]);
          if (j + 1 == tiles) umma_commit(&bars.o_full[w]);
        }
        __syncwarp();
        return true;
      };
      const bool issuer = (warp & 3) == 0;
      auto meet = [&] {  // the tile's four warps
        tc_fence_before();
        named_barrier_sync(1 + w, 128);
        tc_fence_after();
      };

      const uint32_t scores = score_at(w) + quarter, result = out_at(w) + quarter;
      const float factor = cap > 0.0f ? 1.0f : row_scale;
      // Weights are 2^(score - ref + up): ``up`` (10 - the exponent of the
      // values' scales, within -60 .. 100) brings weight * value scale near 2^10
      // in f16; the sum carries it too, which takes it out of the result again.
      float ref = kNone, up = 0.0f, value_limit = 0.0f;
      bool value_set = false, ok = true;
      uint64_t sum = pack2(0.0f, 0.0f);
      const int pos_min = __shfl_sync(0xffffffffu, pos, 0);  // of the warp's rows
      const int pos_max = __shfl_sync(0xffffffffu, pos, 31);
      const int window = p.a.window > 0 ? p.a.window : INT_MAX;
      uint32_t key_scales = 0, value_scales = 0;  // shared-memory addresses
      int token0 = 0;

      // Chunk c (32 tokens) of a tile: scores from TMEM, weights to TMEM.
      auto chunk = [&](auto is_open, int j, int c, float most) {
        constexpr bool kOpen = decltype(is_open)::value;
        uint32_t r[32];
        tmem_ld_32x32b_x32(scores + c * 32, r);
        tmem_wait_ld();
        const uint32_t ks = key_scales + c * 128, vs = value_scales + c * 128;
        uint64_t y[16];
        auto exponents = [&](float less) {  // the largest of y = score + less
          const uint64_t by = pack2(factor, factor), add = pack2(less, less);
          float top = -INFINITY;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            uint64_t k[2];
            lds_pairs(k, ks + x * 16);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint64_t z = mul2(pack2(__uint_as_float(r[4 * x + 2 * h]), __uint_as_float(r[4 * x + 2 * h + 1])), k[h]);
              if constexpr (CAP) {
                float a, b;
                unpack2(z, a, b);
                z = pack2(tanh_fast(a * row_scale) * (cap * kLog2e), tanh_fast(b * row_scale) * (cap * kLog2e));
              }
              z = fma2(z, by, add);
              float a, b;
              unpack2(z, a, b);
              if constexpr (!kOpen) {
                const int back = pos - (token0 + c * 32 + 4 * x + 2 * h);  // tokens behind the query
                if (back < 0 || back >= window) a = -INFINITY;
                if (back < 1 || back - 1 >= window) b = -INFINITY;
                z = pack2(a, b);
              }
              top = max3(top, a, b);
              y[2 * x + h] = z;
            }
          }
          return top;
        };
        // The reference follows a row's maximum only when that has risen by
        // more than 2^4, and the values' exponent only when a weight could
        // leave f16's range.
        float top = exponents(up - ref);
        if (__any_sync(0xffffffffu, top > up + 4.0f || most > value_limit)) {
          top = exponents(0.0f);
          int e = kOpen ? static_cast<int>(__float_as_uint(most) >> 23) : 0;  // an open tile's tokens are all seen
#pragma unroll
          for (int x = 0; x < (kOpen ? 0 : 8); ++x) {
            uint64_t v[2];
            lds_pairs(v, vs + x * 16);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float a, b, va, vb;
              unpack2(y[2 * x + h], a, b);
              unpack2(v[h], va, vb);
              const int ea = static_cast<int>(__float_as_uint(va) >> 23 & 255);
              const int eb = static_cast<int>(__float_as_uint(vb) >> 23 & 255);
              if (a > -INFINITY && ea < 255) e = max(e, ea);
              if (b > -INFINITY && eb < 255) e = max(e, eb);
            }
          }
          float f = 1.0f;  // of what the row has so far
          if (top > ref) {
            const float now = top + 2.0f;  // room, so that it need not move again soon
            f = exp2_fast(ref - now);
            ref = now;
          }
          if (e > 0) {
            const float now = 10.0f - static_cast<float>(min(max(e, 37), 197) - 127);
            if (!value_set || now < up) {
              f *= exp2_fast(now - up);
              up = now;
              value_limit = exp2_fast(11.0f - up);
            }
            value_set = true;
          }
          sum = mul2(sum, pack2(f, f));
          if (__any_sync(0xffffffffu, f != 1.0f)) {
            // the output so far (the scores being there, the products before them are done) ...
            if (j > 0) {
#pragma unroll 1
              for (int d = 0; d < DP; d += 16) {
                uint32_t o[16];
                tmem_ld_x16(result + d, o);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                tmem_st_x16(result + d, o);
              }
            }
            // ... and the tile's earlier weights
            tmem_wait_st();
#pragma unroll 1
            for (int d = 0; d < c; ++d) {
              uint32_t o[16];
              tmem_ld_x16(scores + d * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 16; ++x) {
                const float2 v = unpack_half2(o[x]);
                o[x] = pack_half2(v.x * f, v.y * f);
              }
              tmem_st_x16(scores + d * 16, o);
            }
          }
          exponents(up - ref);
        }
        uint32_t weights[16];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          uint64_t v[2];
          lds_pairs(v, vs + x * 16);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float a, b;
            unpack2(y[2 * x + h], a, b);
            const uint64_t e2 = pack2(exp2_fast(a), exp2_fast(b));
            sum = add2(sum, e2);
            float wa, wb;
            unpack2(mul2(e2, v[h]), wa, wb);
            if constexpr (!kOpen) {  // a token that is not seen may have any scale
              if (a == -INFINITY) wa = 0.0f;
              if (b == -INFINITY) wb = 0.0f;
            }
            weights[2 * x + h] = pack_half2(wa, wb);
          }
        }
        tmem_st_x16(scores + c * 16, weights);
      };

      meet();  // the query tile stands in shared memory
      if (issuer && tiles > 0) ok = score(0);
      for (int j = 0; j < tiles; ++j) {
        // A warp whose wait gave up touches no more of the tensor memory and issues
        // no more products; it still meets the others of its query tile.
        ok = ok && wait_phase(&bars.s_full[w], j & 1, ab, kErrSoftmaxWait);
        ok = ok && wait_phase(&bars.scales_full[j % kScaleSlots], (j / kScaleSlots) & 1, ab, kErrSoftmaxWait);
        tc_fence_after();
        if (!ok) {
          meet();
          continue;
        }
        key_scales = base + L::kScales + (j % kScaleSlots) * 2 * kTokens * 4;
        value_scales = key_scales + kTokens * 4;
        const float* most4 = bars.most[j % kScaleSlots];
        const float most = fmaxf(fmaxf(most4[0], most4[1]), fmaxf(most4[2], most4[3]));
        token0 = (work.lo + j) * kTokens;
        // every row of the warp sees all of the tile's tokens
        if (token0 + kTokens - 1 <= pos_min && pos_max - token0 < window) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) chunk(std::true_type{}, j, c, most);
        } else {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) chunk(std::false_type{}, j, c, most);
        }
        tmem_wait_st();
        meet();
        if (issuer) {
          ok = output(j);
          if (ok && j + 1 < tiles) ok = score(j + 1);
        }
      }

      // --- the result: output over the sum
      if (tiles > 0) ok = ok && wait_phase(&bars.o_full[w], 0, ab, kErrSoftmaxWait);
      if (issuer && !ok) {
        // what was issued still ends before the memory goes
        if (elect_sync()) umma_commit(&bars.drain[w]);
        __syncwarp();
        mbar_wait_drain(&bars.drain[w], 0, 500000000ull);
      }
      tc_fence_after();
      const bool there = ok && tiles > 0;  // the tensor memory holds the result
      float s0, s1;
      unpack2(sum, s0, s1);
      s0 += s1;
      if (p.cluster > 1) {
        named_barrier_sync(3, queries * 128);  // the products of both tiles are done
#pragma unroll 1
        for (int d = 0; d < DP; d += 32) {
          uint32_t r[32];
          if (there) {
            tmem_ld_32x32b_x32(result + d, r);
            tmem_wait_ld();
          }
#pragma unroll
          for (int h = 0; h < 8; ++h)
            *reinterpret_cast<uint4*>(part_at(local, d / 4 + h)) =
                there ? make_uint4(r[4 * h], r[4 * h + 1], r[4 * h + 2], r[4 * h + 3]) : make_uint4(0, 0, 0, 0);
        }
        // the weights carry 2^(up - ref); a wait that gave up leaves NaN
        *part_sum(local) = make_float2(ref - up, ok ? s0 : __int_as_float(0x7fc00000));
      } else {
        const float over = s0 > 0.0f || s0 != s0 ? 1.0f / s0 : 0.0f;
        const uint32_t none = ok ? 0u : 0x7fc07fc0u;  // a wait that gave up leaves NaN
        // the row's values to the query tile's room (its last product is done), from
        // where DP / 8 lanes store each row
        uint8_t* room = smem + L::kQuery + w * L::kMatrix + (warp & 3) * 32 * DP * 2;
#pragma unroll 1
        for (int d = 0; d < DP; d += 32) {
          uint32_t r[32];
          if (there) {
            tmem_ld_32x32b_x32(result + d, r);
            tmem_wait_ld();
          }
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
              v[x] = there ? pack_bf16(__uint_as_float(r[8 * h + 2 * x]) * over, __uint_as_float(r[8 * h + 2 * x + 1]) * over) : none;
            *reinterpret_cast<uint4*>(room + lane * DP * 2 + (((d / 8 + h) ^ (lane & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        __syncwarp();
        Rows row = first_row();
#pragma unroll 4
        for (int x = 0; x < kSteps; ++x) {
          const int at = x * kWarpRows + sub;
          const uint4 v = *reinterpret_cast<const uint4*>(room + at * DP * 2 + ((part ^ (at & 7)) << 4));
          if (row.at < work.rows && part_there)
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.a.out) + offset(row, p.a.out_token, p.a.out_head)) = v;
          next_row(row);
        }
      }
      tc_fence_before();
    }
    if (p.cluster > 1) {
      cluster_sync();
      // --- each CTA joins a share of the rows, four dims a thread
      for (int item = rank * 256 + threadIdx.x; item < work.rows * (DP / 4); item += p.cluster * 256) {
        const int row = item / (DP / 4), part = item % (DP / 4);
        if (part * 4 >= dim) continue;
        float top = 2.0f * kNone;
        for (int c = 0; c < p.cluster; ++c) top = fmaxf(top, cluster_load2(part_sum(row), c).x);
        float s = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = 0; c < p.cluster; ++c) {
          const float2 sums = cluster_load2(part_sum(row), c);
          const float4 v = cluster_load4(part_at(row, part), c);
          const float by = exp2_fast(sums.x - top);
          s += sums.y * by;
          y[0] += v.x * by, y[1] += v.y * by, y[2] += v.z * by, y[3] += v.w * by;
        }
        const float over = s > 0.0f || s != s ? 1.0f / s : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= over;
        const int token = p.group_div.quot(work.row0 + row), head = work.row0 + row - token * p.group;
        Vec<__nv_bfloat16, 4>::store(static_cast<__nv_bfloat16*>(p.a.out) +
                                         static_cast<int64_t>(work.seq.first + token) * p.a.out_token +
                                         static_cast<int64_t>(work.head * p.group + head) * p.a.out_head + part * 4, y);
      }
      cluster_sync();  // no CTA goes while another reads its memory
    }
  } else {
    // ------------------------------------------------------------- converting
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
    const bool keys = warp < 12;
    const int me = threadIdx.x & 127, wv = warp & 3;
    const int8_t* data = keys ? cache.k : cache.v;
    const float* data_scales = keys ? cache.k_scale : cache.v_scale;
    uint8_t* matrices = smem + (keys ? L::kKeys : L::kValues);
    uint64_t* full = keys ? bars.k_full : bars.v_full;
    uint64_t* empty = keys ? bars.k_empty : bars.v_empty;
    constexpr int kChunks = DP / 16;               // 16-byte chunks of an int8 row
    constexpr int kAtOnce = 128 / kChunks;         // rows that the 128 threads take at once
    constexpr int kTurns = kTokens / kAtOnce;
    // lanes so that a quarter of a warp stores to eight different bank groups
    const int chunk = DP == 128 ? (lane & 3) | (lane >> 3 & 1) << 2 : lane & 3;
    const int my_row = DP == 128 ? wv * 4 + ((lane >> 2 & 1) | (lane >> 4 & 1) << 1) : wv * 8 + (lane >> 2);
    int4 x[kTurns];
    float scale = 0.0f;  // of the thread's own token: 0 behind the end, NaN of a bad page

    // A token's page and row, from those of kAtOnce tokens before it.
    auto step = [&](int& index, int& row) {
      row += kAtOnce;
      if (row < cache.page) return;
      const int pages = cache.page >= kAtOnce ? 1 : p.page_div.quot(row);
      index += pages;
      row -= pages * cache.page;
    };
    // (page, head) of a token as looked up: -1: behind the end, -2: a page outside the cache
    auto line_of = [&](int id, int token) {
      if (token >= work.seq.length) return -1;
      if (id >= 0 && id < cache.pages) return id * cache.heads + work.head;
      atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
      return -2;
    };
    const uint32_t line_bytes = static_cast<uint32_t>(cache.page) * dim;
    auto fetch = [&](int j) {
      const int token0 = (work.lo + j) * kTokens;
      const int first = p.page_div.quot(token0 + my_row), first_row = token0 + my_row - first * cache.page;
      const int own = p.page_div.quot(token0 + me), own_row = token0 + me - own * cache.page;
      int id[kTurns], index = first, row = first_row;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        id[i] = token0 + i * kAtOnce + my_row < work.seq.length ? work.table[index] : 0;
        step(index, row);
      }
      const int own_id = token0 + me < work.seq.length ? work.table[own] : 0;
      index = first, row = first_row;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int line = line_of(id[i], token0 + i * kAtOnce + my_row);
        x[i] = make_int4(0, 0, 0, 0);
        if (line >= 0 && chunk * 16 < dim)
          x[i] = *reinterpret_cast<const int4*>(data + static_cast<uint64_t>(static_cast<uint32_t>(line)) * line_bytes +
                                                static_cast<uint32_t>(row * dim + chunk * 16));
        step(index, row);
      }
      const int line = line_of(own_id, token0 + me);
      scale = line >= 0 ? data_scales[static_cast<uint64_t>(static_cast<uint32_t>(line)) * static_cast<uint32_t>(p.blocks) +
                                      p.block_div.quot(own_row)]
                        : line == -1 ? 0.0f : __int_as_float(0x7fc00000);
    };
    if (tiles > 0) fetch(0);
    for (int j = 0; j < tiles; ++j) {
      const int stage = j & 1;
      if (!wait_phase(&empty[stage], ((j >> 1) & 1) ^ 1, ab, kErrConvertWait)) break;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int row = i * kAtOnce + my_row;
        uint8_t* to = matrices + stage * L::kMatrix + chunk / 4 * L::kHalf + row * 128;
        const uint32_t u[4] = {static_cast<uint32_t>(x[i].x) ^ 0x80808080u, static_cast<uint32_t>(x[i].y) ^ 0x80808080u,
                               static_cast<uint32_t>(x[i].z) ^ 0x80808080u, static_cast<uint32_t>(x[i].w) ^ 0x80808080u};
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4*>(to + ((((chunk & 3) * 2 + h) ^ (row & 7)) << 4)) =
              make_uint4(bytes_to_half2<kLow>(u[2 * h]), bytes_to_half2<kHigh>(u[2 * h]),
                         bytes_to_half2<kLow>(u[2 * h + 1]), bytes_to_half2<kHigh>(u[2 * h + 1]));
      }
      fence_proxy_async_smem();
      mbar_arrive(&full[stage]);
      // a slot's softmax is done: the products of tile j - 2, whose stage this was, came behind it
      const int slot = j % kScaleSlots;
      reinterpret_cast<float*>(smem + L::kScales)[slot * 2 * kTokens + (keys ? 0 : kTokens) + me] = scale;
      if (!keys) {
        float most = scale < INFINITY ? scale : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (lane == 0) bars.most[slot][wv] = most;
        __syncwarp();
      }
      mbar_arrive(&bars.scales_full[slot]);
      if (j + 1 < tiles) fetch(j + 1);
    }
    if (p.cluster > 1) {
      cluster_sync();
      cluster_sync();
    }
  }
  __syncthreads();
  if (warp == 15) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP, bool CAP>
cudaError_t launch_dims(const AttendDev& p, cudaStream_t stream) {
  static std::atomic<bool> allowed[kMaxDevices];
  const cudaError_t e = allow_smem(attend_prompt<DP, CAP>, Layout<DP>::kBytes, allowed);
  if (e != cudaSuccess) return e;
  const int64_t slots = first_slot(p.a.batch.tokens, p.a.batch.seqs, p.group, kRows);
  PdlLaunch launch(dim3(static_cast<unsigned>(slots * p.a.cache.heads * p.cluster)), dim3(kThreads), Layout<DP>::kBytes, stream,
                   p.cluster);
  return launch(attend_prompt<DP, CAP>, p, static_cast<int>(slots));
}

}  // namespace

int prompt_clusters(int cluster) {
  // every instance has an SM to itself
  static std::atomic<bool> allowed[kMaxDevices];
  static std::atomic<int> known[3][kMaxDevices];
  auto kernel = attend_prompt<128, false>;
  if (allow_smem(kernel, Layout<128>::kBytes, allowed) != cudaSuccess) return 0;
  return clusters_at_once(kernel, PdlLaunch(dim3(cluster), dim3(kThreads), Layout<128>::kBytes, nullptr, cluster),
                          known[cluster == 8 ? 2 : cluster == 4]);
}

cudaError_t launch_attend_prompt(const AttendDev& p, cudaStream_t stream) {
  const bool cap = p.a.softcap > 0.0f;
  if (p.a.cache.dim <= 64) return cap ? launch_dims<64, true>(p, stream) : launch_dims<64, false>(p, stream);
  return cap ? launch_dims<128, true>(p, stream) : launch_dims<128, false>(p, stream);
}

}  // namespace dev
}  // namespace xt
