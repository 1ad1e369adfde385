// Attention over the paged int8 cache for prompts: many query rows a sequence,
// bound by the tensor cores, where attend.cu's split by tokens is bound by the
// conversion of the cache's bytes.  The mathematics and the roundings are the
// same (attend.cu).
//
// One CTA has 256 packed query rows (new token, head of the group) of one kv
// head, as two tiles of 128, and walks over the cache in tiles of 128 tokens:
//
//   warps 0-3, 4-7   softmax of query tile 0 and 1, one row a thread: scores
//                    from TMEM, weights as f16 back to TMEM over the scores'
//                    columns; they also divide and store the result.  Warps 0
//                    and 4 issue their tile's tcgen05.mma: S = Q K^T (both in
//                    shared memory) and O += P V (P in TMEM, V read N-major)
//   warps 8-11       load the int8 rows, turn them into f16 in shared memory
//                    (128-byte swizzle), two stages each of keys and values
//
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
constexpr int kThreads = 12 * 32;
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
  const int dim = cache.dim;

  griddep_launch_dependents();
  griddep_wait();

  // --- which rows.  Sequence b's row tiles stand from slot starts[b] * group /
  // 256 + b on; the last slots, which see the most tokens, come first.
  Work work;
  {
    const int slot = slots - 1 - static_cast<int>(blockIdx.x) / cache.heads;
    work.head = static_cast<int>(blockIdx.x) % cache.heads;
    auto base = [&](int i) { return static_cast<int64_t>(p.a.batch.starts[i]) * p.group / kRows + i; };
    const int b = last_at_most(p.a.batch.seqs, slot, base);
    work.seq = load_sequence(p.a.batch, cache.page, b);
    work.table = p.a.batch.table + b * p.a.batch.table_stride;
    const int64_t index = slot - base(b);
    if (!work.seq.ok) {
      // its table is wrong: recorded, and its rows are NaN
      if (index != 0) return;
      if (threadIdx.x == 0) atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
      const int64_t first = max(p.a.batch.starts[b], 0), end = min(p.a.batch.starts[b + 1], p.a.batch.tokens);
      const int64_t each = static_cast<int64_t>(p.group) * dim;
      for (int64_t i = threadIdx.x; i < (end - first) * each; i += kThreads) {
        const int64_t token = first + i / each, h = work.head * p.group + i % each / dim;
        static_cast<__nv_bfloat16*>(p.a.out)[token * p.a.out_token + h * p.a.out_head + i % dim] =
            __float2bfloat16(__int_as_float(0x7fc00000));
      }
      return;
    }
    const int64_t row0 = index * kRows, all = static_cast<int64_t>(work.seq.count) * p.group;
    if (index < 0 || row0 >= all) return;
    work.row0 = static_cast<int>(row0);
    work.rows = static_cast<int>(min(all - row0, static_cast<int64_t>(kRows)));
    const int before = work.seq.length - work.seq.count;
    const int pos_first = before + p.group_div.quot(work.row0);
    const int pos_last = before + p.group_div.quot(work.row0 + work.rows - 1);
    const int seen_from = p.a.window > 0 ? pos_first - p.a.window + 1 : 0;
    work.lo = seen_from > 0 ? seen_from / kTokens : 0;
    work.hi = pos_last < 0 ? work.lo : max(pos_last / kTokens + 1, work.lo);
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
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(&bars.scales_full[i], 128);
    bars.abort = 0;
    fence_barrier_init();
  }
  if (warp == 11) {
    tmem_alloc(&bars.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  const Abort ab{&bars.abort, p.a.error_word, kWaitLimitCycles};
  // TMEM columns: scores and weights of the two query tiles, then outputs
  auto score_at = [&](int w) { return tmem + w * 128; };
  auto out_at = [&](int w) { return tmem + 256 + w * 128; };

  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    const int w = warp >> 2;
    if (w < queries) {
      const int local = (threadIdx.x & 127), row = w * kTileRows + local;  // TMEM lane = local
      const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21;      // lane offset 32 * (warp & 3)
      const int packed = work.row0 + row;
      const int i = p.group_div.quot(packed);
      const bool there = row < work.rows;
      const int pos = work.seq.length - work.seq.count + i;
      const int q_head = work.head * p.group + packed - i * p.group;
      const float cap = p.a.softcap;

      // --- the query row as f16 times 2^(10 - exponent of its largest magnitude)
      float row_scale;
      {
        const __nv_bfloat16* from = static_cast<const __nv_bfloat16*>(p.a.q) +
                                    static_cast<int64_t>(work.seq.first + i) * p.a.q_token +
                                    static_cast<int64_t>(q_head) * p.a.q_head;
        float top = 0.0f;
        if (there)
          for (int d = 0; d < dim; d += 4) {
            float v[4];
            Vec<__nv_bfloat16, 4>::load(from + d, v);
            top = fmaxf(fmaxf(fmaxf(top, fabsf(v[0])), fmaxf(fabsf(v[1]), fabsf(v[2]))), fabsf(v[3]));
          }
        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 11), 243);
        const float up = __uint_as_float(static_cast<uint32_t>(264 - e) << 23 | (p.a.scale < 0.0f ? 0x80000000u : 0u));
        row_scale = __uint_as_float(static_cast<uint32_t>(e - 10) << 23) * fabsf(p.a.scale) *
                    (cap > 0.0f ? 1.0f / cap : kLog2e);
        uint8_t* to = smem + L::kQuery + w * L::kMatrix + local * 128;
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) {
          uint32_t h[4] = {0, 0, 0, 0};
          if (there && c * 8 < dim) {
            float v[4], u[4];
            Vec<__nv_bfloat16, 4>::load(from + c * 8, v);
            Vec<__nv_bfloat16, 4>::load(from + c * 8 + 4, u);
            h[0] = pack_half2(v[0] * up, v[1] * up), h[1] = pack_half2(v[2] * up, v[3] * up);
            h[2] = pack_half2(u[0] * up, u[1] * up), h[3] = pack_half2(u[2] * up, u[3] * up);
          }
          *reinterpret_cast<uint4*>(to + c / 8 * L::kHalf + (((c & 7) ^ (local & 7)) << 4)) =
              make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async_smem();
      }

      // --- the tile's products, issued by its first warp
      constexpr uint32_t kScoreDesc = instr_desc(1, 0, 0, 0, 0, 128, kTokens);
      constexpr uint32_t kOutDesc = instr_desc(1, 0, 0, 0, 1, 128, DP);
      const uint32_t base = smem_addr(smem);
      auto score = [&](int j) {  // S = Q K^T of token tile j; false: a wait gave up
        if (!__all_sync(0xffffffffu, mbar_wait(&bars.k_full[j & 1], (j >> 1) & 1, ab, kErrSoftmaxWait))) return false;
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
        if (!__all_sync(0xffffffffu, mbar_wait(&bars.v_full[j & 1], (j >> 1) & 1, ab, kErrSoftmaxWait))) return false;
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
      const float *key_scales = nullptr, *value_scales = nullptr;
      int token0 = 0;

      // Chunk c (32 tokens) of a tile: scores from TMEM, weights to TMEM.
      auto chunk = [&](auto is_open, int j, int c, float most) {
        constexpr bool kOpen = decltype(is_open)::value;
        uint32_t r[32];
        tmem_ld_32x32b_x32(scores + c * 32, r);
        tmem_wait_ld();
        const float4* ks = reinterpret_cast<const float4*>(key_scales + c * 32);
        const float4* vs = reinterpret_cast<const float4*>(value_scales + c * 32);
        uint64_t y[16];
        float less = up - ref;
        // The reference follows a row's maximum only when that has risen by
        // more than 2^4, and the values' exponent only when a weight could
        // leave f16's range, so the first turn is mostly the only one; the
        // second takes the scores themselves.
#pragma unroll 1
        for (int turn = 0;; ++turn) {
          const uint64_t by = pack2(factor, factor), add = pack2(less, less);
          float top = -INFINITY;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float4 k = ks[x];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint64_t z = mul2(pack2(__uint_as_float(r[4 * x + 2 * h]), __uint_as_float(r[4 * x + 2 * h + 1])),
                                h ? pack2(k.z, k.w) : pack2(k.x, k.y));
              if constexpr (CAP) {
                float a, b;
                unpack2(z, a, b);
                z = pack2(tanhf(a * row_scale) * (cap * kLog2e), tanhf(b * row_scale) * (cap * kLog2e));
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
          if (turn == 2) break;
          if (turn == 0) {
            if (!__any_sync(0xffffffffu, top > up + 4.0f || most > value_limit)) break;
            less = 0.0f;
            continue;
          }
          int e = 0;
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            float a, b;
            unpack2(y[x], a, b);
            const float2 v = reinterpret_cast<const float2*>(vs)[x];
            const int ea = static_cast<int>(__float_as_uint(v.x) >> 23 & 255);
            const int eb = static_cast<int>(__float_as_uint(v.y) >> 23 & 255);
            if (a > -INFINITY && ea < 255) e = max(e, ea);
            if (b > -INFINITY && eb < 255) e = max(e, eb);
          }
          float f = 1.0f;  // of what the row has so far
          if (top > ref) {
            f = exp2_fast(ref - top);
            ref = top;
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
          less = up - ref;
        }
        uint32_t weights[16];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float4 v = vs[x];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float a, b;
            unpack2(y[2 * x + h], a, b);
            const uint64_t e2 = pack2(exp2_fast(a), exp2_fast(b));
            sum = add2(sum, e2);
            float wa, wb;
            unpack2(mul2(e2, h ? pack2(v.z, v.w) : pack2(v.x, v.y)), wa, wb);
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
        // A wait that gives up leaves the rest of the loop to run on whatever is
        // there, without another long wait: the barriers below stay whole.
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[w], j & 1, ab, kErrSoftmaxWait)) && ok;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.scales_full[j % kScaleSlots], (j / kScaleSlots) & 1, ab,
                                               kErrSoftmaxWait)) && ok;
        tc_fence_after();
        key_scales = reinterpret_cast<const float*>(smem + L::kScales) + (j % kScaleSlots) * 2 * kTokens;
        value_scales = key_scales + kTokens;
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
          ok = output(j) && ok;
          if (j + 1 < tiles) ok = score(j + 1) && ok;
        }
      }

      // --- the result: output over the sum
      if (tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_full[w], 0, ab, kErrSoftmaxWait)) && ok;
      tc_fence_after();
      float s0, s1;
      unpack2(sum, s0, s1);
      s0 += s1;
      const float over = s0 > 0.0f || s0 != s0 ? 1.0f / s0 : 0.0f;
      __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.a.out) +
                          static_cast<int64_t>(work.seq.first + i) * p.a.out_token + static_cast<int64_t>(q_head) * p.a.out_head;
#pragma unroll 1
      for (int d = 0; d < dim; d += 16) {
        uint32_t o[16];
        if (tiles > 0) {
          tmem_ld_x16(result + d, o);
          tmem_wait_ld();
        }
        if (!there || !ok) continue;
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
          float v[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) v[y] = tiles > 0 ? __uint_as_float(o[x + y]) * over : 0.0f;
          Vec<__nv_bfloat16, 4>::store(to + d + x, v);
        }
      }
      tc_fence_before();
      if (issuer && *ab.flag) {
        // what was issued still ends before the memory goes
        if (elect_sync()) umma_commit(&bars.drain[w]);
        __syncwarp();
        mbar_wait_drain(&bars.drain[w], 0, 500000000ull);
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------- converting
    const int me = threadIdx.x - 256, wv = warp - 8;
    constexpr int kChunks = DP / 16;               // 16-byte chunks of an int8 row
    constexpr int kAtOnce = 128 / kChunks;         // rows that the 128 threads take at once
    constexpr int kTurns = kTokens / kAtOnce;
    // lanes so that a quarter of a warp stores to eight different bank groups
    const int chunk = DP == 128 ? (lane & 3) | (lane >> 3 & 1) << 2 : lane & 3;
    const int my_row = DP == 128 ? wv * 4 + ((lane >> 2 & 1) | (lane >> 4 & 1) << 1) : wv * 8 + (lane >> 2);
    int64_t from[kTurns];  // offset of the thread's chunk of each of its rows; -1: zeros
    int4 k[kTurns], v[kTurns];
    bool ok = true;

    auto line_of = [&](int token, int& row) -> int64_t {  // (page, head) of a token; -1: none, -2: a bad page
      if (token >= work.seq.length) return -1;
      const int index = p.page_div.quot(token);
      row = token - index * cache.page;
      const int id = work.table[index];
      if (id < 0 || id >= cache.pages) {
        atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
        return -2;
      }
      return static_cast<int64_t>(id) * cache.heads + work.head;
    };
    auto look_up = [&](int j) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        int row = 0;
        const int64_t line = line_of((work.lo + j) * kTokens + i * kAtOnce + my_row, row);
        from[i] = line < 0 || chunk * 16 >= dim ? -1 : (line * cache.page + row) * dim + chunk * 16;
      }
    };
    auto fetch = [&](const int8_t* base, int4 (&to)[kTurns]) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i)
        to[i] = from[i] < 0 ? make_int4(0, 0, 0, 0) : *reinterpret_cast<const int4*>(base + from[i]);
    };
    auto convert = [&](uint8_t* matrix, const int4 (&x)[kTurns]) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int row = i * kAtOnce + my_row;
        uint8_t* to = matrix + chunk / 4 * L::kHalf + row * 128;
        const uint32_t u[4] = {static_cast<uint32_t>(x[i].x) ^ 0x80808080u, static_cast<uint32_t>(x[i].y) ^ 0x80808080u,
                               static_cast<uint32_t>(x[i].z) ^ 0x80808080u, static_cast<uint32_t>(x[i].w) ^ 0x80808080u};
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4*>(to + ((((chunk & 3) * 2 + h) ^ (row & 7)) << 4)) =
              make_uint4(bytes_to_half2<kLow>(u[2 * h]), bytes_to_half2<kHigh>(u[2 * h]),
                         bytes_to_half2<kLow>(u[2 * h + 1]), bytes_to_half2<kHigh>(u[2 * h + 1]));
      }
    };
    // the scales of the thread's own token (0 behind the end, NaN of a bad page)
    float ks = 0.0f, vs = 0.0f;
    auto fetch_scales = [&](int j) {
      int row = 0;
      const int64_t line = line_of((work.lo + j) * kTokens + me, row);
      const int64_t at = line * p.blocks + p.block_div.quot(row);
      ks = line >= 0 ? cache.k_scale[at] : line == -1 ? 0.0f : __int_as_float(0x7fc00000);
      vs = line >= 0 ? cache.v_scale[at] : line == -1 ? 0.0f : __int_as_float(0x7fc00000);
    };
    if (tiles > 0) {
      look_up(0);
      fetch(cache.k, k);
      fetch(cache.v, v);
      fetch_scales(0);
    }
    for (int j = 0; j < tiles; ++j) {
      const int stage = j & 1;
      const uint32_t phase = (j >> 1) & 1;
      ok = mbar_wait_warp(&bars.k_empty[stage], phase ^ 1, ab, kErrConvertWait);
      if (!ok) break;
      convert(smem + L::kKeys + stage * L::kMatrix, k);
      fence_proxy_async_smem();
      mbar_arrive(&bars.k_full[stage]);
      // a slot's softmax is done: the scores of tile j - 2, whose stage this was, came behind it
      float* scales = reinterpret_cast<float*>(smem + L::kScales) + (j % kScaleSlots) * 2 * kTokens;
      scales[me] = ks;
      scales[kTokens + me] = vs;
      float most = vs < INFINITY ? vs : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (lane == 0) bars.most[j % kScaleSlots][wv] = most;
      __syncwarp();
      mbar_arrive(&bars.scales_full[j % kScaleSlots]);
      const bool more = j + 1 < tiles;
      if (more) {
        look_up(j + 1);
        fetch(cache.k, k);
        fetch_scales(j + 1);
      }
      ok = mbar_wait_warp(&bars.v_empty[stage], phase ^ 1, ab, kErrConvertWait);
      if (!ok) break;
      convert(smem + L::kValues + stage * L::kMatrix, v);
      fence_proxy_async_smem();
      mbar_arrive(&bars.v_full[stage]);
      if (more) fetch(cache.v, v);
    }
  }
  __syncthreads();
  if (warp == 11) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP, bool CAP>
cudaError_t launch_dims(const AttendDev& p, cudaStream_t stream) {
  static std::atomic<bool> allowed[kMaxDevices];
  const cudaError_t e = allow_smem(attend_prompt<DP, CAP>, Layout<DP>::kBytes, allowed);
  if (e != cudaSuccess) return e;
  const int64_t slots = static_cast<int64_t>(p.a.batch.tokens) * p.group / kRows + p.a.batch.seqs;
  PdlLaunch launch(dim3(static_cast<unsigned>(slots * p.a.cache.heads)), dim3(kThreads), Layout<DP>::kBytes, stream);
  return launch(attend_prompt<DP, CAP>, p, static_cast<int>(slots));
}

}  // namespace

cudaError_t launch_attend_prompt(const AttendDev& p, cudaStream_t stream) {
  const bool cap = p.a.softcap > 0.0f;
  if (p.a.cache.dim <= 64) return cap ? launch_dims<64, true>(p, stream) : launch_dims<64, false>(p, stream);
  return cap ? launch_dims<128, true>(p, stream) : launch_dims<128, false>(p, stream);
}

}  // namespace dev
}  // namespace xt
