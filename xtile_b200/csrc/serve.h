// Launch arguments of the serving operators' kernels: the norm that makes
// int8 rows, rotary positions, the int8 paged cache's append and attention,
// and reading int8 data back.  The C entry points (serve.cpp) check the
// arguments; the launchers assume them checked.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

#include "kernels.h"

namespace xt {
namespace dev {

// Codes the serving kernels write to the error word: device-side tables that
// name something outside the arrays they index.  The access is skipped.
enum : uint32_t {
  kErrRopePosition = 0x301,   // a position outside the rotation table
  kErrAppendTable = 0x302,    // append: a length, start or page outside its range
  kErrAttendTable = 0x303,    // attention: likewise
};

// Division of 0 <= n < 2^31 by a positive d < 2^31 as a multiply and a shift.
struct FastDiv {
  uint32_t d, shift;
  uint64_t mul;
  __host__ void set(uint32_t div) {
    d = div;
    shift = 0;
    while ((uint64_t{1} << shift) < div) ++shift;
    shift += 31;
    mul = (uint64_t{1} << shift) / div + 1;
  }
  __device__ __forceinline__ uint32_t quot(uint32_t n) const { return static_cast<uint32_t>((n * mul) >> shift); }
};

// ---------------------------------------------------------------- rms norm
struct NormArgs {
  const void* x;
  const void* residual;   // null: none
  const void* weight;
  void* y;
  void* sum;              // null: x + residual is not stored
  float* scales;          // one a row, for int8 rows
  int64_t rows, cols;
  int64_t x_stride, residual_stride, y_stride, sum_stride;  // elements between rows
  uint8_t elem;           // of x, residual and sum: kF32 or kBF16
  uint8_t weight_elem;    // kF32 or kBF16
  uint8_t y_elem;         // kF32, kBF16 or kI8
  float eps;
};
cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t stream);

// -------------------------------------------------------------------- rope
struct RopeArgs {
  const void* x;
  void* y;
  const int32_t* positions;
  const float2* table;    // [table_rows, rot / 2] of (cos, sin)
  int64_t tokens, heads, dim, rot, table_rows;
  int64_t x_token, x_head, y_token, y_head;  // strides in elements
  uint8_t elem, y_elem;
  uint8_t interleaved, inverse;
  uint32_t* error_word;
};
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t stream);

// ------------------------------------------------------------- paged cache
struct CacheView {
  int8_t* k;              // [pages, heads, page, dim]
  int8_t* v;
  float* k_scale;         // [pages, heads, page / block]
  float* v_scale;
  int64_t pages;
  int heads, page, dim, block;
};

// A ragged batch: sequence b's new tokens are rows starts[b] .. starts[b+1]-1,
// the last of its lengths[b] tokens; token j lies in page table[b][j / page].
struct BatchView {
  const int32_t* starts;   // [seqs + 1]
  const int32_t* lengths;  // [seqs]
  const int32_t* table;    // [seqs, table_width], rows table_stride apart
  int seqs, tokens, table_width;
  int64_t table_stride;
};

struct AppendArgs {
  CacheView cache;
  BatchView batch;
  const void* k;
  const void* v;
  int64_t k_token, k_head, v_token, v_head;
  const float2* rope;      // null: keys are stored as they are
  int64_t rot, rope_rows;
  uint8_t elem, interleaved;
  uint32_t* error_word;
};
cudaError_t launch_cache_append(const AppendArgs& a, cudaStream_t stream);

struct AttendArgs {
  CacheView cache;
  BatchView batch;
  const void* q;
  void* out;
  int64_t q_token, q_head, out_token, out_head;
  int q_heads;
  int max_new;             // most new tokens of one sequence, as far as the caller knows
  int window;              // 0: none
  float scale, softcap;    // softcap 0: none
  uint8_t elem;            // of q and out
  void* workspace;
  size_t workspace_bytes;
  uint32_t* error_word;
  uint64_t wait_limit_cycles;  // SM cycles a wait may take before the kernel gives up (0: 2 s)
};
// Bytes of device memory that launch_cache_attention needs beside its arguments.
size_t attend_workspace_bytes(const AttendArgs& a);
cudaError_t launch_cache_attention(const AttendArgs& a, cudaStream_t stream);

// -------------------------------------------------------------- dequantize
struct DequantArgs {
  const int8_t* q;
  const float* scales;
  void* out;
  int64_t n, run;          // n elements, one scale for each run of them
  uint8_t elem;
};
cudaError_t launch_dequantize(const DequantArgs& a, cudaStream_t stream);

}  // namespace dev
}  // namespace xt
