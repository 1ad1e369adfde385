// What the kernels of the cache's attention share.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../serve.h"

namespace xt {
namespace dev {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -1e30f;  // reference of a row that has seen no token

struct AttendDev {
  AttendArgs a;
  FastDiv page_div, block_div, group_div;
  int group, blocks;  // query heads a kv head, blocks a page
  float* part;        // [workers][2][rows][dim] partial outputs
  float2* part_ml;    // [workers][2][rows] (reference, sum)
  int64_t workers;
  int cluster;        // CTAs of a segment, where each has a cluster
};

// 2^x, at most 2^-22 of it off; 0 for -inf.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// Two biased bytes (int8 + 128), picked by ``SEL`` from a word, as f16 values:
// the byte lands in the mantissa of 1024, and 1152 is taken off again, exactly.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t biased) {
  const uint32_t h = __byte_perm(biased, 0x64646464u, SEL);
  const uint32_t off = 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr uint32_t kLow = 0x4140u, kHigh = 0x4342u;  // bytes 0, 1 and bytes 2, 3

constexpr int kMaxDevices = 64;

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

// Segments without a scan: sequence b's row tiles of ROWS packed rows stand at
// slots starts[b] * group / ROWS + b on, which leaves room for all of them.
__host__ __device__ inline int64_t first_slot(int64_t start, int b, int group, int rows) { return start * group / rows + b; }

// A sequence whose table is wrong: recorded, and its rows of a kv head are NaN.
template <class T>
__device__ __forceinline__ void refuse_sequence(const AttendDev& p, int b, int head, int thread, int threads) {
  if (thread == 0) atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
  const int dim = p.a.cache.dim;
  const int64_t first = max(p.a.batch.starts[b], 0), end = min(p.a.batch.starts[b + 1], p.a.batch.tokens);
  const int64_t each = static_cast<int64_t>(p.group) * dim;
  for (int64_t i = thread; i < (end - first) * each; i += threads) {
    const int64_t token = first + i / each, h = head * p.group + i % each / dim;
    static_cast<T*>(p.a.out)[token * p.a.out_token + h * p.a.out_head + i % dim] = static_cast<T>(__int_as_float(0x7fc00000));
  }
}

// The tcgen05 kernel for many query rows (attend_prompt.cu): bf16, dim <= 128.
cudaError_t launch_attend_prompt(const AttendDev& p, cudaStream_t stream);

}  // namespace dev
}  // namespace xt
