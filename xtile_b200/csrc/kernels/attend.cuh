// What the kernels of the cache's attention share.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "../serve.h"
#include "pdl.cuh"
#include "sm100.cuh"

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
  int least;          // units a worker takes at least
  int cluster;        // CTAs of a segment, which then has a cluster
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

// What lies at this address in the shared memory of CTA ``rank`` of the cluster.
__device__ __forceinline__ float2 cluster_load2(const float2* p, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(sm100::mapa_shared(sm100::smem_addr(p), rank))
               : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_load4(const float* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(sm100::mapa_shared(sm100::smem_addr(p), rank))
               : "memory");
  return v;
}

// tanh(x) for scores whose weights are rounded to f16: 1 - 2 / (1 + e^2x), at
// most 2^-22 off, and the first terms of its series near 0, where that would
// cancel; 2^-18 of the value at most.  Two chunks of 2048 new tokens behind 2048
// with capped scores took 441 us with tanhf and 405 with this.
__device__ __forceinline__ float tanh_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + exp2_fast(x * (2.0f * kLog2e))));
  const float s = x * x;
  return s < 0.0225f ? x * fmaf(s, fmaf(s, 2.0f / 15.0f, -1.0f / 3.0f), 1.0f) : fmaf(-2.0f, r, 1.0f);
}

// mbar_wait for the attention kernels, whose waits are short: with a limit of the
// caller's own (not the default) a poll does not suspend the warp and is followed
// by a look at the clock, so that a wait of a microsecond can run out.  (One loop
// for both took 129 us where 64 ragged contexts take 122.)
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, const sm100::Abort& ab, uint32_t code) {
  if (ab.limit >= sm100::kWaitLimitCycles) return sm100::mbar_wait(bar, parity, ab, code);
  const uint64_t t0 = clock64();
  while (!sm100::mbar_test_wait(bar, parity)) {
    if (*ab.flag) return false;
    if (clock64() - t0 > ab.limit) {
      *ab.flag = 1;
      atomicCAS(ab.error_word, 0u, code);
      return false;
    }
  }
  return true;
}

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

// Clusters of a launch that the GPU runs at once, asked once a device.
template <class K>
int clusters_at_once(K kernel, PdlLaunch launch, std::atomic<int> (&known)[kMaxDevices]) {
  int device = 0, n = 0;
  cudaGetDevice(&device);
  const bool keep = device >= 0 && device < kMaxDevices;
  if (keep && known[device]) return known[device];
  launch.attrs[0] = launch.attrs[1];  // the question knows no other attribute
  launch.cfg.attrs = launch.attrs;
  launch.cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &launch.cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (keep) known[device] = n;
  return n;
}

// Segments without a scan: sequence b's row tiles of ROWS packed rows stand at
// slots starts[b] * group / ROWS + b on, which leaves room for all of them
// where starts never fall (0 for a start that is negative, whose sequence is
// refused).
__host__ __device__ inline int64_t first_slot(int64_t start, int b, int group, int rows) {
  return (start > 0 ? start : 0) * group / rows + b;
}

// New tokens of a sequence, as far as the caller knows; else their mean.
inline int new_tokens(const AttendDev& p) {
  const int mean = (p.a.batch.tokens + p.a.batch.seqs - 1) / p.a.batch.seqs;
  return p.a.max_new > 0 ? (p.a.max_new < p.a.batch.tokens ? p.a.max_new : p.a.batch.tokens) : mean;
}

// Tokens that a query tile of a sequence sees, at most, as far as the host knows.
inline int64_t longest_seen(const AttendDev& p, int tile) {
  const int64_t room = static_cast<int64_t>(p.a.batch.table_width) * p.a.cache.page;
  if (p.a.window <= 0) return room;
  // a window starts and ends inside a tile
  return std::min<int64_t>(room, static_cast<int64_t>(p.a.window) + new_tokens(p) + tile - 1);
}

// Segments of ``rows`` query rows.
inline int64_t segments_of(const AttendDev& p, int rows) {
  const int64_t tiles = (static_cast<int64_t>(new_tokens(p)) * p.group + rows - 1) / rows;
  return static_cast<int64_t>(p.a.batch.seqs) * p.a.cache.heads * tiles;
}

// A sequence whose table is wrong: its rows of a kv head are NaN.
template <class T>
__device__ __noinline__ void refuse_sequence(const AttendDev& p, int b, int head, int thread, int threads) {
  const int dim = p.a.cache.dim;
  const int64_t first = max(p.a.batch.starts[b], 0), end = min(p.a.batch.starts[b + 1], p.a.batch.tokens);
  const int64_t each = static_cast<int64_t>(p.group) * dim;
  for (int64_t i = thread; i < (end - first) * each; i += threads) {
    const int64_t token = first + i / each, h = head * p.group + i % each / dim;
    static_cast<T*>(p.a.out)[token * p.a.out_token + h * p.a.out_head + i % dim] = static_cast<T>(__int_as_float(0x7fc00000));
  }
}

// Starts that fall: recorded, and every row of the batch is NaN.  Each CTA of the
// grid has a share of them.
template <class T>
__device__ __noinline__ void refuse_batch(const AttendDev& p) {
  if (threadIdx.x == 0) atomicCAS(p.a.error_word, 0u, static_cast<uint32_t>(kErrAttendTable));
  const int dim = p.a.cache.dim;
  const int64_t each = static_cast<int64_t>(p.a.q_heads) * dim;
  for (int64_t token = blockIdx.x; token < p.a.batch.tokens; token += gridDim.x)
    for (int64_t i = threadIdx.x; i < each; i += blockDim.x)
      static_cast<T*>(p.a.out)[token * p.a.out_token + i / dim * p.a.out_head + i % dim] = static_cast<T>(__int_as_float(0x7fc00000));
}

// The tcgen05 kernel for many query rows (attend_prompt.cu): bf16, dim <= 128.
// Each segment of 256 rows has p.cluster CTAs.
cudaError_t launch_attend_prompt(const AttendDev& p, cudaStream_t stream);
int prompt_clusters(int cluster);  // clusters of 2, 4 or 8 CTAs that run at once

}  // namespace dev
}  // namespace xt
