// 16-byte and single-element access to f32 and bf16 arrays as f32 values, and
// the int8 rounding that the serving kernels share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

namespace xt {
namespace dev {

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Two f32 rounded to bf16 (to nearest even), ``lo`` in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// V consecutive elements as f32: 16-byte loads where V fills them, else one
// element.  ``p`` is aligned to the access.
template <class T, int V>
struct Vec;

template <>
struct Vec<float, 4> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};

template <>
struct Vec<__nv_bfloat16, 4> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(t.x), v[1] = bf16_hi(t.x), v[2] = bf16_lo(t.y), v[3] = bf16_hi(t.y);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
  }
};

template <>
struct Vec<__nv_bfloat16, 8> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    v[0] = bf16_lo(t.x), v[1] = bf16_hi(t.x), v[2] = bf16_lo(t.y), v[3] = bf16_hi(t.y);
    v[4] = bf16_lo(t.z), v[5] = bf16_hi(t.z), v[6] = bf16_lo(t.w), v[7] = bf16_hi(t.w);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
};

template <>
struct Vec<float, 8> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};

template <>
struct Vec<float, 1> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[1]) { v[0] = *p; }
  static __device__ __forceinline__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
};

template <>
struct Vec<__nv_bfloat16, 1> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[1]) { v[0] = __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16_rn(v[0]); }
};

// The larger of two values; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// int8 scale of values whose largest magnitude is ``top``: top / 127, and 0
// (all values round to 0) for a top under 1e-36, whose reciprocal would leave
// f32's range.  A top that is NaN or infinite gives a NaN scale, so that whoever
// reads the values back sees it (of an infinite one the bytes have no sign).
constexpr float kQuantTiny = 1e-36f;
__device__ __forceinline__ float quant_scale(float top) {
  return top < kQuantTiny ? 0.0f : top < INFINITY ? top * (1.0f / 127.0f) : __int_as_float(0x7fc00000);
}
__device__ __forceinline__ float quant_inverse(float scale) { return scale > 0.0f ? 1.0f / scale : 0.0f; }

// x * inverse rounded to the nearest whole number (ties to even) in the low
// byte of a float's bits: 1.5 * 2^23 leaves no bits behind the point.  For
// |x * inverse| < 2^22, so for any value under its block's scale; NaN and
// infinities give some byte (their scale is NaN).
__device__ __forceinline__ uint32_t quantize_bits(float x, float inverse) {
  return __float_as_uint(__fmaf_rn(x, inverse, 12582912.0f));
}
__device__ __forceinline__ int quantize(float x, float inverse) { return static_cast<int8_t>(quantize_bits(x, inverse)); }

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040u), __byte_perm(c, d, 0x0040u), 0x5410u);
}

// Four int8 values times ``ratio`` (at most 1), rounded again.
__device__ __forceinline__ int requantize(int w, float ratio) {
  auto value = [&](int shift) { return static_cast<float>(static_cast<int8_t>(w >> shift)); };
  return static_cast<int>(low_bytes(quantize_bits(value(0), ratio), quantize_bits(value(8), ratio),
                                    quantize_bits(value(16), ratio), quantize_bits(value(24), ratio)));
}

// V values as int8 at ``p`` (aligned to V bytes).
template <int V>
__device__ __forceinline__ void store_i8(int8_t* p, const float (&x)[V], float inverse) {
  if constexpr (V >= 4) {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = low_bytes(quantize_bits(x[4 * i], inverse), quantize_bits(x[4 * i + 1], inverse),
                       quantize_bits(x[4 * i + 2], inverse), quantize_bits(x[4 * i + 3], inverse));
    if constexpr (V == 8)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(p) = w[0];
  } else {
    *p = static_cast<int8_t>(quantize(x[0], inverse));
  }
}

}  // namespace dev
}  // namespace xt
