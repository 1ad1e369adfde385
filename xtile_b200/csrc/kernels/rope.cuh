// Rotary positions on register vectors.  A pair (a, b) of a head turns by the
// angle of its position and frequency:
//
//   a' = a cos - b sin,   b' = a sin + b cos.
//
// Pair i of the first ``rot`` elements is (2i, 2i + 1) in the interleaved
// layout and (i, i + rot/2) in the half layout.
#pragma once

#include <cuda_runtime.h>

#include "vec.cuh"

namespace xt {
namespace dev {

// Where item ``c`` of a head's dim / (2 V) items lives: two vectors of V
// elements, ``first`` and ``second``, and the pair index of its first pair
// (-1: behind the rotated part, copied as it is).
struct RopeSpan {
  int first, second, pair;
};

template <int V>
__device__ __forceinline__ RopeSpan rope_span(int c, int rot, bool interleaved) {
  const int at = 2 * V * c;
  if (at >= rot) return {at, at + V, -1};
  if (interleaved) return {at, at + V, V * c};
  return {V * c, V * c + rot / 2, V * c};
}

// V pairs' (cos, sin).
template <int V>
__device__ __forceinline__ void load_turns(const float2* row, float2 (&cs)[V]) {
  if constexpr (V == 1) {
    cs[0] = *row;
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float4 t = *reinterpret_cast<const float4*>(row + j);
      cs[j] = make_float2(t.x, t.y);
      cs[j + 1] = make_float2(t.z, t.w);
    }
  }
}

__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
  const float x = a * cs.x - b * cs.y;
  b = a * cs.y + b * cs.x;
  a = x;
}

// Rotates an item's vectors: pairs run across (half layout) or along them.
template <int V>
__device__ __forceinline__ void rope_item(float (&first)[V], float (&second)[V], const float2 (&cs)[V], bool interleaved) {
  if (!interleaved) {
#pragma unroll
    for (int j = 0; j < V; ++j) turn(first[j], second[j], cs[j]);
  } else if constexpr (V == 1) {
    turn(first[0], second[0], cs[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      turn(first[j], first[j + 1], cs[j / 2]);
      turn(second[j], second[j + 1], cs[V / 2 + j / 2]);
    }
  }
}

}  // namespace dev
}  // namespace xt
