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
// (-1: behind the rotated part, copied as it is).  Neighbouring items' first
// vectors are neighbours, and so are their second ones, so that a warp reads
// and writes whole lines.
struct RopeSpan {
  int first, second, pair;
};

template <int V>
__device__ __forceinline__ RopeSpan rope_span(int c, int rot, int dim, bool interleaved) {
  const int turned = rot / (2 * V);
  if (c >= turned) return {rot + V * (c - turned), rot + V * (c - turned) + (dim - rot) / 2, -1};
  if (V == 1 && interleaved) return {2 * c, 2 * c + 1, c};
  return {V * c, V * c + rot / 2, interleaved ? V * c / 2 : V * c};
}

// (cos, sin) of an item's pairs from the position's row of the table: V pairs
// across the vectors, or V / 2 in the first one and V / 2 in the second.
template <int V>
__device__ __forceinline__ void load_turns(const float2* row, const RopeSpan& span, int rot, bool interleaved, float2 (&cs)[V]) {
  const float2* from = row + max(span.pair, 0);
  if constexpr (V == 1) {
    cs[0] = *from;
  } else {
    const int ahead = interleaved ? rot / 4 - V / 2 : 0;  // from the first vector's last pair to the second's first
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float4 t = *reinterpret_cast<const float4*>(from + j + (j < V / 2 ? 0 : ahead));
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
