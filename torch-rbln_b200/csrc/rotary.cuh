// Rotary positions, shared by the rotary kernel (rotary.cu) and the kernel
// that rotates, quantises and writes a step's keys (rotary_write.cu).
//
// Pair i of a row at position p turns by the angle p * inv_freq[i]:
//   y1 = m (x1 cos - x2 sin),  y2 = m (x2 cos + x1 sin)
// with (x1, x2) = (x[i], x[i + R/2]) in the half layout and
// (x[2i], x[2i + 1]) in the interleaved one; dimensions past R pass through.
// The factor m scales both (a long-context extension's attention factor).
// The transposed map, which the gradient needs, is the same with sin negated.
#pragma once

#include "common.cuh"

namespace rbln {

// (m cos, m sin) of p * inv_freq. The product has up to 53 + 24 significant
// bits and the angle of a far position many turns, so both are taken in
// double: turns = p * inv_freq / 2 pi, less its nearest whole number, leaves
// at most half a turn, which float holds to 2^-26 of a turn. One evaluation
// serves all heads of a token, so its 64-bit part costs little.
__device__ __forceinline__ float2 rotary_cos_sin(double pos, float inv_freq, float mscale) {
  const double turns = pos * (double)inv_freq * 0.15915494309189535;
  const float part = (float)(turns - rint(turns));
  float s, c;
  sincospif(2.f * part, &s, &c);
  return make_float2(c * mscale, s * mscale);
}

// One item of the vector paths: V consecutive pairs (V = 16 bytes of
// elements), i.e. two 16-byte vectors of a row. Half layout: vectors at
// element c V and R/2 + c V; interleaved, and pass-through items (2 c V >= R)
// in both layouts: 2 c V and 2 c V + V.
struct RotaryItem {
  int e0, e1;  // element offsets of the two vectors
  bool turned;
};
__device__ __forceinline__ RotaryItem rotary_item(int c, int V, int R, bool interleaved) {
  RotaryItem it;
  it.turned = 2 * c * V < R;
  if (it.turned && !interleaved) {
    it.e0 = c * V;
    it.e1 = R / 2 + c * V;
  } else {
    it.e0 = 2 * c * V;
    it.e1 = it.e0 + V;
  }
  return it;
}

// x[0..V) and x[V..2V) hold the item's two vectors; cs its V (cos, sin).
template <int V>
__device__ __forceinline__ void rotary_turn(float (&x)[2 * V], const float2 (&cs)[V], bool interleaved) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (interleaved) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * cs[i].x - b * cs[i].y;
      x[2 * i + 1] = b * cs[i].x + a * cs[i].y;
    } else {
      const float a = x[i], b = x[V + i];
      x[i] = a * cs[i].x - b * cs[i].y;
      x[V + i] = b * cs[i].x + a * cs[i].y;
    }
  }
}

}  // namespace rbln
