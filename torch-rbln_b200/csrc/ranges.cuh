// Whole-number arithmetic that has to hold at the ends of its range. Plain
// C++, so that a host compiler takes it too.
#pragma once

#ifdef __CUDACC__
#define RBLN_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define RBLN_HOST_DEVICE inline
#endif

namespace rbln {

// How many positions a sequence sees whose new token is at pos: [0, pos], cut
// to the span, none below 0. A position past the span is any int up to the
// largest, for which pos + 1 would overflow.
RBLN_HOST_DEVICE int positions_seen(int pos, int span) { return pos < 0 ? 0 : pos >= span ? span : pos + 1; }

// Where CTA c's part begins of a line that is cut into shares, its end for
// CTAs behind the last one with a part: few long shares leave most CTAs there,
// at a product past 32 bits.
RBLN_HOST_DEVICE int share_start(int c, int share, int line) {
  const long long at = (long long)c * share;
  return at < line ? (int)at : line;
}

}  // namespace rbln
