// Rotary embedding of 64-element head rows, shared by every kernel that rotates queries and keys, so that a row's
// bits do not depend on which kernel rotated it.
#pragma once

#include "nsx_common.h"

#include <math.h>

constexpr int ATTN_D = 64;        // head_dim (GPT-OSS)
constexpr int ATTN_MAX_REP = 16;  // query heads per kv head (columns of the matrix-core step)
// A running maximum's start. Finite, not -infinity: keys that all score -infinity (overflowed scores) then get weight
// e^-infinity = 0 beside it, where the difference of two infinities would make the head NaN.
constexpr float ATTN_LOWEST = -3.4028235e38f;

// Rotary of element d of a 64-element head row at position p: x = the
// element, partner = element d ^ 32 (both with bias), rotate_half pairing
// (gpt_oss.py:42-58, ops.py:95-104). Explicit fmaf so that every kernel that
// applies it rounds the same way.
__device__ __forceinline__ float rope_elem(float x, float partner, int d, int p, const float* __restrict__ inv_freq,
                                           float amp) {
  const float ang = (float)p * inv_freq[d & (ATTN_D / 2 - 1)];  // fp32, as positions.float() * inv
  float s, c;
  sincosf(ang, &s, &c);
  c *= amp;
  s *= amp;
  const float ps = partner * s;
  return d < ATTN_D / 2 ? fmaf(x, c, -ps) : fmaf(x, c, ps);
}

// The same for the pair (element d < 32, element d + 32): one sine and cosine serve both.
__device__ __forceinline__ void rope_pair(float& x0, float& x1, int p, float inv_freq, float amp) {
  const float ang = (float)p * inv_freq;
  float s, c;
  sincosf(ang, &s, &c);
  c *= amp;
  s *= amp;
  const float y0 = fmaf(x0, c, -(x1 * s));
  x1 = fmaf(x1, c, x0 * s);
  x0 = y0;
}
