// 2^(scale2 d) in 64 bits for differences d <= 0 of logits: what verification and sampling take a token's weight from.
#pragma once

#include "nsx_common.h"

// 2^(j / 32) in LDS: 32 entries, one on each pair of the 64 banks.
struct Pow2 {
  double t[32];
  __device__ __forceinline__ void fill() {
    if (threadIdx.x < 32) t[threadIdx.x] = exp2((double)threadIdx.x / 32);
  }
};

// The exponent is n + j / 32 + r with |r| <= 1 / 64 by adding 1.5 * 2^47; 2^r - 1 = r (ln2 + ..) to the sixth power of r
// leaves out 2^-58: with the roundings 2^-51 of the weight (to the fourth power 2^-39), beside what the product with scale2
// loses, as any exp(x / T) does. d no lower than -1000 / scale2.
__device__ __forceinline__ double nsx_pow2(double d, double scale2, const Pow2& tab) {
  const double t = fma(d, scale2, 0x1.8p47);
  const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, t);
  const double r = fma(d, scale2, -(t - 0x1.8p47));
  double h = 0.00015403530393381609;  // ln2^6 / 720, ln2^5 / 120, ..
  h = fma(r, h, 0.0013333558146428443);
  h = fma(r, h, 0.0096181291076284772);
  h = fma(r, h, 0.055504108664821580);
  h = fma(r, h, 0.24022650695910071);
  h = fma(r, h, 0.69314718055994531);
  const double c = tab.t[k & 31], w = fma(r * h, c, c);
  const uint64_t bits = __builtin_bit_cast(uint64_t, w);
  const uint32_t high = (uint32_t)(bits >> 32) + ((k & ~31u) << 15);  // 2^n into the exponent
  return __builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)bits);
}
