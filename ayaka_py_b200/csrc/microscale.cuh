// Blocks of 32 numbers that share a power of two: rows as e4m3, weights as e2m1, scales as e8m0 (the biased exponent; 255: NaN).
#pragma once

#include "common.cuh"

constexpr int MX_BLOCK = 32;

// The scale's code for a block whose largest magnitude has these float bits: the smallest power of two with
// largest / 2^e <= 448 = 1.75 * 2^8, in whole numbers: a mantissa above 1.75 carries into the exponent.  Infinities and NaN (whose
// bits are the largest) give 255, zeros and what lies below 2^-119 the smallest scale, 2^-127.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t largest_bits) {
  if (largest_bits >= 0x7f800000u) return 255u;
  const int e = (int)((largest_bits + 0x1fffffu) >> 23) - 8;
  return e > 0 ? (uint32_t)e : 0u;
}
// 2^-e for a scale's code: the factor that takes numbers to their codes.  (254 - code: the factor's biased exponent; 127 of 2^-127
// is a plain number, and the largest code that mx_scale_code gives, 247, leaves 7.)
__device__ __forceinline__ float mx_inverse(uint32_t code) { return __uint_as_float(code == 255u ? 0x7fffffffu : (254u - code) << 23); }

// Two numbers to e4m3, rounded to the nearest (ties to even); the first in the low byte.  A NaN stays one.
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// The largest magnitude's bits are compared as whole numbers, so that a NaN is the largest of all.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
