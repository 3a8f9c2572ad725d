// What the 8-bit kernels share: the quantisation rule of a group of values with one scale, and 16-bit / 8-bit
// conversions.
//
// A group of values a with the largest magnitude M is held as q = the integer nearest to 127 a / M (ties to even) and a
// scale proportional to M / 127.  The rule is exact, not "nearest up to the rounding of a division": which integer is
// nearest does not depend on how the quotient was formed, so codes can be compared for equality.
#pragma once
#include "common.h"

// 127 / M for the fast quotient, and whether the fast quotient can be used (M neither so small that 127 / M or its
// products leave the normal range nor 0).
struct QuantStep {
  float m, inv;
  bool plain;
};
Q3_DEV QuantStep quant_step(float m) {
  const bool plain = m >= 0x1p-90f && m <= 0x1p120f;
  return {m, plain ? 127.f / m : 0.f, plain};
}

// The integer nearest to 127 a / m, |a| <= m, as a float.  a (127 / m) is off by less than 127 * 2^-22 = 3e-5, so only
// quotients within 1e-4 of a half are decided exactly, in 64 bits, where 127 a and (k + 1/2) m have no rounding: a and m
// have at most 24 bits.
Q3_DEV float quant_code(float a, const QuantStep& s) {
  const float t = a * s.inv;
  float q = rintf(t);
  if (!s.plain || fabsf(t - q) > 0.4999f) {
    if (!(s.m > 0.f)) return 0.f;
    const double u = 127.0 * (double)a, m = (double)s.m;
    const double k = floor(s.plain ? (double)t : u / m);
    // k is the floor of the quotient up to one step at a whole number, where either neighbour below is decided alike
    const double mid = (k + 0.5) * m;
    const double lo = u < mid ? k : u > mid ? k + 1.0 : 2.0 * rint(0.5 * k + 0.25);  // tie: the even one
    q = (float)lo;
  }
  return q;
}

// The largest magnitude as bits: the order of the non-negative floats is that of their bits, and NaN lies above
// infinity, so a group that holds either cannot pass for a finite one.
Q3_DEV uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
Q3_DEV bool bits_finite(uint32_t b) { return b < 0x7f800000u; }

// Four codes (as floats in [-127, 127]) packed into one word, the first in the low byte.
Q3_DEV int pack_codes(float a, float b, float c, float d) {
  return (int)(((uint32_t)(int)a & 0xffu) | (((uint32_t)(int)b & 0xffu) << 8) | (((uint32_t)(int)c & 0xffu) << 16) |
               ((uint32_t)(int)d << 24));
}

template <int WIDTH> Q3_DEV uint32_t group_umax(uint32_t x) {
#pragma unroll
  for (int o = 1; o < WIDTH; o <<= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, o, 64);
    x = x > y ? x : y;
  }
  return x;
}
