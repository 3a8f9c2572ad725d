// What the 8-bit kernels share: the quantisation rule of a group of values with one scale, and 16-bit / 8-bit
// conversions.
//
// A group of values a with the largest magnitude M is held as q = the integer nearest to 127 a / M (ties to even) and a
// scale proportional to M / 127.  The rule is exact, not "nearest up to the rounding of a division": which integer is
// nearest does not depend on how the quotient was formed, so codes can be compared for equality.
#pragma once
#include <type_traits>

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

// The integer nearest to 127 a / m, |a| <= m, decided in 64 bits, where 127 a and (k + 1/2) m have no rounding (a and m have
// at most 24 bits).
Q3_DEV int quant_exact(float a, float m) {
  if (!(m > 0.f)) return 0;
  const double u = 127.0 * (double)a, top = (double)m, k = floor(u / top);
  // k is the floor up to one step at a whole number, where either neighbour below is decided alike
  const double mid = (k + 0.5) * top;
  return (int)(u < mid ? k : u > mid ? k + 1.0 : 2.0 * rint(0.5 * k + 0.25));  // tie: the even one
}

// Codes of 8 values, four to a word, the first in the low byte.  a (127 / m) + 1.5 * 2^23 in one fma leaves the nearest
// integer in the low bits, in two's complement; 127 / m and with it the quotient is off by at most 2^-24, 7.6e-6 of 127, so only
// those that lie within 1e-5 of a half are decided exactly, behind one branch for all 8.
Q3_DEV i32x2 quant_codes(const float (&a)[8], const QuantStep& s) {
  constexpr float kMagic = 12582912.f;
  constexpr float kNear = 0.49999f;
  float d[8], worst = 0.f;
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float r = fmaf(a[e], s.inv, kMagic);
    b[e] = __float_as_uint(r);
    d[e] = fabsf(fmaf(a[e], s.inv, kMagic - r));
    worst = fmaxf(worst, d[e]);
  }
  if (!s.plain || worst > kNear) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!s.plain || d[e] > kNear) b[e] = (uint32_t)quant_exact(a[e], s.m);
  }
  i32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x0c0c0400u);
    w[h] = (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return w;
}

// The largest magnitude as bits: the order of the non-negative floats is that of their bits, and NaN lies above
// infinity, so a group that holds either cannot pass for a finite one.
Q3_DEV uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
Q3_DEV bool bits_finite(uint32_t b) { return b < 0x7f800000u; }

// The same over packed 16-bit values, two to a word: the largest magnitude's 15 bits of either half, and as a float's bits.
Q3_DEV uint32_t mag_max16(uint32_t m, uint32_t x) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                __builtin_bit_cast(u16x2, x & 0x7fff7fffu)));
}
template <typename T> Q3_DEV uint32_t mag_bits16(uint32_t m) {
  const uint32_t lo = m & 0xffffu, hi = m >> 16;
  return __float_as_uint(to_f32<T>((u16)(lo > hi ? lo : hi)));
}

// Largest magnitude over a wave, every lane with the result.
Q3_DEV uint32_t wave_umax(uint32_t x) {
  auto dpp = [](uint32_t v, auto ctrl) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, decltype(ctrl)::value, 0xF, 0xF, true);
    return v > y ? v : y;
  };
  x = dpp(x, std::integral_constant<int, 0xB1>{});
  x = dpp(x, std::integral_constant<int, 0x4E>{});
  x = dpp(x, std::integral_constant<int, 0x141>{});
  x = dpp(x, std::integral_constant<int, 0x140>{});
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, o, 64);
    x = x > y ? x : y;
  }
  return x;
}
