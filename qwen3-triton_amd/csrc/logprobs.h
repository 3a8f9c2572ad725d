// Softmax statistics of parts of a row of logits (logprobs.hip, and the LM head's epilogue in gemm_tile.h).
#pragma once
#include "common.h"

namespace q3lp {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Logarithms of e^d as factors beside e^d itself: from here on down that is 0, and the product has to be (not 0 times infinity, nor
// times what an upstream gradient makes of a larger number).
constexpr float kDeep = -300.f;

// Statistics of a part of a row: its maximum m, rest = the sum of e^d over all but one element that is m, and u = the sum of
// e^d d, d counted from m in base 2.  m = -inf: nothing but -inf there (rest 0, or NaN where there is a NaN too).
struct Part {
  float m, rest, u;
};
Q3_DEV float part_total(const Part& a) { return a.m == -INFINITY ? a.rest : 1.f + a.rest; }
// c2 = log2(e) / temperature
Q3_DEV Part join(const Part& a, const Part& b, float c2) {
  const bool first = a.m >= b.m;
  const Part &hi = first ? a : b, &lo = first ? b : a;
  if (lo.m == -INFINITY) return Part{hi.m, hi.rest + lo.rest, hi.u};
  const float d = (lo.m - hi.m) * c2, w = __builtin_amdgcn_exp2f(d), t = 1.f + lo.rest;
  return Part{hi.m, fmaf(t, w, hi.rest), fmaf(w, fmaf(t, fmaxf(d, kDeep), lo.u), hi.u)};
}

// Statistics of N values of a thread.  One element that is the maximum is taken out on the way to it (each step keeps the larger
// and stores the smaller), in four chains.  d comes as fma(x, c2, -m c2): one rounding, and what the product m c2 lost to its own is
// the same factor of every term.  It is at most 1 in base 2 while |m c2| <= 2^24; beyond (finite masks, 1e-6 as the temperature) the
// factor itself could leave the numbers, and d comes from the difference.  Maxima and minima here hand NaN on.
template <int N> Q3_DEV Part part_of(const float (&v)[N], float c2) {
  static_assert(N % 4 == 0, "four chains");
  float x[N], top[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    top[k] = v[k];
#pragma unroll
    for (int i = k + 4; i < N; i += 4) {
      x[i] = __builtin_elementwise_minimum(top[k], v[i]);
      top[k] = __builtin_elementwise_maximum(top[k], v[i]);
    }
  }
  Part p{top[0], 0.f, 0.f};
#pragma unroll
  for (int k = 1; k < 4; ++k) {
    x[k] = __builtin_elementwise_minimum(p.m, top[k]);
    p.m = __builtin_elementwise_maximum(p.m, top[k]);
  }
  const bool nan = p.m != p.m;
  if (nan) p.m = -INFINITY;
  if (__any(fabsf(p.m * c2) > 0x1p24f && p.m != -INFINITY)) {
    const float ref = p.m == -INFINITY ? 0.f : p.m;
#pragma unroll
    for (int i = 1; i < N; ++i) {
      const float d = (x[i] - ref) * c2, e = __builtin_amdgcn_exp2f(d);
      p.rest += e;
      p.u = fmaf(e, fmaxf(d, kDeep), p.u);
    }
  } else {
    const float mc = p.m == -INFINITY ? 0.f : p.m * c2, lost = p.m == -INFINITY ? 0.f : fmaf(p.m, c2, -mc);
    float rest[2] = {0.f, 0.f}, u[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 1; i < N; ++i) {
      const float d = fmaf(x[i], c2, -mc), e = __builtin_amdgcn_exp2f(d);
      rest[i & 1] += e;
      u[i & 1] = fmaf(e, fmaxf(d, kDeep), u[i & 1]);
    }
    const float k = __builtin_amdgcn_exp2f(-lost), r = rest[0] + rest[1];
    p.rest = r * k;
    p.u = k * fmaf(-lost, r, u[0] + u[1]);
  }
  if (nan || p.m == INFINITY) p.rest = NAN;  // inf - inf
  return p;
}

// What the LM head keeps of a logit for its gradient: how far it lies below the maximum of its 128 columns, in base 2 at the
// temperature, as 16 bits of a range of 64 (one conversion for two, which clamps).  A probability formed from it is off by at most
// 0.034 % (half a step of 64 / 65535, times ln 2), a tenth of the rounding of a bf16 gradient and less than that of an fp16 one, at a
// third of the memory and traffic of fp32 logits beside their gradient; below 2^-64 of the group's largest it is 0, as that of a
// logit of -inf is.
// (The difference comes first: of m k, which is large at a small temperature, a rounding error would stay, 1 % of a probability for m
// = 40 at 1e-4.  The distance in fp16 would be off by up to 0.4 % at e^-8, as much as the bf16 gradient's rounding.)
constexpr float kGapRange = 64.f, kGapStep = kGapRange / 65535.f;
Q3_DEV uint32_t gap2(float z0, float z1, float m, float c2) {
  const float k = c2 * (1.f / kGapRange);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16((m - z0) * k, (m - z1) * k));
}

}  // namespace q3lp
