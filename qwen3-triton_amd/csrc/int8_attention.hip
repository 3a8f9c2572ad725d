// Causal grouped-query attention over the key/value cache in 8 bits (int8_cache.hip): any number of new queries, which are
// the last S of the cache's positions.  Head dim 128.
//
// Per wave: 16 RT query rows (the G = Hq / Hkv heads of a position are rows of their own: row r is position r / G, head
// r % G) against one 64-position block after another.
//   S^T = K Q^T   v_mfma_f32_16x16x32, K codes as exact 16-bit numbers (|code| <= 127), the block's key scale on the fp32
//                 result; tile t of the block takes keys 16 (i / 4) + 4 t + i % 4 as its rows i, so that the four tiles
//                 leave lane (g, j) with the scores of row j for keys 16 g .. 16 g + 15 in order;
//   O^T += V^T P  v_mfma_f32_16x16x32_f16: V lies transposed in its block, so lane (g, i)'s operand, 16 keys of one dim, is
//                 16 contiguous bytes, and P is the lane's own scores: neither goes through LDS nor another lane.
// The value scale rides on P: P' = p * scale / unit in fp16, O in units of `unit`, a power of two that follows the blocks'
// scales only when one is more than 16 times off it.  P in fp16 has 11 bits where bf16 has 8, and unit keeps it in range.
// The running maximum and sum of the softmax are per row, replicated over the 4 lane groups.
// The unfinished block is read from the 16-bit tail in the same lane order (V tail transposed as well).
// Bound by HBM at one token over a long cache (8 rows x 20001 positions x 8 heads: 58.8 us, 5.6 TB/s), by latency over a short
// one (2048 positions: 5.8 us + 2.2 - 3.3 for the join); with many queries by the vector units (exponentials, conversions) beside
// the matrix cores: by counters 2490 and 2050 of the 4600 cycles that a CU takes for a 256-row block, LDS 1290 without bank
// conflicts (8192 queries of 32 heads: 537 - 575 us, as the 16-bit kernel's 501 - 576; 1024 queries at 3000: 79 - 86 us + 9.5).
#include <algorithm>

#include "int8_cache.h"

namespace {

using namespace q3kv8;

constexpr float kLow = -3.402823466e38f;  // below every score: exp2(-inf - kLow) is 0, exp2(kLow - kLow) multiplies 0

struct AttnArgs {
  const u16* q;
  int64_t qb, qs, qh;  // element strides of batch, position, head
  const int8_t *ck, *cv;
  const float *sk, *sv;
  const u16 *tk, *tv;
  u16* o;
  int64_t ob, os, oh;
  float *po, *pm, *pl;  // split partials: unnormalised O [rows][D], maximum, sum
  int64_t S, start, capacity;
  const int64_t* start_dev;
  int Hkv, G, splits, max_splits, minper;
  float scale2;  // softmax scale * log2(e)
};

// NaN as a value that the compiler does not know (this file is compiled on the promise that results of arithmetic are not NaN).
Q3_DEV float quiet_nan() {
  uint32_t x;
  asm("v_mov_b32 %0, 0x7fc00000" : "=v"(x));
  return __uint_as_float(x);
}

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
Q3_DEV int pack_f16x2(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(int, __builtin_convertvector(v, f16x2_t));
}

// P with 11 bits leaves bf16 outputs 0.6 % farther from 64 bits than a 32-bit P (their own rounding is 8 times as large); its
// remainder in a second product would cost few rows 2 - 4 % (2048 positions 7.7 -> 8.1 us, 8 x 20001 57.2 -> 58.2).  To fp16
// outputs 11 bits add as much error as their own rounding (1.4 - 1.6 times a 32-bit P's in all), so there the kernel of few
// rows, which waits for memory, takes the remainder p - fp16(p).  The kernel of many rows has no registers for it (85 spilled);
// its sums are of the rounded P, which leaves 1.25 - 1.4.
template <typename T> constexpr bool kTwoTerms = T::code == Q3_F16;
Q3_DEV int pack_rest_f16x2(float lo, float hi, int packed) {
  const f16x2_t h = __builtin_bit_cast(f16x2_t, packed);
  return pack_f16x2(lo - (float)h[0], hi - (float)h[1]);
}
// The same in the activation type, for the tail's P.
template <typename T> Q3_DEV int pack_rest2(float lo, float hi, int packed) {
  return (int)pack2<T>(lo - to_f32<T>((u16)((uint32_t)packed & 0xffffu)), hi - to_f32<T>((u16)((uint32_t)packed >> 16)));
}

// Both halves onto a sum in fp32 (subnormal halves count: 40000 weights of e^-11 beside one of 1 are summed right).
Q3_DEV float sum_f16x2(int x, float sum) {
  const f16x2_t one = {(_Float16)1.f, (_Float16)1.f};
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, x), one, sum, false);
}

// 8 codes -> 8 exact 16-bit numbers.  fp16: the code + 128 as the low bits of 1024 + x, less 1152.
template <typename T> Q3_DEV bf16x8_t codes16(int lo, int hi) {
  i32x4 r;
  if constexpr (T::code == Q3_F16) {
    const f16x2_t bias = {(_Float16)1152.f, (_Float16)1152.f};
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t w = (uint32_t)(p < 2 ? lo : hi) ^ 0x80808080u;
      const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w, (p & 1) ? 0x04030402u : 0x04010400u);
      r[p] = __builtin_bit_cast(int, __builtin_bit_cast(f16x2_t, u) - bias);
    }
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t w = (uint32_t)(p < 2 ? lo : hi);
      const int s = 16 * (p & 1);
      r[p] = (int)pack_bf16x2((float)(int8_t)(w >> s), (float)(int8_t)(w >> (s + 8)));
    }
  }
  return __builtin_bit_cast(bf16x8_t, r);
}

// One block's operands in flight: K codes of 4 tiles x 2 halves of D, V codes of 8 dim tiles.
struct Raw {
  i32x4 k[4][2], v[8];
};

template <typename T, int RT> struct Rows {
  bf16x8_t q[RT][2][2];  // [row tile][64-dim half c][8-dim half h]: dims 64 c + 16 g + 8 h .. + 7
  f32x4 o[RT][8];        // O^T: dims 16 t + 4 g + e
  float m[RT], l[RT];
  float unit, inv;       // of O: a power of two (0: nothing yet), and 1 / unit
  float least;           // 2^-76 of the largest unit so far
};

Q3_DEV float xmax4(float x) {  // max over lanes {l, l ^ 16, l ^ 32, l ^ 48}
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}

// Raw scores of a block (S^T) -> p in s: 2^(c s - m) * factor, with the running maximum and sum, and O rescaled, also by
// `units`, in one place (every branch that touches O costs its registers twice).  The maximum moves only when a score
// passes it by more than 8 (p <= 2^8 is as exact in every type that P takes), so O is rarely rescaled.
// mask: positions key0 + 4 t + e past a row's own are hidden.
template <typename T, int RT>
Q3_DEV void softmax_step(Rows<T, RT>& w, f32x4 (&s)[RT][4], float c, float log2_factor, float inv_factor, float units,
                         bool mask, int key0, const int (&qpos)[RT]) {
  if (mask) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][t][e] = key0 + 4 * t + e > qpos[r] ? -INFINITY : s[r][t][e];
  }
  float mx[RT];
  bool up = units != 1.f;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float x = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) x = fmaxf(x, s[r][t][e]);
    mx[r] = xmax4(x) * c;
    up = up || mx[r] > w.m[r] + 8.f;
  }
  if (__any(up)) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float m = fmaxf(w.m[r], mx[r]), alpha = __builtin_amdgcn_exp2f(w.m[r] - m), f = alpha * units;
      w.m[r] = m;
      w.l[r] *= alpha;
#pragma unroll
      for (int t = 0; t < 8; ++t) w.o[r][t] *= f;
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float off = log2_factor - w.m[r];
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[r][t][e] = __builtin_amdgcn_exp2f(fmaf(s[r][t][e], c, off));
        sum += s[r][t][e];
      }
    w.l[r] = fmaf(sum, inv_factor, w.l[r]);
  }
}

// A value that is the same in every lane, in a scalar register.
Q3_DEV float uniform(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); }

// A block's factor of the raw scores.  A factor of 0 would turn hidden positions' minus infinity into NaN.  Keys that are all zero
// have scale 0, and their raw scores are 0 whatever the factor; a product that fell below 2^-149 makes scores of 0 too (raw scores
// stay below 2^30 for queries below 2^16).
Q3_DEV float score_factor(float kscale, float scale2) {
  const float c = uniform(kscale * scale2);
  return __float_as_uint(c) == 0 ? 0x1p-126f : c;
}

// How a block's value scale meets O's unit: O is to be multiplied by `units`, and P' = p * scale / unit.
struct UnitStep {
  float units, ratio, log2_factor, inv_factor;
  bool rides, nan;  // the factor rides in the exponent; if not, it is 0, far below the unit, or NaN
};
template <typename T, int RT> Q3_DEV UnitStep unit_step(Rows<T, RT>& w, float vscale) {
  // A value scale within 16 times of the unit leaves it; one 2^76 below the largest unit so far adds nothing worth a new one.
  // (Below the largest, not the last: O grows by old unit / new unit with each fall, and passes 2^128 after a few.  |O| is at
  // most 128 * 16 * 2^8 a position in its unit, 2^50 at 2^31 positions, so a fall by 2^76 in all leaves it finite.)
  const uint32_t vb = __float_as_uint(uniform(vscale));  // >= 0, or NaN
  UnitStep u;
  u.units = 1.f;
  u.ratio = uniform(vscale * w.inv);
  const uint32_t kMost = 0x41800000u, kLeast = 0x3d800000u;  // 16, 1 / 16
  uint32_t rb = __float_as_uint(u.ratio);
  if (vb < 0x7f800000u && vb > 0 && (w.inv == 0.f || rb > kMost || (rb < kLeast && vb > __float_as_uint(w.least)))) {
    const uint32_t e = min(max(vb & 0x7f800000u, 0x00800000u), 0x7e000000u);  // the power of two below, 2^-126 .. 2^125
    const float inv = __uint_as_float(0x7f000000u - e);
    u.units = uniform(w.unit * inv);
    w.unit = __uint_as_float(e);
    w.inv = inv;
    w.least = uniform(fmaxf(w.least, w.unit * 0x1p-76f));
    u.ratio = uniform(vscale * inv);
    rb = __float_as_uint(u.ratio);
  }
  u.rides = rb >= kLeast && rb <= kMost;
  u.nan = vb > 0x7f800000u;
  u.log2_factor = u.rides ? uniform(__builtin_amdgcn_logf(u.ratio)) : 0.f;  // base 2
  u.inv_factor = u.rides ? uniform(__builtin_amdgcn_exp2f(-u.log2_factor)) : 1.f;
  return u;
}

// A block in 8 bits: P' = p * scale / unit as fp16 operands.
template <typename T, int RT>
Q3_DEV void softmax_codes(Rows<T, RT>& w, f32x4 (&s)[RT][4], float c, float vscale, bool mask, int key0,
                          const int (&qpos)[RT], i32x4 (&p)[RT][2], i32x4 (&rest)[RT][2]) {
  const UnitStep u = unit_step(w, vscale);
  softmax_step<T, RT>(w, s, c, u.log2_factor, u.inv_factor, u.units, mask, key0, qpos);
  if (!u.rides) {  // zero, far below the unit, or NaN, for every row: 16 rows' positions lie closer than a block's
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][t][e] = s[r][t][e] * u.ratio;
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int x = pack_f16x2(s[r][t][2 * e], s[r][t][2 * e + 1]);
        p[r][t >> 1][2 * (t & 1) + e] = x;
        if constexpr (kTwoTerms<T>) rest[r][t >> 1][2 * (t & 1) + e] = pack_rest_f16x2(s[r][t][2 * e], s[r][t][2 * e + 1], x);
      }
}

// What a wave of either kernel knows of its launch (positions and blocks fit 32 bits: capacity does).
struct Span {
  int start, total, whole, b0, b_end;  // positions before the queries and in all; blocks in 8 bits; this split's blocks
  int rows, row0, bh;
  const int8_t *ck, *cv;
  const float *sk, *sv;
};

// Blocks a split takes: at least minper, all of them over at most max_splits.  It follows from the positions alone, not from
// the span that a launch covers, so a captured step and an eager call of one length form the same sums.
template <int RT> Q3_DEV Span span_of(const AttnArgs& a, int b, int hk, int split, int row0) {
  Span p;
  const int cap = (int)a.capacity;
  p.start = (int)min(max(a.start_dev ? *a.start_dev : a.start, (int64_t)-1), a.capacity);
  p.total = min(p.start + (int)a.S, cap);
  p.whole = p.total / BLK;
  p.rows = (int)a.S * a.G;
  p.row0 = row0;
  p.bh = b * a.Hkv + hk;
  const int64_t cblocks = (cap + BLK - 1) / BLK;
  const int all = (p.total + BLK - 1) / BLK, per = max((all + a.max_splits - 1) / a.max_splits, a.minper);
  p.b0 = split * per;
  p.b_end = min(p.b0 + per, all);
  p.ck = a.ck + p.bh * cblocks * (BLK * D);
  p.cv = a.cv + p.bh * cblocks * (BLK * D);
  p.sk = a.sk + p.bh * cblocks;
  p.sv = a.sv + p.bh * cblocks;
  return p;
}

// The wave's query rows in registers, nothing summed yet.
template <typename T, int RT>
Q3_DEV void load_rows(const AttnArgs& a, const Span& p, int b, int hk, int g, int j, Rows<T, RT>& w, int (&qpos)[RT]) {
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int rc = min(p.row0 + 16 * r + j, p.rows - 1), s = rc / a.G, h = hk * a.G + (rc - s * a.G);
    qpos[r] = s;  // relative to start: the last visible position is start + qpos
    const u16* qp = a.q + b * a.qb + s * a.qs + h * a.qh + 16 * g;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) w.q[r][c][e] = *reinterpret_cast<const bf16x8_t*>(qp + 64 * c + 8 * e);
    w.m[r] = kLow;
    w.l[r] = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) w.o[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  w.unit = w.inv = w.least = 0.f;
}

// The tail block, in 16 bits: P in T, as V is, in two terms: its rounding and the remainder's (over the first 63 positions of
// a request the tail is all there is, and one bf16 term there left outputs 1.2 - 1.3 times as far from 64 bits as a 32-bit P's;
// it is one block in a row's pass).  Slots past the last position hold anything and read as zeros.  One row tile
// takes all of V before its scores are formed (a wait less); two have no registers for that and take two dim tiles at a time.
// An infinity or NaN among the values makes the rows that see its position NaN, as the whole block will be; the others, whose
// P is 0 there, are kept clear of it (0 times it is NaN) by reading zeros from that slot on.
template <typename T, int RT>
Q3_DEV void tail_block(const AttnArgs& a, const Span& p, int g, int j, Rows<T, RT>& w, const int (&qpos)[RT]) {
  const int left = p.total - p.whole * BLK, krow = 16 * (j >> 2) + (j & 3);
  f32x4 s[RT][4];
  constexpr int VT = RT == 1 ? 8 : 2;  // dim tiles of V in registers
  i32x4 v[VT][2];
  auto load_v = [&](int t, i32x4 (&x)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) x[h] = *reinterpret_cast<const i32x4*>(a.tv + (int64_t)p.bh * (BLK * D) + (16 * t + j) * BLK + 16 * g + 8 * h);
  };
  bf16x8_t tkf[RT == 1 ? 4 : 1][2][2];
  auto load_k = [&](int t, bf16x8_t (&x)[2][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        x[h][e] = *reinterpret_cast<const bf16x8_t*>(a.tk + (int64_t)p.bh * (BLK * D) + (krow + 4 * t) * D + 64 * h + 16 * g + 8 * e);
  };
  if constexpr (RT == 1) {
#pragma unroll
    for (int t = 0; t < 4; ++t) load_k(t, tkf[t]);
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (RT > 1) load_k(t, tkf[0]);
#pragma unroll
    for (int r = 0; r < RT; ++r) s[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bf16x8_t kf = tkf[RT == 1 ? t : 0][h][e];
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][t] = mfma_16x16x32<T>(kf, w.q[r][h][e], s[r][t]);
      }
    if constexpr (RT > 1) __builtin_amdgcn_sched_barrier(0);  // a tile's operands at a time: registers
  }
  if constexpr (VT == 8) {
#pragma unroll
    for (int t = 0; t < 8; ++t) load_v(t, v[t]);
  }
  // O back to plain units: the tail's values are what they are
  softmax_step<T, RT>(w, s, a.scale2, 0.f, 1.f, w.unit, true, p.whole * BLK - p.start + 16 * g, qpos);
  w.unit = w.inv = 1.f;
  bf16x8_t pf[RT][2], prest[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = s[r][2 * h + (e >> 1)][2 * (e & 1)], hi = s[r][2 * h + (e >> 1)][2 * (e & 1) + 1];
        x[e] = (int)pack2<T>(lo, hi);
        y[e] = pack_rest2<T>(lo, hi, x[e]);
      }
      pf[r][h] = __builtin_bit_cast(bf16x8_t, x);
      prest[r][h] = __builtin_bit_cast(bf16x8_t, y);
    }
#pragma unroll
  for (int t0 = 0; t0 < 8; t0 += VT) {
    if constexpr (VT < 8) {
#pragma unroll
      for (int t = 0; t < VT; ++t) load_v(t0 + t, v[t]);
    }
    uint32_t most = 0;
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = mag_max16(most, (uint32_t)v[t][h][e]);
    int lim = left;
    if (__any(!bits_finite(mag_bits16<T>(most)))) {
      uint32_t before = 0;  // 64 - the first slot that is not finite
#pragma unroll
      for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (!bits_finite(mag_bits(to_f32<T>((u16)((uint32_t)v[t][h][e >> 1] >> (16 * (e & 1)))))))
              before = max(before, (uint32_t)(64 - (16 * g + 8 * h + e)));
      const int first = 64 - (int)wave_umax(before);
      if (first < left) {
        lim = first;
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if (p.whole * BLK - p.start + first <= qpos[r]) w.l[r] = quiet_nan();
      }
    }
    uint32_t keep[2][4];  // the slots below lim, two to a word (masks, not branches: 9.5 against 11.7 us at 2047 positions)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) keep[h][e] = (uint32_t)~(~0ull << 16 * min(max(lim - (16 * g + 8 * h + 2 * e), 0), 2));
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        i32x4 x = v[t][h];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] &= (int)keep[h][e];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          w.o[r][t0 + t] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, x), pf[r][h], w.o[r][t0 + t]);
          w.o[r][t0 + t] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, x), prest[r][h], w.o[r][t0 + t]);
        }
      }
    if constexpr (VT < 8) __builtin_amdgcn_sched_barrier(0);
  }
}

// Row sums over the lane groups, O in plain units.
template <typename T, int RT> Q3_DEV void close_rows(Rows<T, RT>& w) {
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    w.l[r] += __shfl_xor(w.l[r], 16, 64);
    w.l[r] += __shfl_xor(w.l[r], 32, 64);
#pragma unroll
    for (int t = 0; t < 8; ++t) w.o[r][t] *= w.unit;
  }
}

// O / l to the output, or this split's (O, m, l).  A split without a visible position leaves l = 0 and no O.
template <typename T, int RT>
Q3_DEV void store_rows(const AttnArgs& a, const Span& p, int b, int hk, int split, int g, int j, const Rows<T, RT>& w) {
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = p.row0 + 16 * r + j;
    if (row >= p.rows) continue;
    if (a.splits == 1) {
      const int64_t s = row / a.G, h = hk * a.G + (row - s * a.G);
      u16* op = a.o + b * a.ob + s * a.os + h * a.oh + 4 * g;
      const float inv = 1.f / w.l[r];
#pragma unroll
      for (int t = 0; t < 8; ++t)
        *reinterpret_cast<i32x2*>(op + 16 * t) = i32x2{(int)pack2<T>(w.o[r][t][0] * inv, w.o[r][t][1] * inv),
                                                       (int)pack2<T>(w.o[r][t][2] * inv, w.o[r][t][3] * inv)};
    } else {
      const int64_t pr = ((int64_t)p.bh * p.rows + row) * a.splits + split;
      if (g == 0) {
        a.pm[pr] = w.m[r];
        a.pl[pr] = w.l[r];
      }
      if (w.l[r] == 0.f) continue;
#pragma unroll
      for (int t = 0; t < 8; ++t) *reinterpret_cast<f32x4*>(a.po + pr * D + 16 * t + 4 * g) = w.o[r][t];
    }
  }
}

// Few rows (at most 16 per key/value head: one token of a group, a few of a small one): four waves share the rows and take
// every fourth block each, their K and V fragments straight from memory, and join through LDS.  Heads before splits in the
// grid: a head's splits on one XCD, where the join finds them (2048 positions 8.5 us with the join, splits first 10.5; at
// 8 x 20001 positions splits first is 5 % faster).
template <typename T> __global__ __launch_bounds__(256) void kv8_attn_rows_kernel(AttnArgs a) {
  constexpr int RT = 1, WK = 4;
  const int lane = threadIdx.x & 63, wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int b = blockIdx.x / a.Hkv, hk = blockIdx.x % a.Hkv, split = blockIdx.z;
  const Span sp = span_of<RT>(a, b, hk, split, 0);
  Rows<T, RT> w;
  int qpos[RT];
  load_rows<T, RT>(a, sp, b, hk, g, j, w, qpos);
  const int wend = min(sp.b_end, sp.whole);
  int blk = sp.b0 + wk;

  Raw raw;
  float sk = 0.f, sv = 0.f;
  const int krow = 16 * (j >> 2) + (j & 3);
  auto load_k = [&](int i) {
    const int8_t* p = sp.ck + (int64_t)i * (BLK * D) + krow * D + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) raw.k[t][c] = *reinterpret_cast<const i32x4*>(p + t * 4 * D + 64 * c);
    sk = sp.sk[i];
    sv = sp.sv[i];
  };
  auto load_v = [&](int i) {
    const int8_t* p = sp.cv + (int64_t)i * (BLK * D) + j * BLK + 16 * g;
#pragma unroll
    for (int t = 0; t < 8; ++t) raw.v[t] = *reinterpret_cast<const i32x4*>(p + t * 16 * BLK);
  };
  if (blk < wend) {
    load_k(blk);
    load_v(blk);
  }
  for (; blk < wend; blk += WK) {
    f32x4 s[RT][4];
    const float c = score_factor(sk, a.scale2);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          s[0][t] = mfma_16x16x32<T>(codes16<T>(raw.k[t][h][2 * e], raw.k[t][h][2 * e + 1]), w.q[0][h][e], s[0][t]);
    }
    const float vs = sv;
    if (blk + WK < wend) load_k(blk + WK);
    i32x4 p[RT][2], rest[RT][2];
    softmax_codes<T, RT>(w, s, c, vs, (blk + 1) * BLK > sp.start + 1, blk * BLK - sp.start + 16 * g, qpos, p, rest);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bf16x8_t v = codes16<F16>(raw.v[t][2 * e], raw.v[t][2 * e + 1]);
        w.o[0][t] = mfma_16x16x32<F16>(v, __builtin_bit_cast(bf16x8_t, p[0][e]), w.o[0][t]);
        if constexpr (kTwoTerms<T>) w.o[0][t] = mfma_16x16x32<F16>(v, __builtin_bit_cast(bf16x8_t, rest[0][e]), w.o[0][t]);
      }
    }
    if (blk + WK < wend) load_v(blk + WK);
  }
  if (blk == sp.whole && blk < sp.b_end) tail_block<T, RT>(a, sp, g, j, w, qpos);
  close_rows<T, RT>(w);
  // the waves joined in halves, in a fixed order
  __shared__ f32x4 jo[WK / 2][8][64];
  __shared__ float jm[WK / 2][64], jl[WK / 2][64];
#pragma unroll
  for (int half = WK / 2; half >= 1; half >>= 1) {
    if (wk >= half && wk < 2 * half) {
      jm[wk - half][lane] = w.m[0];
      jl[wk - half][lane] = w.l[0];
#pragma unroll
      for (int t = 0; t < 8; ++t) jo[wk - half][t][lane] = w.o[0][t];
    }
    __syncthreads();
    if (wk < half) {
      const float m2 = jm[wk][lane], m = fmaxf(w.m[0], m2);
      const float f1 = __builtin_amdgcn_exp2f(w.m[0] - m), f2 = __builtin_amdgcn_exp2f(m2 - m);
      w.l[0] = w.l[0] * f1 + jl[wk][lane] * f2;
      w.m[0] = m;
#pragma unroll
      for (int t = 0; t < 8; ++t) w.o[0][t] = w.o[0][t] * f1 + jo[wk][t][lane] * f2;
    }
    __syncthreads();
  }
  if (wk == 0) store_rows<T, RT>(a, sp, b, hk, split, g, j, w);
}

// Barrier that leaves global loads in flight: this wave's LDS accesses are done, then s_barrier.
Q3_DEV void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Many rows: eight waves of 32 rows each share every block.  Its codes become 16-bit fragments once per workgroup, in LDS in
// the order in which the lanes read them (a wave-wide kilobyte per fragment: no bank conflicts).
// Pipeline: while the exponentials of block n run on the vector units, the matrix cores form P V of block n - 1 and the scores
// of block n + 1, in eight steps of eight products each, and the codes of K(n + 2) and V(n) become fragments; K and V keep two
// stages each.  One barrier per block.  O follows a change of the maximum or of its unit a block late (`pend`), between P V of
// the block before the change and of the block after it.
template <typename T> __global__ __launch_bounds__(512, 2) void kv8_attn_tile_kernel(AttnArgs a) {
  constexpr int RT = 2, WR = 8;
  __shared__ __attribute__((aligned(16))) i32x4 lk[2][4][4][64], lv[2][8][2][64];  // [stage][tile][16-byte step][lane]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int b = blockIdx.x / a.Hkv, hk = blockIdx.x % a.Hkv, split = blockIdx.z;
  const int rb = gridDim.y - 1 - blockIdx.y;  // the rows that see most first
  const int wg0 = rb * (16 * RT * WR);
  const Span sp = span_of<RT>(a, b, hk, split, wg0 + wave * 16 * RT);
  Rows<T, RT> w;
  int qpos[RT];
  load_rows<T, RT>(a, sp, b, hk, g, j, w, qpos);
  auto seen = [&](int row0, int n) { return sp.start + (min(row0 + n, sp.rows) - 1) / a.G; };  // last position of n rows
  // blocks of 8 bits: n = 0 .. nb - 1 are the split's, as far as the workgroup's rows see
  const int nb = min(min(sp.b_end, sp.whole), seen(wg0, 16 * RT * WR) / BLK + 1) - sp.b0;
  const int first_pos = sp.start + min(sp.row0, sp.rows - 1) / a.G;
  const int clear = min((first_pos + 1) / BLK - sp.b0, nb);  // blocks before this one need no mask

  if (nb > 0) {
    // codes in flight: this wave's 16-byte pieces, K tile wave / 2, half wave % 2, and V dim tile `wave` (past the end: the
    // last block again)
    i32x4 rk, rv;
    const uint32_t klane = ((wave >> 1) * 4 + 16 * (j >> 2) + (j & 3)) * D + 64 * (wave & 1) + 16 * g;
    const uint32_t vlane = (16 * wave + j) * BLK + 16 * g;
    auto codes_of = [&](const int8_t* base, int n) { return base + (int64_t)(sp.b0 + min(n, nb - 1)) * (BLK * D); };
    auto fetch_k = [&](int n) { rk = *reinterpret_cast<const i32x4*>(codes_of(sp.ck, n) + klane); };
    auto fetch_v = [&](int n) { rv = *reinterpret_cast<const i32x4*>(codes_of(sp.cv, n) + vlane); };
    auto spread_k = [&](int st) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        lk[st][wave >> 1][2 * (wave & 1) + e][lane] = __builtin_bit_cast(i32x4, codes16<T>(rk[2 * e], rk[2 * e + 1]));
    };
    auto spread_v = [&](int st) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        lv[st][wave][e][lane] = __builtin_bit_cast(i32x4, codes16<F16>(rv[2 * e], rv[2 * e + 1]));
    };
    // the operands of step i: two of V (dim tile i) and two of K (half a tile of keys)
    auto read_v = [&](bf16x8_t (&f)[2], int st, int i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) f[e] = __builtin_bit_cast(bf16x8_t, lv[st][i][e][lane]);
    };
    auto read_k = [&](bf16x8_t (&f)[2], int st, int i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) f[e] = __builtin_bit_cast(bf16x8_t, lk[st][i >> 1][2 * (i & 1) + e][lane]);
    };
    auto pv_step = [&](const bf16x8_t (&f)[2], const i32x4 (&p)[RT][2], int i) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int r = 0; r < RT; ++r) w.o[r][i] = mfma_16x16x32<F16>(f[e], __builtin_bit_cast(bf16x8_t, p[r][e]), w.o[r][i]);
    };
    auto qk_step = [&](const bf16x8_t (&f)[2], f32x4 (&s)[RT][4], int i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = i >> 1, e = 2 * (i & 1) + h;
#pragma unroll
        for (int r = 0; r < RT; ++r)
          s[r][t] = mfma_16x16x32<T>(f[h], w.q[r][e >> 1][e & 1], e == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[r][t]);
      }
    };
    float pend[RT] = {1.f, 1.f};
    bool late = false;
    auto rescale = [&]() {
      if (!late) return;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < 8; ++t) w.o[r][t] *= pend[r];
    };
    float nsk = sp.sk[sp.b0], nsv = sp.sv[sp.b0];
    // block n: s its scores, p becomes its P', sn the scores of block n + 1, pp the P' of block n - 1
    auto block = [&](int n, f32x4 (&s)[RT][4], i32x4 (&p)[RT][2], f32x4 (&sn)[RT][4], const i32x4 (&pp)[RT][2], auto par) {
      constexpr int W = decltype(par)::value, R = W ^ 1;  // stages written and read
      lds_barrier();
      bf16x8_t fv[2][2], fk[2];
      read_v(fv[0], R, 0);
      rescale();
      float c = score_factor(nsk, a.scale2);
      const UnitStep u = unit_step(w, nsv);
      if (n >= clear) {
        const int key0 = (sp.b0 + n) * BLK - sp.start + 16 * g;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[r][t][e] = key0 + 4 * t + e > qpos[r] ? -INFINITY : s[r][t][e];
      }
      if (__float_as_uint(c) > 0x7f800000u) {  // keys that were not finite: NaN for the rows that see the block, no others
        const float nan = c;
        c = 1.f;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (__float_as_uint(s[r][t][e]) != 0xff800000u) s[r][t][e] = nan;
      }
      float mx[RT];
      bool up = u.units != 1.f;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float x = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) x = fmaxf(x, s[r][t][e]);
        mx[r] = xmax4(x) * c;
        up = up || mx[r] > w.m[r] + 8.f;
      }
      late = __any(up);
      if (late) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float m = fmaxf(w.m[r], mx[r]), alpha = __builtin_amdgcn_exp2f(w.m[r] - m);
          w.m[r] = m;
          w.l[r] *= alpha;
          pend[r] = alpha * u.units;
        }
      }
      if (!u.rides) {  // no values worth a product (or NaN): their part of the sums here, then scores that give P' 0 (or NaN)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = fmaf(s[r][t][e], c, -w.m[r]);
              asm volatile("" : "+v"(x));  // not the expression of the steps below, or both are formed up here
              w.l[r] += __builtin_amdgcn_exp2f(x);
              // hidden positions (minus infinity, by its bits) stay hidden
              if (__float_as_uint(s[r][t][e]) != 0xff800000u) s[r][t][e] = u.nan ? u.ratio : -INFINITY;
            }
      }
      float off[RT], sum[RT] = {0.f, 0.f};
#pragma unroll
      for (int r = 0; r < RT; ++r) off[r] = u.log2_factor - w.m[r];
      nsk = sp.sk[sp.b0 + min(n + 1, nb - 1)];
      nsv = sp.sv[sp.b0 + min(n + 1, nb - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        read_k(fk, R, i);  // V's are here a step early: their products cover the wait for K's
        if (i < 7) read_v(fv[(i + 1) & 1], R, i + 1);
        if (i == 0) spread_k(W);
        if (i == 0) fetch_k(n + 3);
        if (i == 3) spread_v(W);
        if (i == 3) fetch_v(n + 1);
        pv_step(fv[i & 1], pp, i);
        qk_step(fk, sn, i);
        const int r = i >> 2, t = i & 3;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][t][e] = __builtin_amdgcn_exp2f(fmaf(s[r][t][e], c, off[r]));
        int lo = pack_f16x2(s[r][t][0], s[r][t][1]), hi = pack_f16x2(s[r][t][2], s[r][t][3]);
        asm volatile("" : "+v"(lo), "+v"(hi));  // formed here, beside the products, not where the next block uses them
        sum[r] = sum_f16x2(hi, sum_f16x2(lo, sum[r]));
        p[r][t >> 1][2 * (t & 1)] = lo;
        p[r][t >> 1][2 * (t & 1) + 1] = hi;
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < RT; ++r) w.l[r] = fmaf(sum[r], u.inv_factor, w.l[r]);
    };

    f32x4 sa[RT][4], sb[RT][4];
    i32x4 pa[RT][2], pb[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) pb[r][e] = i32x4{0, 0, 0, 0};
    fetch_k(0);
    spread_k(0);
    fetch_k(1);
    spread_k(1);
#pragma unroll
    for (int e = 0; e < 2; ++e) lv[1][wave][e][lane] = i32x4{0, 0, 0, 0};  // P V "of block -1"
    fetch_k(2);
    fetch_v(0);
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bf16x8_t f[2];
      read_k(f, 0, i);
      qk_step(f, sa, i);
    }
    int n = 0;
    for (; n + 2 <= nb; n += 2) {
      block(n, sa, pa, sb, pb, std::integral_constant<int, 0>{});
      block(n + 1, sb, pb, sa, pa, std::integral_constant<int, 1>{});
    }
    if (n < nb) {
      block(n, sa, pa, sb, pb, std::integral_constant<int, 0>{});
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) pb[r][e] = pa[r][e];
    }
    lds_barrier();  // V of the last block
    rescale();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bf16x8_t f[2];
      read_v(f, (nb - 1) & 1, i);
      pv_step(f, pb, i);
    }
  }
  const int my_end = sp.row0 < sp.rows ? seen(sp.row0, 16 * RT) / BLK + 1 : 0;  // blocks this wave's rows see
  if (sp.b0 <= sp.whole && sp.whole < sp.b_end && sp.whole < my_end) tail_block<T, RT>(a, sp, g, j, w, qpos);
  close_rows<T, RT>(w);
  store_rows<T, RT>(a, sp, b, hk, split, g, j, w);
}

// out = sum_j 2^(m_j - M) o_j / sum_j 2^(m_j - M) l_j over a row's splits, in fixed order: 32 lanes per row, 4 dims each; a
// split's weight sits in lane j % 32.  Bound by the partials' traffic at many rows, by latency at few: NJ splits' outputs are
// in flight before their weights are known.
template <typename T, int NJ> __global__ __launch_bounds__(256) void kv8_merge_kernel(AttnArgs a) {
  const int64_t rows = a.S * a.G, i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), bh = blockIdx.y;
  const int lane = threadIdx.x & 31;
  const int64_t p0 = (bh * rows + min(i, rows - 1)) * a.splits;
  float mx = kLow;
  for (int k = lane; k < a.splits; k += 32) mx = fmaxf(mx, a.pm[p0 + k]);
  mx = group_max<32>(mx);
  float l = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < a.splits; k0 += 32) {
    const int n = min(32, a.splits - k0);
    float wgt = 0.f;
    if (lane < n) {
      const float pl = a.pl[p0 + k0 + lane];
      wgt = pl == 0.f ? 0.f : __builtin_amdgcn_exp2f(a.pm[p0 + k0 + lane] - mx);  // l = 0: nothing stored
      l += wgt * pl;
    }
    for (int k1 = 0; k1 < n; k1 += NJ) {
      f32x4 o[NJ];
#pragma unroll
      for (int k = 0; k < NJ; ++k) o[k] = *reinterpret_cast<const f32x4*>(a.po + (p0 + k0 + min(k1 + k, n - 1)) * D + 4 * lane);
#pragma unroll
      for (int k = 0; k < NJ; ++k) {
        const float f = k1 + k < n ? __shfl(wgt, min(k1 + k, n - 1), 32) : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += f == 0.f ? 0.f : f * o[k][e];
      }
    }
  }
  l = group_sum<32>(l);
  if (i >= rows) return;
  const float inv = 1.f / l;
  const int64_t s = i / a.G, h = (bh % a.Hkv) * a.G + (i - s * a.G);
  *reinterpret_cast<i32x2*>(a.o + (bh / a.Hkv) * a.ob + s * a.os + h * a.oh + 4 * lane) =
      i32x2{(int)pack2<T>(x[0] * inv, x[1] * inv), (int)pack2<T>(x[2] * inv, x[3] * inv)};
}

struct Plan {
  bool tile;
  int max_splits, minper, splits;
  int64_t row_blocks;
};

// Rows of one key/value head -> kernel and splits; the positions that a launch may span only bound the grid.
Plan plan_for(int64_t B, int64_t Hkv, int64_t rows, int64_t span) {
  Plan p;
  p.tile = rows > 16;
  p.row_blocks = p.tile ? (rows + 255) / 256 : 1;
  // Eight waves on every CU.  A split takes at least four blocks: one for each wave of the rows kernel, and enough for the tile
  // kernel's start (17 queries at 2000: 41.8 us at sixteen, 28.1 at eight, 21.6 at four, 19.6 at two; but 200 at 0 16.4, 16.4,
  // 16.3 and 19.6).  Where the rows fill the CUs without splits, sixteen, to pay for the join (32 x 300 positions: 13.1 us in two
  // splits, 10.7 in one).
  const int64_t wgs = B * Hkv * p.row_blocks;
  p.max_splits = (int)std::min<int64_t>(1024, std::max<int64_t>(1, (p.tile ? 256 : 512) / wgs));
  p.minper = wgs >= 256 ? 16 : 4;
  const int64_t blocks = (span + BLK - 1) / BLK;
  p.splits = (int)std::min<int64_t>(p.max_splits, (blocks + p.minper - 1) / p.minper);
  return p;
}

template <typename T> int launch(const Plan& p, const AttnArgs& a, int64_t bh, hipStream_t s) {
  const dim3 g((unsigned)bh, (unsigned)p.row_blocks, (unsigned)p.splits);
  if (p.tile) kv8_attn_tile_kernel<T><<<g, 512, 0, s>>>(a);
  else kv8_attn_rows_kernel<T><<<g, 256, 0, s>>>(a);
  if (p.splits > 1) {
    const dim3 mg((unsigned)((a.S * a.G + 7) / 8), (unsigned)bh);
    if (p.splits <= 2) kv8_merge_kernel<T, 2><<<mg, 256, 0, s>>>(a);
    else kv8_merge_kernel<T, 8><<<mg, 256, 0, s>>>(a);
  }
  return (int)hipGetLastError();
}

bool al16(const void* p) { return p && ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" {

size_t q3_kv8_attention_workspace_bytes(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t span) {
  if (B < 1 || S < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || span < 1) return 0;
  const Plan p = plan_for(B, Hkv, S * (Hq / Hkv), span);
  return p.splits > 1 ? (size_t)B * Hq * S * p.splits * (D + 2) * sizeof(float) : 0;
}

int q3_kv8_attention(int dtype, const void* q, int64_t qsb, int64_t qss, int64_t qsh, const int8_t* cache_k,
                     const int8_t* cache_v, const float* scale_k, const float* scale_v, const void* tail_k,
                     const void* tail_v, void* out, int64_t osb, int64_t oss, int64_t osh, void* workspace,
                     size_t workspace_bytes, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t d, int64_t capacity,
                     int64_t start, const int64_t* start_dev, float scale, hipStream_t stream) {
  Q3_REQUIRE((dtype == Q3_BF16 || dtype == Q3_F16) && d == D && al16(q) && out && ((uintptr_t)out & 7) == 0);
  Q3_REQUIRE(al16(cache_k) && al16(cache_v) && scale_k && scale_v && al16(tail_k) && al16(tail_v));
  Q3_REQUIRE(B > 0 && S > 0 && Hkv > 0 && Hq >= Hkv && Hq % Hkv == 0 && capacity > 0 && capacity < (1ll << 31) - 64);
  Q3_REQUIRE(B < 65536 && Hq < 65536 && B * Hkv < 65536);
  Q3_REQUIRE(start_dev ? S == 1 : (start >= 0 && start <= capacity && S <= capacity - start));
  for (int64_t st : {qsb, qss, qsh}) Q3_REQUIRE(st % 8 == 0);
  for (int64_t st : {osb, oss, osh}) Q3_REQUIRE(st % 4 == 0);
  Q3_REQUIRE(scale > 0.f && scale < 1e30f);  // the running maximum is of unscaled scores
  const int64_t rows = S * (Hq / Hkv);
  const Plan p = plan_for(B, Hkv, rows, start_dev ? capacity : start + S);
  Q3_REQUIRE(rows < (1ll << 31) - 128 && p.row_blocks < 65536);
  const int64_t parts = B * Hkv * rows * p.splits;
  if (p.splits > 1) Q3_REQUIRE(al16(workspace) && workspace_bytes >= (size_t)parts * (D + 2) * sizeof(float));
  float* ws = (float*)workspace;
  const AttnArgs a{(const u16*)q, qsb, qss, qsh, cache_k, cache_v, scale_k, scale_v, (const u16*)tail_k,
                   (const u16*)tail_v, (u16*)out, osb, oss, osh, ws, ws + parts * D, ws + parts * (D + 1), S, start,
                   capacity, start_dev, (int)Hkv, (int)(Hq / Hkv), p.splits, p.max_splits, p.minper,
                   scale * 1.4426950408889634f};
  return dtype == Q3_BF16 ? launch<BF16>(p, a, B * Hkv, stream) : launch<F16>(p, a, B * Hkv, stream);
}

}  // extern "C"
