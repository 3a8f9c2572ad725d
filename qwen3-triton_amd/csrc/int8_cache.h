// The key/value cache in 8 bits: its layout, and the writing of new positions.
//
// Blocks of 64 positions with one scale per block and key/value head for the keys and one for the values.  A block is
// quantised once, from the 16-bit values, when its last position is written; until then its positions stay as they are in
// the tail.  So the stored codes do not depend on how a prompt was cut into chunks, no value is rounded twice, and the newest
// tokens are exact.  Layout per layer (Cb = capacity / 64 blocks, rounded up):
//   k [B, H, 64 Cb, 128] int8    v [B, H, Cb, 128, 64] int8: transposed within a block, so that the products of the
//   attention read 16-byte fragments of both as they lie    k_scale, v_scale [B, H, Cb] fp32
//   k_tail [B, H, 64, 128]    v_tail [B, H, 128, 64] in the activation type: position p at slot p % 64.
#pragma once
#include "int8.h"

namespace q3kv8 {

constexpr int D = 128, BLK = 64;

struct CacheArgs {
  const u16 *k, *v;                // new tokens [B, S, H, D]
  int64_t kb, ks, kh, vb, vs, vh;  // element strides (batch, position, head)
  int8_t *ck, *cv;
  float *sk, *sv;
  u16 *tk, *tv;
  int64_t S, H, capacity, start;
  const int64_t* start_dev;
  // with the Q/K-norm and rotation: k as projected, and the query rows beside it
  const u16 *q, *qw, *kw, *cs, *sn;  // q [B, S, Hq, D], norm weights [D], tables [B, S, D]
  int64_t qb, qs, qh;
  u16* yq;  // [B, S, Hq, D]
  int64_t B, Hq;
  int blocks;  // workgroups per head and batch row of the cache's part
  float eps;
};

// RMSNorm and split-half rotation of a 128-dim row whose dims 8 i .. + 7 sit in lane i of an aligned 16 (the partner dims, 64
// away, in lane i ^ 8), rounded once.
template <typename T>
Q3_DEV i32x4 norm_rope16(i32x4 x, const u16* w, const u16* cs, const u16* sn, float eps, int i) {
  const Vec<T> f = unpack_vec<T>(x), wf = load_vec<T>(w), cf = load_vec<T>(cs), sf = load_vec<T>(sn);
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += f.v[e] * f.v[e];
  const float inv = rsqrtf(group_sum<16>(ss) * (1.f / (float)D) + eps), sign = i < 8 ? -1.f : 1.f;
  Vec<T> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float n = f.v[e] * inv * wf.v[e];
    const float o = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, n), 0x128, 0xF, 0xF, true));
    y.v[e] = fmaf(n, cf.v[e], sign * (o * sf.v[e]));
  }
  i32x4 r;
#pragma unroll
  for (int p = 0; p < 4; ++p) r[p] = (int)pack2<T>(y.v[2 * p], y.v[2 * p + 1]);
  return r;
}

// LDS image of a block's V codes, transposed: word (d, r) holds the codes of dim d at positions 4 r .. + 3.  Dims of one lane
// group 16 words apart, lane groups 144, and r permuted by the group: the 64 words that a wave writes (or reads) for one dim
// per lane, and the 16-byte pieces of a dim, touch every bank once.
constexpr int kVWords = 16 * 144;
Q3_DEV int vword(int d, int r) { return (d >> 3) * 144 + (d & 7) * 16 + (r ^ (4 * (d >> 5))); }

// The new positions start .. end - 1 as far as block `part` (counted from the first one touched) goes; part 0 also writes the
// last, unfinished block's into the tail, after it has read the tail, which may hold the first block's positions in the same
// slots.  Keys and values are a workgroup's each (V).  256 threads: thread t owns positions 4 (t / 16) .. + 3 of the block and
// dims 8 (t % 16) .. + 7.
// NR: the keys come as projected and are normed and rotated here.
template <typename T, bool NR, bool V>
Q3_DEV void append_part(const CacheArgs& a, int part, int h, int b, int64_t start) {
  __shared__ __attribute__((aligned(16))) int vt[V ? kVWords : 4];
  __shared__ uint32_t red[4];
  const int tid = threadIdx.x, r = tid >> 4, i = tid & 15;
  const int64_t end = min(start + a.S, a.capacity);
  if (start < 0 || end <= start) return;
  const int64_t first = start / BLK, last = end / BLK;  // last: the first block that is not whole
  const int64_t blk = first + part;
  const int64_t bh = (int64_t)b * a.H + h, cblocks = (a.capacity + BLK - 1) / BLK;
  u16* tail = (V ? a.tv : a.tk) + bh * (BLK * D);
  const u16* src = V ? a.v + b * a.vb + h * a.vh : a.k + b * a.kb + h * a.kh;
  const int64_t stride = V ? a.vs : a.ks;
  auto fetch = [&](int64_t pos) {  // a new position's 8 dims
    i32x4 x = *reinterpret_cast<const i32x4*>(src + (pos - start) * stride + 8 * i);
    if constexpr (NR && !V) {
      const int64_t at = (b * a.S + pos - start) * D + 8 * i;
      x = norm_rope16<T>(x, a.kw + 8 * i, a.cs + at, a.sn + at, a.eps, i);
    }
    return x;
  };
  if (blk < last) {
    const int64_t pos0 = blk * BLK;
    const bool mixed = pos0 < start;  // positions before start are in the tail, V's transposed already
    i32x4 x[4];
    const int d = tid >> 1, half = (tid & 1) * 32;  // V, mixed: dim d, slots half .. + 31
    if (V && mixed) {
      const int from = (int)(start - pos0) - half;  // the first new one among this thread's slots
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = *reinterpret_cast<const i32x4*>(tail + d * BLK + half + 8 * c);
      u16 fresh[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) fresh[e] = src[(int64_t)max(e - from, 0) * stride + d];  // (no branch: the first one again)
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const uint32_t w = (uint32_t)x[e >> 3][(e >> 1) & 3], n = fresh[e];
        const uint32_t y = (e & 1) ? (w & 0xffffu) | (n << 16) : (w & 0xffff0000u) | n;
        x[e >> 3][(e >> 1) & 3] = (int)(e >= from ? y : w);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int64_t pos = pos0 + 4 * r + c;
        if (!V && pos < start) x[c] = *reinterpret_cast<const i32x4*>(tail + (4 * r + c) * D + 8 * i);
        else x[c] = fetch(pos);
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int p = 0; p < 4; ++p) m = mag_max16(m, (uint32_t)x[c][p]);
    m = wave_umax(mag_bits16<T>(m));
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    const bool finite = bits_finite(m);
    const QuantStep st = quant_step(finite ? __uint_as_float(m) : 0.f);
    if (tid == 0) (V ? a.sv : a.sk)[bh * cblocks + blk] = finite ? st.m / 127.f : __uint_as_float(0x7fc00000u);
    i32x2 q[4];  // the codes, in the order of x
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = finite ? quant_codes(unpack_vec<T>(x[c]).v, st) : i32x2{0, 0};
    int8_t* out = (V ? a.cv : a.ck) + (bh * cblocks + blk) * (D * BLK);
    if (!V) {
#pragma unroll
      for (int c = 0; c < 4; ++c) *reinterpret_cast<i32x2*>(out + (4 * r + c) * D + 8 * i) = q[c];
    } else if (mixed) {
      *reinterpret_cast<i32x4*>(out + d * BLK + half) = i32x4{q[0][0], q[0][1], q[1][0], q[1][1]};
      *reinterpret_cast<i32x4*>(out + d * BLK + half + 16) = i32x4{q[2][0], q[2][1], q[3][0], q[3][1]};
    } else {
#pragma unroll
      for (int w = 0; w < 2; ++w) {  // 4 dims x 4 positions: 4 positions of one dim to a word
        const uint32_t x0 = (uint32_t)q[0][w], x1 = (uint32_t)q[1][w], x2 = (uint32_t)q[2][w], x3 = (uint32_t)q[3][w];
        const uint32_t a01 = __builtin_amdgcn_perm(x1, x0, 0x05010400u), a23 = __builtin_amdgcn_perm(x3, x2, 0x05010400u);
        const uint32_t b01 = __builtin_amdgcn_perm(x1, x0, 0x07030602u), b23 = __builtin_amdgcn_perm(x3, x2, 0x07030602u);
        vt[vword(8 * i + 4 * w, r)] = (int)__builtin_amdgcn_perm(a23, a01, 0x05040100u);
        vt[vword(8 * i + 4 * w + 1, r)] = (int)__builtin_amdgcn_perm(a23, a01, 0x07060302u);
        vt[vword(8 * i + 4 * w + 2, r)] = (int)__builtin_amdgcn_perm(b23, b01, 0x05040100u);
        vt[vword(8 * i + 4 * w + 3, r)] = (int)__builtin_amdgcn_perm(b23, b01, 0x07060302u);
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int chunk = tid + 256 * c, vd = chunk >> 2, p = chunk & 3;  // dim, positions 16 p .. + 15
        *reinterpret_cast<i32x4*>(out + chunk * 16) = *reinterpret_cast<const i32x4*>(&vt[vword(vd, 4 * p)]);
      }
    }
  }
  if (part != 0) return;
  // the last, unfinished block: every tail read above is done (the barrier), by this workgroup alone
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int slot = 4 * r + c;
    const int64_t pos = last * BLK + slot;
    if (pos < start || pos >= end) continue;
    const i32x4 x = fetch(pos);
    if (!V) {
      *reinterpret_cast<i32x4*>(tail + slot * D + 8 * i) = x;
    } else {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        tail[(8 * i + 2 * p) * BLK + slot] = (u16)((uint32_t)x[p] & 0xffffu);
        tail[(8 * i + 2 * p + 1) * BLK + slot] = (u16)((uint32_t)x[p] >> 16);
      }
    }
  }
}

}  // namespace q3kv8
