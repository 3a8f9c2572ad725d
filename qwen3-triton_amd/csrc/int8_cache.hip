// The key/value cache in 8 bits: blocks of 64 positions with one scale per block and key/value head for the keys and one
// for the values, written as tokens come and read back to 16 or 32 bits.
//
// A block is quantised once, from the 16-bit values, when its last position is written; until then its positions stay as
// they are in the tail.  So the stored codes do not depend on how a prompt was cut into chunks, no value is rounded twice,
// and the newest tokens are exact.  Layout per layer (Cb = capacity / 64 blocks, rounded up):
//   k [B, H, 64 Cb, 128] int8    v [B, H, Cb, 128, 64] int8: transposed within a block, so that the products of the
//   attention read 16-byte fragments of both as they lie    k_scale, v_scale [B, H, Cb] fp32
//   k_tail [B, H, 64, 128]    v_tail [B, H, 128, 64] in the activation type: position p at slot p % 64.
// Both kernels are bound by HBM (a prompt's 2 + 1 bytes per value), by latency at one token.
#include "int8.h"

namespace {

constexpr int D = 128, BLK = 64;

struct CacheArgs {
  const u16 *k, *v;              // new tokens [B, S, H, D]
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

// RMSNorm and split-half rotation of a 128-dim row whose dims 32 i .. + 31 sit in lane i of an aligned quad (the partner
// dims, 64 away, in lane i ^ 2), rounded once: x holds 32 16-bit values.
template <typename T>
Q3_DEV void norm_rope_quad(i32x4 (&x)[4], const u16* w, const u16* cs, const u16* sn, float eps, int quarter) {
  Vec<T> f[4];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    f[c] = unpack_vec<T>(x[c]);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += f[c].v[e] * f[c].v[e];
  }
  ss = group_sum<4>(ss);
  const float inv = rsqrtf(ss * (1.f / (float)D) + eps), sign = quarter < 2 ? -1.f : 1.f;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const Vec<T> wf = load_vec<T>(w + 8 * c), cf = load_vec<T>(cs + 8 * c), sf = load_vec<T>(sn + 8 * c);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      float y[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = 2 * p + h;
        const float n = f[c].v[e] * inv * wf.v[e];
        const float o = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, n), 0x4E, 0xF, 0xF, true));
        y[h] = n * cf.v[e] + sign * o * sf.v[e];
      }
      x[c][p] = (int)pack2<T>(y[0], y[1]);
    }
  }
}

// One workgroup per (touched block, head, batch row); the one of the first block also writes the last, unfinished block's
// new positions into the tail (after it has read the tail, which may hold the first block's positions in the same slots).
// Thread t owns position t / 4 of the block and dims 32 (t % 4) .. + 31.
// NR: the rows come as projected and are normed and rotated here (values as they are); the workgroups behind the cache's
// take the query rows, 64 each.
template <typename T, bool NR> __global__ __launch_bounds__(256) void kv8_append_kernel(CacheArgs a) {
  __shared__ uint32_t red[2][4];
  __shared__ __attribute__((aligned(16))) int8_t vt[D][BLK + 16];
  const int tid = threadIdx.x, row = tid >> 2, d0 = (tid & 3) * 32;
  int64_t job = blockIdx.x;
  if constexpr (NR) {
    const int64_t cache_jobs = a.blocks * a.H * a.B;
    if (job >= cache_jobs) {
      const int64_t i = (job - cache_jobs) * 64 + row, n = a.B * a.S * a.Hq;  // whole quads: row is a quad's
      if (i >= n) return;
      const int64_t bs = i / a.Hq, qh = i - bs * a.Hq, qb = bs / a.S, qs = bs - qb * a.S;
      const u16* p = a.q + qb * a.qb + qs * a.qs + qh * a.qh + d0;
      i32x4 x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = *reinterpret_cast<const i32x4*>(p + 8 * c);
      norm_rope_quad<T>(x, a.qw + d0, a.cs + bs * D + d0, a.sn + bs * D + d0, a.eps, tid & 3);
#pragma unroll
      for (int c = 0; c < 4; ++c) *reinterpret_cast<i32x4*>(a.yq + i * D + d0 + 8 * c) = x[c];
      return;
    }
  }
  const int part = (int)(job % a.blocks);
  job /= a.blocks;
  const int h = (int)(job % a.H), b = (int)(job / a.H);
  const int64_t start = a.start_dev ? *a.start_dev : a.start;
  const int64_t end = min(start + a.S, a.capacity);
  if (start < 0 || end <= start) return;
  const int64_t first = start / BLK, last = end / BLK;  // last: the first block that is not whole
  const int64_t blk = first + part;
  const int64_t bh = (int64_t)b * a.H + h, cblocks = (a.capacity + BLK - 1) / BLK;
  u16* tk = a.tk + bh * (BLK * D);
  u16* tv = a.tv + bh * (BLK * D);
  const u16* kp = a.k + b * a.kb + h * a.kh;
  const u16* vp = a.v + b * a.vb + h * a.vh;
  if (blk < last) {
    const int64_t pos = blk * BLK + row;
    i32x4 kr[4], vr[4];
    if (pos >= start) {
      const u16* kq = kp + (pos - start) * a.ks + d0;
      const u16* vq = vp + (pos - start) * a.vs + d0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        kr[c] = *reinterpret_cast<const i32x4*>(kq + 8 * c);
        vr[c] = *reinterpret_cast<const i32x4*>(vq + 8 * c);
      }
      if constexpr (NR) {
        const int64_t at = (b * a.S + pos - start) * D + d0;
        norm_rope_quad<T>(kr, a.kw + d0, a.cs + at, a.sn + at, a.eps, tid & 3);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        kr[c] = *reinterpret_cast<const i32x4*>(tk + row * D + d0 + 8 * c);
#pragma unroll
        for (int p = 0; p < 4; ++p)
          vr[c][p] = (int)((uint32_t)tv[(d0 + 8 * c + 2 * p) * BLK + row] |
                           ((uint32_t)tv[(d0 + 8 * c + 2 * p + 1) * BLK + row] << 16));
      }
    }
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const Vec<T> x = unpack_vec<T>(kr[c]), y = unpack_vec<T>(vr[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        mk = max(mk, mag_bits(x.v[e]));
        mv = max(mv, mag_bits(y.v[e]));
      }
    }
    mk = group_umax<64>(mk);
    mv = group_umax<64>(mv);
    if ((tid & 63) == 0) {
      red[0][tid >> 6] = mk;
      red[1][tid >> 6] = mv;
    }
    __syncthreads();
    mk = max(max(red[0][0], red[0][1]), max(red[0][2], red[0][3]));
    mv = max(max(red[1][0], red[1][1]), max(red[1][2], red[1][3]));
    const bool fk = bits_finite(mk), fv = bits_finite(mv);
    const QuantStep sk = quant_step(fk ? __uint_as_float(mk) : 0.f), sv = quant_step(fv ? __uint_as_float(mv) : 0.f);
    if (tid == 0) {
      const float nan = __uint_as_float(0x7fc00000u);
      a.sk[bh * cblocks + blk] = fk ? sk.m / 127.f : nan;
      a.sv[bh * cblocks + blk] = fv ? sv.m / 127.f : nan;
    }
    int kc[8];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const Vec<T> x = unpack_vec<T>(kr[c]), y = unpack_vec<T>(vr[c]);
      float q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = fk ? quant_code(x.v[e], sk) : 0.f;
      kc[2 * c] = pack_codes(q[0], q[1], q[2], q[3]);
      kc[2 * c + 1] = pack_codes(q[4], q[5], q[6], q[7]);
#pragma unroll
      for (int e = 0; e < 8; ++e) vt[d0 + 8 * c + e][row] = (int8_t)(fv ? (int)quant_code(y.v[e], sv) : 0);
    }
    int8_t* ck = a.ck + (bh * cblocks * BLK + pos) * D + d0;
    *reinterpret_cast<i32x4*>(ck) = i32x4{kc[0], kc[1], kc[2], kc[3]};
    *reinterpret_cast<i32x4*>(ck + 16) = i32x4{kc[4], kc[5], kc[6], kc[7]};
    __syncthreads();
    int8_t* cv = a.cv + (bh * cblocks + blk) * (D * BLK);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int chunk = tid + 256 * i;  // dim chunk / 4, positions 16 (chunk % 4) .. + 15
      *reinterpret_cast<i32x4*>(cv + chunk * 16) = *reinterpret_cast<const i32x4*>(&vt[chunk >> 2][(chunk & 3) * 16]);
    }
  }
  if (part != 0) return;
  // the last, unfinished block: every tail read above is done (the barriers), by this workgroup alone
  const int64_t pos = last * BLK + row;
  if (pos < start || pos >= end) return;
  const u16* kq = kp + (pos - start) * a.ks + d0;
  const u16* vq = vp + (pos - start) * a.vs + d0;
  i32x4 kr[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) kr[c] = *reinterpret_cast<const i32x4*>(kq + 8 * c);
  if constexpr (NR) {
    const int64_t at = (b * a.S + pos - start) * D + d0;
    norm_rope_quad<T>(kr, a.kw + d0, a.cs + at, a.sn + at, a.eps, tid & 3);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    *reinterpret_cast<i32x4*>(tk + row * D + d0 + 8 * c) = kr[c];
    const i32x4 x = *reinterpret_cast<const i32x4*>(vq + 8 * c);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      tv[(d0 + 8 * c + 2 * p) * BLK + row] = (u16)((uint32_t)x[p] & 0xffffu);
      tv[(d0 + 8 * c + 2 * p + 1) * BLK + row] = (u16)((uint32_t)x[p] >> 16);
    }
  }
}

struct ReadArgs {
  const int8_t *ck, *cv;
  const float *sk, *sv;
  const u16 *tk, *tv;
  void *k, *v;  // [B, H, length, D]
  int64_t H, capacity, length;
};

// out = code * scale, rounded once; tail positions converted as they are.  One workgroup per (block, head, batch row).
template <typename T, typename O> __global__ __launch_bounds__(256) void kv8_read_kernel(ReadArgs a) {
  __shared__ __attribute__((aligned(16))) int8_t vt[D][BLK + 16];
  typedef typename O::storage out_t;
  const int tid = threadIdx.x, row = tid >> 2, d0 = (tid & 3) * 32;
  const int64_t blk = blockIdx.x, bh = (int64_t)blockIdx.z * a.H + blockIdx.y, cblocks = (a.capacity + BLK - 1) / BLK;
  const int64_t pos = blk * BLK + row;
  const bool whole = (blk + 1) * BLK <= a.length;
  float x[32], y[32];
  if (whole) {
    const int8_t* cv = a.cv + (bh * cblocks + blk) * (D * BLK);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int chunk = tid + 256 * i;
      *reinterpret_cast<i32x4*>(&vt[chunk >> 2][(chunk & 3) * 16]) = *reinterpret_cast<const i32x4*>(cv + chunk * 16);
    }
    const int8_t* ck = a.ck + (bh * cblocks * BLK + pos) * D + d0;
    const float sk = a.sk[bh * cblocks + blk], sv = a.sv[bh * cblocks + blk];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const i32x4 w = *reinterpret_cast<const i32x4*>(ck + 16 * c);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[16 * c + e] = (float)(int8_t)((uint32_t)w[e >> 2] >> (8 * (e & 3))) * sk;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 32; ++e) y[e] = (float)vt[d0 + e][row] * sv;
  } else {
    if (pos >= a.length) return;
    const u16* tk = a.tk + bh * (BLK * D) + row * D + d0;
    const u16* tv = a.tv + bh * (BLK * D) + d0 * BLK + row;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      x[e] = to_f32<T>(tk[e]);
      y[e] = to_f32<T>(tv[e * BLK]);
    }
  }
  out_t* ko = reinterpret_cast<out_t*>(a.k) + (bh * a.length + pos) * D + d0;
  out_t* vo = reinterpret_cast<out_t*>(a.v) + (bh * a.length + pos) * D + d0;
#pragma unroll
  for (int c = 0; c < 32 / O::vec; ++c) {
    Vec<O> p, q;
#pragma unroll
    for (int e = 0; e < O::vec; ++e) {
      p.v[e] = x[c * O::vec + e];
      q.v[e] = y[c * O::vec + e];
    }
    store_vec<O>(ko + c * O::vec, p);
    store_vec<O>(vo + c * O::vec, q);
  }
}

bool al16(const void* p) { return p && ((uintptr_t)p & 15) == 0; }

bool cache_ok(const void* ck, const void* cv, const float* sk, const float* sv, const void* tk, const void* tv, int64_t B,
              int64_t H, int64_t capacity) {
  return al16(ck) && al16(cv) && sk && sv && al16(tk) && al16(tv) && B > 0 && B < 65536 && H > 0 && H < 65536 &&
         capacity > 0 && capacity < (1ll << 31) - 64;
}

// Workgroups per head: the blocks that the new positions complete, at least one (the tail's).
int append_blocks(const CacheArgs& a) {
  const int64_t whole = a.start_dev ? 1 : (a.start + a.S) / BLK - a.start / BLK;
  return (int)(whole > 1 ? whole : 1);
}

template <typename T> int read_as(int out, const ReadArgs& a, dim3 g, hipStream_t s) {
  switch (out) {
    case Q3_F32: kv8_read_kernel<T, F32><<<g, 256, 0, s>>>(a); break;
    case Q3_F16: kv8_read_kernel<T, F16><<<g, 256, 0, s>>>(a); break;
    default: kv8_read_kernel<T, BF16><<<g, 256, 0, s>>>(a); break;
  }
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

int q3_kv8_append(int dtype, const void* k, int64_t ksb, int64_t kss, int64_t ksh, const void* v, int64_t vsb, int64_t vss,
                  int64_t vsh, int8_t* cache_k, int8_t* cache_v, float* scale_k, float* scale_v, void* tail_k, void* tail_v,
                  int64_t B, int64_t S, int64_t H, int64_t d, int64_t capacity, int64_t start, const int64_t* start_dev,
                  hipStream_t stream) {
  Q3_REQUIRE((dtype == Q3_BF16 || dtype == Q3_F16) && d == D && al16(k) && al16(v));
  Q3_REQUIRE(cache_ok(cache_k, cache_v, scale_k, scale_v, tail_k, tail_v, B, H, capacity));
  Q3_REQUIRE(S > 0 && (start_dev ? S == 1 : (start >= 0 && start <= capacity && S <= capacity - start)));
  for (int64_t st : {ksb, kss, ksh, vsb, vss, vsh}) Q3_REQUIRE(st % 8 == 0);
  CacheArgs a{(const u16*)k, (const u16*)v, ksb, kss, ksh, vsb, vss, vsh, cache_k, cache_v, scale_k, scale_v,
              (u16*)tail_k, (u16*)tail_v, S, H, capacity, start, start_dev};
  a.B = B;
  a.blocks = append_blocks(a);
  Q3_REQUIRE(a.blocks * H * B < (1ll << 31));
  const unsigned g = (unsigned)(a.blocks * H * B);
  if (dtype == Q3_BF16) kv8_append_kernel<BF16, false><<<g, 256, 0, stream>>>(a);
  else kv8_append_kernel<F16, false><<<g, 256, 0, stream>>>(a);
  return (int)hipGetLastError();
}

int q3_kv8_norm_rope_append(int dtype, const void* q, int64_t qsb, int64_t qss, int64_t qsh, const void* k, int64_t ksb,
                            int64_t kss, int64_t ksh, const void* v, int64_t vsb, int64_t vss, int64_t vsh, const void* wq,
                            const void* wk, const void* cos, const void* sin, void* yq, int8_t* cache_k, int8_t* cache_v,
                            float* scale_k, float* scale_v, void* tail_k, void* tail_v, int64_t B, int64_t S, int64_t Hq,
                            int64_t H, int64_t d, int64_t capacity, int64_t start, const int64_t* start_dev, float eps,
                            hipStream_t stream) {
  Q3_REQUIRE((dtype == Q3_BF16 || dtype == Q3_F16) && d == D && al16(q) && al16(k) && al16(v) && al16(wq) && al16(wk) &&
             al16(cos) && al16(sin) && al16(yq) && Hq > 0 && Hq < 65536 && eps >= 0.f);
  Q3_REQUIRE(cache_ok(cache_k, cache_v, scale_k, scale_v, tail_k, tail_v, B, H, capacity));
  Q3_REQUIRE(S > 0 && (start_dev ? S == 1 : (start >= 0 && start <= capacity && S <= capacity - start)));
  for (int64_t st : {qsb, qss, qsh, ksb, kss, ksh, vsb, vss, vsh}) Q3_REQUIRE(st % 8 == 0);
  CacheArgs a{(const u16*)k, (const u16*)v, ksb, kss, ksh, vsb, vss, vsh, cache_k, cache_v, scale_k, scale_v,
              (u16*)tail_k, (u16*)tail_v, S, H, capacity, start, start_dev, (const u16*)q, (const u16*)wq, (const u16*)wk,
              (const u16*)cos, (const u16*)sin, qsb, qss, qsh, (u16*)yq, B, Hq, 0, eps};
  a.blocks = append_blocks(a);
  const int64_t g = a.blocks * H * B + (B * S * Hq + 63) / 64;
  Q3_REQUIRE(g < (1ll << 31));
  if (dtype == Q3_BF16) kv8_append_kernel<BF16, true><<<(unsigned)g, 256, 0, stream>>>(a);
  else kv8_append_kernel<F16, true><<<(unsigned)g, 256, 0, stream>>>(a);
  return (int)hipGetLastError();
}

int q3_kv8_read(int dtype, int out_dtype, const int8_t* cache_k, const int8_t* cache_v, const float* scale_k,
                const float* scale_v, const void* tail_k, const void* tail_v, void* k, void* v, int64_t B, int64_t H,
                int64_t d, int64_t capacity, int64_t length, hipStream_t stream) {
  Q3_REQUIRE((dtype == Q3_BF16 || dtype == Q3_F16) && out_dtype >= Q3_F32 && out_dtype <= Q3_BF16 && d == D);
  Q3_REQUIRE(cache_ok(cache_k, cache_v, scale_k, scale_v, tail_k, tail_v, B, H, capacity) && al16(k) && al16(v));
  Q3_REQUIRE(length > 0 && length <= capacity);
  const ReadArgs a{cache_k, cache_v, scale_k, scale_v, (const u16*)tail_k, (const u16*)tail_v, k, v, H, capacity, length};
  const dim3 g((unsigned)((length + BLK - 1) / BLK), (unsigned)H, (unsigned)B);
  return dtype == Q3_BF16 ? read_as<BF16>(out_dtype, a, g, stream) : read_as<F16>(out_dtype, a, g, stream);
}

}  // extern "C"
