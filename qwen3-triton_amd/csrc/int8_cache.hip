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
};

// One workgroup per (touched block, head, batch row); the one of the first block also writes the last, unfinished block's
// new positions into the tail (after it has read the tail, which may hold the first block's positions in the same slots).
// Thread t owns position t / 4 of the block and dims 32 (t % 4) .. + 31.
template <typename T> __global__ __launch_bounds__(256) void kv8_append_kernel(CacheArgs a) {
  __shared__ uint32_t red[2][4];
  __shared__ __attribute__((aligned(16))) int8_t vt[D][BLK + 16];
  const int tid = threadIdx.x, row = tid >> 2, d0 = (tid & 3) * 32;
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t start = a.start_dev ? *a.start_dev : a.start;
  const int64_t end = min(start + a.S, a.capacity);
  if (start < 0 || end <= start) return;
  const int64_t first = start / BLK, last = end / BLK;  // last: the first block that is not whole
  const int64_t blk = first + blockIdx.x;
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
  if (blockIdx.x != 0) return;
  // the last, unfinished block: every tail read above is done (the barriers), by this workgroup alone
  const int64_t pos = last * BLK + row;
  if (pos < start || pos >= end) return;
  const u16* kq = kp + (pos - start) * a.ks + d0;
  const u16* vq = vp + (pos - start) * a.vs + d0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    *reinterpret_cast<i32x4*>(tk + row * D + d0 + 8 * c) = *reinterpret_cast<const i32x4*>(kq + 8 * c);
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
  const CacheArgs a{(const u16*)k, (const u16*)v, ksb, kss, ksh, vsb, vss, vsh, cache_k, cache_v, scale_k, scale_v,
                    (u16*)tail_k, (u16*)tail_v, S, H, capacity, start, start_dev};
  // whole blocks touched, at least one workgroup (the tail's)
  const int64_t whole = start_dev ? 1 : (start + S) / BLK - start / BLK;
  const dim3 g((unsigned)(whole > 1 ? whole : 1), (unsigned)H, (unsigned)B);
  if (dtype == Q3_BF16) kv8_append_kernel<BF16><<<g, 256, 0, stream>>>(a);
  else kv8_append_kernel<F16><<<g, 256, 0, stream>>>(a);
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
