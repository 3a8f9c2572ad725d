// Writing new positions into the key/value cache in 8 bits (int8_cache.h), and reading the cache back to 16 or 32 bits.
// Bound by HBM (a prompt's 2 + 1 bytes per value, and back), by latency at one token.  Measured with 8 heads: 8192 positions
// appended in 15.8 us (3.2 TB/s; a copy of the same bytes 11.7 us, the quantisation about 4 on top of it), read back in 9.0
// (5.6 TB/s); one token of 8 rows 2.3 us, 5.8 - 8.3 us where it completes a block, whose 64 positions are then read from the
// tail, in one chain of three waits.
#include "int8_cache.h"

namespace {

using namespace q3kv8;

// Two workgroups per (touched block, head, batch row), for the keys and the values (in one, a token that completes a block took
// 8.7 us, not 5.6); with the norm and rotation, the ones behind them take 16 query rows each.
template <typename T, bool NR> __global__ __launch_bounds__(256) void kv8_append_kernel(CacheArgs a) {
  int64_t job = blockIdx.x;
  if constexpr (NR) {
    const int64_t cache_jobs = 2 * a.blocks * a.H * a.B;
    if (job >= cache_jobs) {
      const int tid = threadIdx.x, i = tid & 15;
      const int64_t at = (job - cache_jobs) * 16 + (tid >> 4);  // a 16-lane row's query
      if (at >= a.B * a.S * a.Hq) return;
      const int64_t bs = at / a.Hq, qh = at - bs * a.Hq, qb = bs / a.S, qs = bs - qb * a.S;
      const i32x4 x = *reinterpret_cast<const i32x4*>(a.q + qb * a.qb + qs * a.qs + qh * a.qh + 8 * i);
      *reinterpret_cast<i32x4*>(a.yq + at * D + 8 * i) =
          norm_rope16<T>(x, a.qw + 8 * i, a.cs + bs * D + 8 * i, a.sn + bs * D + 8 * i, a.eps, i);
      return;
    }
  }
  const bool values = job & 1;
  job >>= 1;
  const int h = (int)(job % a.H);  // heads next to each other, as their rows are in memory
  job /= a.H;
  const int64_t start = a.start_dev ? *a.start_dev : a.start;
  const int b = (int)(job % a.B), part = (int)(job / a.B);  // the parts that may read the tail first: they take longest
  if (values) append_part<T, NR, true>(a, part, h, b, start);
  else append_part<T, NR, false>(a, part, h, b, start);
}

struct ReadArgs {
  const int8_t *ck, *cv;
  const float *sk, *sv;
  const u16 *tk, *tv;
  void *k, *v;  // [B, H, length, D]
  int64_t H, capacity, length;
};

// out = code * scale, rounded once; tail positions converted as they are.  One workgroup per (block, head, batch row), threads
// and LDS image as in append_part.
template <typename T, typename O> __global__ __launch_bounds__(256) void kv8_read_kernel(ReadArgs a) {
  __shared__ __attribute__((aligned(16))) int vt[kVWords];
  typedef typename O::storage out_t;
  const int tid = threadIdx.x, r = tid >> 4, i = tid & 15;
  const int64_t blk = blockIdx.x, bh = (int64_t)blockIdx.z * a.H + blockIdx.y, cblocks = (a.capacity + BLK - 1) / BLK;
  const int64_t pos0 = blk * BLK + 4 * r;
  out_t* ko = reinterpret_cast<out_t*>(a.k) + (bh * a.length + pos0) * D + 8 * i;
  out_t* vo = reinterpret_cast<out_t*>(a.v) + (bh * a.length + pos0) * D + 8 * i;
  auto store = [&](out_t* p, const float (&x)[8]) {
#pragma unroll
    for (int c = 0; c < 8 / O::vec; ++c) {
      Vec<O> y;
#pragma unroll
      for (int e = 0; e < O::vec; ++e) y.v[e] = x[c * O::vec + e];
      store_vec<O>(p + c * O::vec, y);
    }
  };
  if ((blk + 1) * BLK <= a.length) {
    const int8_t* cv = a.cv + (bh * cblocks + blk) * (D * BLK);
    const int8_t* ck = a.ck + (bh * cblocks * BLK + pos0) * D + 8 * i;
    i32x4 vraw[2];
    i32x2 kraw[4];
#pragma unroll
    for (int c = 0; c < 2; ++c) vraw[c] = *reinterpret_cast<const i32x4*>(cv + (tid + 256 * c) * 16);
#pragma unroll
    for (int c = 0; c < 4; ++c) kraw[c] = *reinterpret_cast<const i32x2*>(ck + c * D);
    const float sk = a.sk[bh * cblocks + blk], sv = a.sv[bh * cblocks + blk];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int chunk = tid + 256 * c;
      *reinterpret_cast<i32x4*>(&vt[vword(chunk >> 2, 4 * (chunk & 3))]) = vraw[c];
    }
    float x[8];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)((uint32_t)kraw[c][e >> 2] >> (8 * (e & 3))) * sk;
      store(ko + c * D, x);
    }
    __syncthreads();
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = (uint32_t)vt[vword(8 * i + e, r)];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)(w[e] >> (8 * c)) * sv;
      store(vo + c * D, x);
    }
    return;
  }
  const u16* tk = a.tk + bh * (BLK * D) + 4 * r * D + 8 * i;
  const u16* tv = a.tv + bh * (BLK * D) + 8 * i * BLK + 4 * r;
  i32x4 kraw[4];
  i32x2 vraw[8];  // a dim's four positions
#pragma unroll
  for (int c = 0; c < 4; ++c) kraw[c] = *reinterpret_cast<const i32x4*>(tk + c * D);
#pragma unroll
  for (int e = 0; e < 8; ++e) vraw[e] = *reinterpret_cast<const i32x2*>(tv + e * BLK);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (pos0 + c >= a.length) continue;
    const Vec<T> k = unpack_vec<T>(kraw[c]);
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = k.v[e];
      y[e] = to_f32<T>((u16)((uint32_t)vraw[e][c >> 1] >> (16 * (c & 1))));
    }
    store(ko + c * D, x);
    store(vo + c * D, y);
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
  Q3_REQUIRE(2 * a.blocks * H * B < (1ll << 31));
  const unsigned g = (unsigned)(2 * a.blocks * H * B);
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
  const int64_t g = 2 * a.blocks * H * B + (B * S * Hq + 15) / 16;
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
