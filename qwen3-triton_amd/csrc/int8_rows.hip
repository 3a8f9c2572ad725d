// Rows of activations (or weight channels) in 8 bits with one scale per row, and RMSNorm with that output.
//
//   quantize_rows: M = max |x|, q = nearest(127 x / M), scale = M / 127.
//   rms_norm:      t = round(x + residual), a = t w, M = max |a|, q = nearest(127 a / M),
//                  scale = M / 127 * rsqrt(mean t^2 + eps).
// The norm's 1 / rms is common to a row, so it belongs into the scale alone: the codes need no square root and no
// rounded normalised value, and a = t w of two 16-bit numbers is exact in 32 bits.
//
// Bound by HBM at many rows (2 bytes in, 1 out per value, 4 more with a residual and its sum), by latency at few: a row
// is read once, held packed in registers by TPR threads, and both reductions (sum of squares, largest magnitude) share
// one pair of barriers.  Threads per row by its length, so that each holds two vectors up to 8192 values and four above (all
// of a row's loads in flight at once).  Measured: norm with residual over 8192 x 4096 42.5 us (5.5 TB/s), rows of 1500 x 12288
// 11.2 us (4.9 TB/s), one row of 4096 2.6 us, a launch's own time.
#include "int8.h"

namespace {

constexpr int64_t kMaxRow = 32768;  // values that 1024 threads hold in 4 vectors each

struct RowArgs {
  const u16* x;
  int64_t ldx;
  const u16* res;
  int64_t ldres;
  const u16* w;
  int8_t* q;
  float* scale;
  u16* total;
  int64_t rows;
  int h;
  float eps;
};

// TPR threads per row, MAXV 16-byte vectors per thread; TPR / 64 waves reduce through LDS when a row spans several.
template <typename T, int TPR, int MAXV, int BLOCK, bool NORM, bool RES>
__global__ __launch_bounds__(BLOCK) void quant_rows_kernel(RowArgs a) {
  constexpr int RPB = BLOCK / TPR, NWR = TPR / 64;
  __shared__ float red_s[BLOCK / 64];
  __shared__ uint32_t red_m[BLOCK / 64];
  const int t = threadIdx.x % TPR, nvec = a.h / 8;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const bool live = row < a.rows;
  const int64_t rc = live ? row : a.rows - 1;
  const u16* xp = a.x + rc * a.ldx;
  i32x4 tv[MAXV], rv[RES ? MAXV : 1], wv[NORM ? MAXV : 1];
#pragma unroll
  for (int j = 0; j < MAXV; ++j) {
    const int v = min(t + j * TPR, nvec - 1);
    tv[j] = *reinterpret_cast<const i32x4*>(xp + v * 8);
    if constexpr (RES) rv[j] = *reinterpret_cast<const i32x4*>(a.res + rc * a.ldres + v * 8);
    if constexpr (NORM) wv[j] = *reinterpret_cast<const i32x4*>(a.w + v * 8);
  }
  float ss = 0.f;
  uint32_t mb = 0;
#pragma unroll
  for (int j = 0; j < MAXV; ++j) {
    const bool in = t + j * TPR < nvec;
    Vec<T> x = unpack_vec<T>(tv[j]);
    if constexpr (RES) {
      const Vec<T> r = unpack_vec<T>(rv[j]);
#pragma unroll
      for (int p = 0; p < 4; ++p)
        tv[j][p] = (int)pack2<T>(x.v[2 * p] + r.v[2 * p], x.v[2 * p + 1] + r.v[2 * p + 1]);
      x = unpack_vec<T>(tv[j]);
      if (in && live) *reinterpret_cast<i32x4*>(a.total + row * a.h + (t + j * TPR) * 8) = tv[j];
    }
    if (in) {
      if constexpr (NORM) {
        const Vec<T> w = unpack_vec<T>(wv[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss += x.v[e] * x.v[e];
          mb = max(mb, mag_bits(x.v[e] * w.v[e]));
        }
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) mb = mag_max16(mb, (uint32_t)tv[j][p]);
      }
    }
  }
  if constexpr (!NORM) mb = mag_bits16<T>(mb);
  mb = wave_umax(mb);
  if constexpr (NORM) ss = group_sum<64>(ss);
  if constexpr (NWR > 1) {
    const int wv_id = threadIdx.x >> 6, w0 = (threadIdx.x / TPR) * NWR;
    if (lane_id() == 0) {
      red_m[wv_id] = mb;
      red_s[wv_id] = ss;
    }
    __syncthreads();
    mb = red_m[w0];
    ss = red_s[w0];
#pragma unroll
    for (int i = 1; i < NWR; ++i) {
      mb = mb > red_m[w0 + i] ? mb : red_m[w0 + i];
      ss += red_s[w0 + i];
    }
  }
  if (!live) return;
  const bool finite = bits_finite(mb);
  const float m = finite ? __uint_as_float(mb) : 0.f;
  if (t == 0) {
    float s = finite ? m / 127.f : __uint_as_float(0x7fc00000u);
    if constexpr (NORM) s *= rsqrtf(ss * (1.f / (float)a.h) + a.eps);
    a.scale[row] = s;
  }
  const QuantStep st = quant_step(m);
#pragma unroll
  for (int j = 0; j < MAXV; ++j) {
    if (t + j * TPR >= nvec) continue;
    Vec<T> x = unpack_vec<T>(tv[j]);
    if constexpr (NORM) {
      const Vec<T> w = unpack_vec<T>(wv[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x.v[e] *= w.v[e];
    }
    *reinterpret_cast<i32x2*>(a.q + row * a.h + (t + j * TPR) * 8) = finite ? quant_codes(x.v, st) : i32x2{0, 0};
  }
}

template <typename T, int TPR, int MAXV, int BLOCK> int launch_rows(const RowArgs& a, hipStream_t s) {
  const unsigned g = (unsigned)((a.rows + BLOCK / TPR - 1) / (BLOCK / TPR));
  if (a.w && a.res) quant_rows_kernel<T, TPR, MAXV, BLOCK, true, true><<<g, BLOCK, 0, s>>>(a);
  else if (a.w) quant_rows_kernel<T, TPR, MAXV, BLOCK, true, false><<<g, BLOCK, 0, s>>>(a);
  else quant_rows_kernel<T, TPR, MAXV, BLOCK, false, false><<<g, BLOCK, 0, s>>>(a);
  return (int)hipGetLastError();
}

template <typename T> int rows_for(const RowArgs& a, hipStream_t s) {
  if (a.h <= 512) return launch_rows<T, 64, 1, 256>(a, s);
  if (a.h <= 1024) return launch_rows<T, 64, 2, 256>(a, s);
  if (a.h <= 2048) return launch_rows<T, 256, 1, 256>(a, s);
  if (a.h <= 4096) return launch_rows<T, 256, 2, 256>(a, s);
  if (a.h <= 8192) return launch_rows<T, 512, 2, 512>(a, s);
  if (a.h <= 16384) return launch_rows<T, 512, 4, 512>(a, s);
  return launch_rows<T, 1024, 4, 1024>(a, s);
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int rows_call(int dtype, const RowArgs& a, hipStream_t s) {
  Q3_REQUIRE(dtype == Q3_BF16 || dtype == Q3_F16);
  Q3_REQUIRE(a.x && a.q && a.scale && a.rows > 0 && a.rows < (1ll << 31) && a.h >= 16 && a.h % 16 == 0 && a.h <= kMaxRow);
  Q3_REQUIRE(al16(a.x) && al16(a.q) && ((uintptr_t)a.scale & 3) == 0 && a.ldx >= a.h && a.ldx % 8 == 0);
  return dtype == Q3_BF16 ? rows_for<BF16>(a, s) : rows_for<F16>(a, s);
}

}  // namespace

extern "C" {

int q3_quant_rows(int dtype, const void* x, int64_t ldx, int8_t* q, float* scale, int64_t rows, int64_t h,
                  hipStream_t stream) {
  Q3_REQUIRE(h > 0 && h <= kMaxRow);
  RowArgs a{};
  a.x = (const u16*)x;
  a.ldx = ldx;
  a.q = q;
  a.scale = scale;
  a.rows = rows;
  a.h = (int)h;
  return rows_call(dtype, a, stream);
}

int q3_rmsnorm_quant(int dtype, const void* x, int64_t ldx, const void* res, int64_t ldres, const void* w, int8_t* q,
                     float* scale, void* total, int64_t rows, int64_t h, float eps, hipStream_t stream) {
  Q3_REQUIRE(h > 0 && h <= kMaxRow && w && al16(w) && !res == !total && eps >= 0.f);
  if (res) Q3_REQUIRE(al16(res) && al16(total) && ldres >= h && ldres % 8 == 0);
  RowArgs a{};
  a.x = (const u16*)x;
  a.ldx = ldx;
  a.res = (const u16*)res;
  a.ldres = ldres;
  a.w = (const u16*)w;
  a.q = q;
  a.scale = scale;
  a.total = (u16*)total;
  a.rows = rows;
  a.h = (int)h;
  a.eps = eps;
  return rows_call(dtype, a, stream);
}

}  // extern "C"
