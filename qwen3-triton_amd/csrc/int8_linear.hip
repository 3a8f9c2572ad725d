// Products of at most 16 rows of 8-bit codes (a decode step) with weights in 8 bits: y = (x W^T) s ws (+ res), and the
// gate/up + SwiGLU form; up to three weights of one input in a launch.
//
// Bound by the weights' bytes.  A workgroup owns 16 output channels and streams their rows straight into registers as the
// B operand of v_mfma_i32_16x16x64_i8 (lane (r, kq): 16 codes of row r at k = 16 kq of every 64), the token rows as the A
// operand; its 8 waves take 256-wide k blocks in turn, P of them in flight, and fold their int32 tiles in LDS: exact, so in
// any order.
#include "gemm_tile.h"

namespace q3gemm {

template <typename T, int EPI, int P> __global__ __launch_bounds__(512) void gemm_rows_q8_kernel(Args a) {
  constexpr int NW = 8, NB = EPI == 3 ? 2 : 1;
  __shared__ i32x4 red[NW - 1][NB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, kq = lane >> 4;
  const int M = (int)a.M, K = (int)a.K * 2;  // codes
  int tile = blockIdx.x, s = 0;
  if (EPI != 3 && a.axis == 2)
    while (s + 1 < a.pieces && tile >= ((int)a.len[s] + 15) / 16) tile -= ((int)a.len[s++] + 15) / 16;
  const int ncols = EPI == 3 ? (int)a.N / 2 : a.axis == 2 ? (int)a.len[s] : (int)a.N, n0 = tile * 16;
  const int8_t* x = reinterpret_cast<const int8_t*>(a.a.p[0]) + (int64_t)min(r, M - 1) * a.a.ld[0] * 2 + 16 * kq;
  const int8_t* w[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int i = EPI == 3 ? j : s;
    w[j] = reinterpret_cast<const int8_t*>(a.b.p[i]) + (int64_t)min(n0 + r, ncols - 1) * a.b.ld[i] * 2 + 16 * kq;
  }
  const bool live = r < M;
  i32x4 acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j] = i32x4{0, 0, 0, 0};
  auto blocks = [&](auto qc, int b) {  // k blocks b, b + NW, ...: every load before the first product
    constexpr int Q = decltype(qc)::value;
    i32x4 wv[Q][NB][4], xv[Q][4];
#pragma unroll
    for (int p = 0; p < Q; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int k = (b + p * NW) * 256 + 64 * c;
        const bool ok = k + 16 * kq < K;
#pragma unroll
        for (int j = 0; j < NB; ++j) wv[p][j][c] = ok ? *reinterpret_cast<const i32x4*>(w[j] + k) : i32x4{0, 0, 0, 0};
        xv[p][c] = ok && live ? *reinterpret_cast<const i32x4*>(x + k) : i32x4{0, 0, 0, 0};
      }
#pragma unroll
    for (int p = 0; p < Q; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < NB; ++j)
          mfma_acc(acc[j], __builtin_bit_cast(bf16x8_t, xv[p][c]), __builtin_bit_cast(bf16x8_t, wv[p][j][c]));
  };
  const int nblk = (K + 255) / 256;
  int b = wave;
  for (; b + (P - 1) * NW < nblk; b += P * NW) blocks(std::integral_constant<int, P>{}, b);
  for (; b < nblk; b += NW) blocks(std::integral_constant<int, 1>{}, b);
  if (wave > 0) {
#pragma unroll
    for (int j = 0; j < NB; ++j) red[wave - 1][j][lane] = acc[j];
  }
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < NW - 1; ++i) acc[j] += red[i][j][lane];
  // lane holds rows 4 kq + e of column n0 + r
  const int n = n0 + r;
  if (n >= ncols) return;
  const float cs = a.cscale[EPI == 3 ? 0 : s][n], cu = EPI == 3 ? a.cscale[1][n] : 0.f;
  u16* y = reinterpret_cast<u16*>(a.c[EPI == 3 ? 0 : s]);
  const int64_t ldc = a.ldc[EPI == 3 ? 0 : s];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int m = 4 * kq + e;
    if (m >= M) continue;
    const float rs = a.rscale[m];
    float v = (float)acc[0][e] * rs * cs;
    if constexpr (EPI == 3) v = v * q3_sigmoid(v) * ((float)acc[NB - 1][e] * rs * cu);
    else if (a.res) v += to_f32<T>(a.res[m * a.ldres + n]);
    y[m * ldc + n] = from_f32<T>(v);
  }
}

template <typename T> static int rows_q8(int epi, const Args& a, hipStream_t s) {
  int64_t tiles = 0;
  if (epi == 3) tiles = (a.N / 2 + 15) / 16;
  else if (a.axis == 2)
    for (int i = 0; i < a.pieces; ++i) tiles += (a.len[i] + 15) / 16;
  else tiles = (a.N + 15) / 16;
  if (epi == 3) gemm_rows_q8_kernel<T, 3, 2><<<(unsigned)tiles, 512, 0, s>>>(a);
  else gemm_rows_q8_kernel<T, 0, 2><<<(unsigned)tiles, 512, 0, s>>>(a);
  return (int)hipGetLastError();
}

int launch_rows_q8(int dtype, int epi, const Args& a, hipStream_t s) {
  return dtype == Q3_BF16 ? rows_q8<BF16>(epi, a, s) : rows_q8<F16>(epi, a, s);
}

}  // namespace q3gemm
