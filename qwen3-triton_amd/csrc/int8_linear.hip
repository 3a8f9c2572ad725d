// Products of at most 16 rows of 8-bit codes (a decode step) with weights in 8 bits: y = (x W^T) s ws (+ res), and the
// gate/up + SwiGLU form; up to three weights of one input in a launch.
//
// Bound by the weights' bytes.  A tile is 16 output channels, whose rows stream straight into registers as the B operand of
// v_mfma_i32_16x16x64_i8 (lane (r, kq): 16 codes of row r at k = 16 kq of every 64), the token rows as the A operand; a
// workgroup's 8 waves take 256-wide k blocks in turn, P of them in flight, and fold their int32 tiles in LDS: exact, so in any
// order.  A workgroup takes every kResident-th tile, the next one's first blocks in flight while this one is folded; the waves
// end a tile each in turn.  One workgroup per tile took 27.1 us for gate/up at 8 rows (12288 x 4096, twice), this 22.1; linear
// 6144 x 4096 10.5 and 9.8.  P = 4, 4 or 16 waves, non-temporal loads: no faster.
// Measured at one row: 6144 x 4096 8.4 us (3.0 TB/s, half of it start and end), 12288 x 4096 11.5 (4.4 TB/s), 4096 x 12288 12.7.
// Up to 16 rows stream the same weights (16 at 6144 x 4096: 10.8); the tile kernel takes 9.0 us for 17 rows of 4096 x 4096, this
// one 6.1 for one.
#include <algorithm>

#include "gemm_tile.h"
#include "int8.h"

namespace q3gemm {

// What the rows are: their codes (R = 0), or R 16-bit rows that every workgroup turns into codes itself, in LDS, while its
// first weights are on their way: quantize_rows, or with NORM rms_norm.  Each workgroup repeats that work on rows that sit
// in L2; it saves a launch and its wait, and a decode step has one before each of its four products.  One row: 9.2 against
// 12.0 us (6144 x 4096 after a norm), 13.0 against 16.0 (4096 x 12288), 20.6 against 25.1 (gate/up); two rows 9.9, 14.3 and 22.1
// against 12.1, 16.0 and 25.4.  Four rows are level (11.6 against 12.5, 19.5 against 18.4, 29.4 against 27.6; 4096 x 4096 9.7 and
// 10.9), three likewise: it stops at two.
// V: 16-byte pieces of a row per thread.
template <typename T, int EPI, int P, int R, int V, bool NORM>
__global__ __launch_bounds__(512) void gemm_rows_q8_kernel(Args a, RowIn in, int tiles) {
  constexpr int NW = 8, NB = EPI == 3 ? 2 : 1, PAD = 16;  // PAD: the rows of codes start in different banks
  extern __shared__ __attribute__((aligned(16))) int8_t xs[];
  __shared__ i32x4 red[2][NW - 1][NB][64];
  __shared__ uint32_t red_m[NW][R ? R : 1];
  __shared__ float red_s[NW][R ? R : 1], xscale[R ? R : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kq = lane >> 4;
  const int M = (int)a.M, K = (int)a.K * 2;  // codes
  const int nblk = (K + 255) / 256;
  const int8_t* x = reinterpret_cast<const int8_t*>(a.a.p[0]) + (int64_t)min(r, M - 1) * a.a.ld[0] * 2 + 16 * kq;
  // a tile of 16 channels: its piece, first channel and number of channels, and this lane's weight rows and scales
  int s = 0, n0 = 0, ncols = 0;
  const int8_t* w[NB];
  float cs[NB];
  auto at_tile = [&](int t) {
    s = 0;
    if (EPI != 3 && a.axis == 2)
      while (s + 1 < a.pieces && t >= ((int)a.len[s] + 15) / 16) t -= ((int)a.len[s++] + 15) / 16;
    ncols = EPI == 3 ? (int)a.N / 2 : a.axis == 2 ? (int)a.len[s] : (int)a.N;
    n0 = t * 16;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int i = EPI == 3 ? j : s, n = min(n0 + r, ncols - 1);
      w[j] = reinterpret_cast<const int8_t*>(a.b.p[i]) + (int64_t)n * a.b.ld[i] * 2 + 16 * kq;
      cs[j] = a.cscale[i][n];
    }
  };
  int tile = blockIdx.x;
  at_tile(tile);
  // 16-bit rows first in the queue, then the first weights behind them
  [[maybe_unused]] i32x4 rv[R ? R : 1][V], nv[V];
  if constexpr (R > 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = min((v * 512 + tid) * 8, K - 8);
#pragma unroll
      for (int m = 0; m < R; ++m) rv[m][v] = *reinterpret_cast<const i32x4*>(in.x + (int64_t)min(m, M - 1) * in.ldx + at);
      if constexpr (NORM) nv[v] = *reinterpret_cast<const i32x4*>(in.w + at);
    }
  }
  i32x4 wv[P][NB][4], xv[P][4];
  // k block i of this lane's weights (and codes); chunks past the end read the row's last one again, against zeros.  With 16-bit
  // rows there is no branch in it: one here costs the waits of the rows' work their knowledge of what is in flight (14.2
  // against 12.8 us at 4096 x 12288); without, a block that is not there is not loaded.
  const int whole = K / 256;
  auto load = [&](int p, int i) {
    if (R == 0 && i >= nblk) return;
    const bool full = R == 0 && i < whole;
    if (full) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        xv[p][c] = *reinterpret_cast<const i32x4*>(x + i * 256 + 64 * c);
#pragma unroll
        for (int j = 0; j < NB; ++j) wv[p][j][c] = *reinterpret_cast<const i32x4*>(w[j] + i * 256 + 64 * c);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int k = min(i * 256 + 64 * c, K - 16 - 16 * kq);
        if constexpr (R == 0) xv[p][c] = *reinterpret_cast<const i32x4*>(x + k);
#pragma unroll
        for (int j = 0; j < NB; ++j) wv[p][j][c] = *reinterpret_cast<const i32x4*>(w[j] + k);
      }
    }
  };
#pragma unroll
  for (int p = 0; p < P; ++p) load(p, wave + p * NW);
  if constexpr (R > 0) {
    float ss[R];
    uint32_t mb[R];
#pragma unroll
    for (int m = 0; m < R; ++m) {
      ss[m] = 0.f;
      mb[m] = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if ((v * 512 + tid) * 8 >= K) continue;
        if constexpr (NORM) {
          const Vec<T> xf = unpack_vec<T>(rv[m][v]), wf = unpack_vec<T>(nv[v]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            ss[m] += xf.v[e] * xf.v[e];
            mb[m] = max(mb[m], mag_bits(xf.v[e] * wf.v[e]));
          }
        } else {
#pragma unroll
          for (int p = 0; p < 4; ++p) mb[m] = mag_max16(mb[m], (uint32_t)rv[m][v][p]);
        }
      }
      if constexpr (!NORM) mb[m] = mag_bits16<T>(mb[m]);
      mb[m] = wave_umax(mb[m]);
      if constexpr (NORM) ss[m] = group_sum<64>(ss[m]);
    }
    if (lane == 0) {
#pragma unroll
      for (int m = 0; m < R; ++m) {
        red_m[wave][m] = mb[m];
        red_s[wave][m] = ss[m];
      }
    }
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0): the weights stay in flight
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int m = 0; m < R; ++m) {
      uint32_t top = red_m[0][m];
      float sum = red_s[0][m];
#pragma unroll
      for (int i = 1; i < NW; ++i) {
        top = top > red_m[i][m] ? top : red_m[i][m];
        sum += red_s[i][m];
      }
      const bool finite = bits_finite(top);
      const QuantStep st = quant_step(finite ? __uint_as_float(top) : 0.f);
      if (tid == 0) {
        float sc = finite ? st.m / 127.f : __uint_as_float(0x7fc00000u);
        if constexpr (NORM) sc *= rsqrtf(sum * (1.f / (float)K) + in.eps);
        xscale[m] = sc;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if ((v * 512 + tid) * 8 >= K) continue;
        Vec<T> xf = unpack_vec<T>(rv[m][v]);
        if constexpr (NORM) {
          const Vec<T> wf = unpack_vec<T>(nv[v]);
#pragma unroll
          for (int e = 0; e < 8; ++e) xf.v[e] *= wf.v[e];
        }
        *reinterpret_cast<i32x2*>(xs + m * (K + PAD) + (v * 512 + tid) * 8) = finite ? quant_codes(xf.v, st) : i32x2{0, 0};
      }
    }
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  const int8_t* xl = xs + min(r, R ? R - 1 : 0) * (K + PAD) + 16 * kq;
  const int groups = (nblk + P * NW - 1) / (P * NW);
  float rs[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int m = min(4 * kq + e, M - 1);
    rs[e] = R ? xscale[min(m, R ? R - 1 : 0)] : a.rscale[m];
  }
  for (int it = 0;; ++it) {
    i32x4 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = i32x4{0, 0, 0, 0};
    const int next = tile + (int)gridDim.x, n = n0 + r, cols = ncols, piece = s;
    const bool more = next < tiles;
    float sc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) sc[j] = cs[j];
    for (int g = 0; g < groups; ++g) {
      const bool last = g + 1 == groups;
      if (last && more) at_tile(next);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int i = wave + (g * P + p) * NW;
        if (R > 0 || i < nblk) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int k = i * 256 + 64 * c;
            i32x4 xc;
            if constexpr (R > 0) xc = *reinterpret_cast<const i32x4*>(xl + min(k, K - 16 - 16 * kq));
            else xc = xv[p][c];
            if (R > 0 || i == whole) {
#pragma unroll
              for (int e = 0; e < 4; ++e) xc[e] = k + 16 * kq < K ? xc[e] : 0;
            }
#pragma unroll
            for (int j = 0; j < NB; ++j)
              mfma_acc(acc[j], __builtin_bit_cast(bf16x8_t, xc), __builtin_bit_cast(bf16x8_t, wv[p][j][c]));
          }
        }
        if (!last || more) load(p, last ? wave + p * NW : i + P * NW);
      }
    }
    const int own = it & (NW - 1), buf = it & 1;  // the wave that ends this tile
    if (wave != own) {
#pragma unroll
      for (int j = 0; j < NB; ++j) red[buf][wave - (wave > own)][j][lane] = acc[j];
    }
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0): the next weights stay in flight
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (wave == own) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < NW - 1; ++i) acc[j] += red[buf][i][j][lane];
      // lane holds rows 4 kq + e of column n
      if (n < cols) {
        u16* y = reinterpret_cast<u16*>(a.c[EPI == 3 ? 0 : piece]);
        const int64_t ldc = a.ldc[EPI == 3 ? 0 : piece];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int m = 4 * kq + e;
          if (m >= M) continue;
          float v = (float)acc[0][e] * rs[e] * sc[0];
          if constexpr (EPI == 3) v = v * q3_sigmoid(v) * ((float)acc[NB - 1][e] * rs[e] * sc[NB - 1]);
          else if (a.res) v += to_f32<T>(a.res[m * a.ldres + n]);
          y[m * ldc + n] = from_f32<T>(v);
        }
      }
    }
    if (!more) return;
    tile = next;
  }
}

template <typename T, int EPI, int P, int R, int V, bool NORM>
static int launch_rows(const Args& a, const RowIn& in, int64_t tiles, hipStream_t s) {
  constexpr int64_t kResident = EPI == 3 && (R == 0 || V > 1) ? 256 : 512;  // workgroups that the registers let run at a time
  const size_t lds = R ? (size_t)R * (size_t)(2 * a.K + 16) : 0;
  gemm_rows_q8_kernel<T, EPI, P, R, V, NORM><<<(unsigned)std::min(tiles, kResident), 512, lds, s>>>(a, in, (int)tiles);
  return (int)hipGetLastError();
}
// V, P: pieces of a row per thread, and k blocks of a wave in flight, no more than the row has.
template <typename T, int EPI, int R, bool NORM>
static int rows_of(const Args& a, const RowIn& in, int64_t tiles, hipStream_t s) {
  if (a.K <= 1024) return launch_rows<T, EPI, 1, R, 1, NORM>(a, in, tiles, s);
  if (a.K <= 2048) return launch_rows<T, EPI, 2, R, 1, NORM>(a, in, tiles, s);
  return launch_rows<T, EPI, 2, R, 4, NORM>(a, in, tiles, s);
}
template <typename T, int EPI> static int rows_q8(const Args& a, const RowIn& in, int64_t tiles, hipStream_t s) {
  if (!in.x) return launch_rows<T, EPI, 2, 0, 1, false>(a, in, tiles, s);
  if (a.M == 1) return in.w ? rows_of<T, EPI, 1, true>(a, in, tiles, s) : rows_of<T, EPI, 1, false>(a, in, tiles, s);
  return in.w ? rows_of<T, EPI, 2, true>(a, in, tiles, s) : rows_of<T, EPI, 2, false>(a, in, tiles, s);
}

int launch_rows_q8(int dtype, int epi, const Args& a, const RowIn& in, hipStream_t s) {
  int64_t tiles = 0;
  if (epi == 3) tiles = (a.N / 2 + 15) / 16;
  else if (a.axis == 2)
    for (int i = 0; i < a.pieces; ++i) tiles += (a.len[i] + 15) / 16;
  else tiles = (a.N + 15) / 16;
  if (epi == 3) return dtype == Q3_BF16 ? rows_q8<BF16, 3>(a, in, tiles, s) : rows_q8<F16, 3>(a, in, tiles, s);
  return dtype == Q3_BF16 ? rows_q8<BF16, 0>(a, in, tiles, s) : rows_q8<F16, 0>(a, in, tiles, s);
}

}  // namespace q3gemm
