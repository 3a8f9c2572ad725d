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
#include <algorithm>

#include "int8.h"

namespace {

constexpr int D = 128, BLK = 64;
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
  int Hkv, G, splits;
  float scale2;  // softmax scale * log2(e)
};

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
Q3_DEV int pack_f16x2(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(int, __builtin_convertvector(v, f16x2_t));
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
  float unit;            // of O
};

// Scores (already S^T) of a block -> P in fp16 operands, with the running maximum, sum and O rescaled.
// RAW_V: the block's values are 16-bit numbers, not codes (the tail): vscale is 1.
template <typename T, int RT, bool MASK>
Q3_DEV void softmax_step(Rows<T, RT>& w, f32x4 (&s)[RT][4], float c, float vscale, int key0, const int (&qpos)[RT],
                         i32x4 (&p)[RT][2]) {
  // units: a value scale within 16 times of the unit leaves it; one far below all others adds nothing worth a new unit
  float ratio = w.unit > 0.f ? vscale / w.unit : 0.f;
  if (vscale > 0.f && (w.unit == 0.f || ratio > 16.f || (ratio < 0.0625f && ratio > 0x1p-60f))) {
    const float unit = __uint_as_float(__float_as_uint(vscale) & 0x7f800000u);  // the power of two below
    const float u = unit > 0.f ? unit : 0x1p-126f;
    const float f = w.unit > 0.f ? w.unit / u : 0.f;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < 8; ++t) w.o[r][t] *= f;
    w.unit = u;
    ratio = vscale / u;
  } else if (vscale != vscale) {
    ratio = vscale;
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float mx = w.m[r];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[r][t][e] *= c;
        if (MASK && key0 + 4 * t + e > qpos[r]) s[r][t][e] = -INFINITY;
        mx = fmaxf(mx, s[r][t][e]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float alpha = __builtin_amdgcn_exp2f(w.m[r] - mx);
    w.m[r] = mx;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __builtin_amdgcn_exp2f(s[r][t][e] - mx);
        sum += x;
        s[r][t][e] = MASK && key0 + 4 * t + e > qpos[r] ? 0.f : x * ratio;
      }
      p[r][t >> 1][2 * (t & 1)] = pack_f16x2(s[r][t][0], s[r][t][1]);
      p[r][t >> 1][2 * (t & 1) + 1] = pack_f16x2(s[r][t][2], s[r][t][3]);
    }
    w.l[r] = w.l[r] * alpha + sum;
#pragma unroll
    for (int t = 0; t < 8; ++t) w.o[r][t] *= alpha;
  }
}

// WK waves share the rows and split the blocks (joined through LDS), 4 / WK groups of waves have rows of their own.
template <typename T, int RT, int WK> __global__ __launch_bounds__(256) void kv8_attn_kernel(AttnArgs a) {
  constexpr int WR = 4 / WK, ROWS = 16 * RT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int wk = wave % WK, wr = wave / WK;
  const int b = blockIdx.z / a.Hkv, hk = blockIdx.z % a.Hkv, split = blockIdx.x;
  const int64_t start = a.start_dev ? *a.start_dev : a.start;
  const int rows = (int)(a.S * a.G), row0 = ((int)blockIdx.y * WR + wr) * ROWS;
  const int64_t total = min(start + a.S, a.capacity), cblocks = (a.capacity + BLK - 1) / BLK;
  const int64_t whole = total / BLK;  // blocks in 8 bits; block `whole` is the tail
  const int64_t bh = (int64_t)b * a.Hkv + hk;
  const int8_t* ck = a.ck + bh * cblocks * (BLK * D);
  const int8_t* cv = a.cv + bh * cblocks * (BLK * D);
  const float* skp = a.sk + bh * cblocks;
  const float* svp = a.sv + bh * cblocks;

  Rows<T, RT> w;
  int qpos[RT];  // relative to start: the last visible key is start + qpos
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int rc = min(row0 + 16 * r + j, rows - 1), s = rc / a.G, h = hk * a.G + (rc - s * a.G);
    qpos[r] = s;
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
  w.unit = 0.f;
  // this wave's blocks: those of the split, every WK-th, as far as its last row sees
  const int64_t last_pos = start + min(row0 + ROWS, rows) / a.G - (min(row0 + ROWS, rows) % a.G ? 0 : 1);
  const int64_t nblk = row0 < rows ? min(last_pos, total - 1) / BLK + 1 : 0;
  const int64_t all = (total + BLK - 1) / BLK, per = (all + a.splits - 1) / a.splits;
  const int64_t b_end = min(nblk, (split + 1) * per), b0 = split * per + wk;
  const int64_t wend = min(b_end, whole);
  const int64_t first_pos = start + min(row0, rows - 1) / a.G;  // blocks before it need no mask

  Raw raw;
  float sk = 0.f, sv = 0.f;
  const int krow = 16 * (j >> 2) + (j & 3);
  auto load_k = [&](int64_t blk) {
    const int8_t* p = ck + blk * (BLK * D) + krow * D + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) raw.k[t][c] = *reinterpret_cast<const i32x4*>(p + t * 4 * D + 64 * c);
    sk = skp[blk];
  };
  auto load_v = [&](int64_t blk) {
    const int8_t* p = cv + blk * (BLK * D) + j * BLK + 16 * g;
#pragma unroll
    for (int t = 0; t < 8; ++t) raw.v[t] = *reinterpret_cast<const i32x4*>(p + t * 16 * BLK);
    sv = svp[blk];
  };
  int64_t blk = b0;
  if (blk < wend) {
    load_k(blk);
    load_v(blk);
  }
  for (; blk < wend; blk += WK) {
    f32x4 s[RT][4];
    const float c = sk * a.scale2;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      bf16x8_t kf[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) kf[h][e] = codes16<T>(raw.k[t][h][2 * e], raw.k[t][h][2 * e + 1]);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        s[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[r][t] = mfma_16x16x32<T>(kf[h][e], w.q[r][h][e], s[r][t]);
      }
    }
    const float vs = sv;
    if (blk + WK < wend) load_k(blk + WK);
    i32x4 p[RT][2];
    if ((blk + 1) * BLK > first_pos + 1) {
      softmax_step<T, RT, true>(w, s, c, vs, (int)(blk * BLK - start) + 16 * g, qpos, p);
    } else {
      softmax_step<T, RT, false>(w, s, c, vs, 0, qpos, p);
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const bf16x8_t v0 = codes16<F16>(raw.v[t][0], raw.v[t][1]), v1 = codes16<F16>(raw.v[t][2], raw.v[t][3]);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        w.o[r][t] = mfma_16x16x32<F16>(v0, __builtin_bit_cast(bf16x8_t, p[r][0]), w.o[r][t]);
        w.o[r][t] = mfma_16x16x32<F16>(v1, __builtin_bit_cast(bf16x8_t, p[r][1]), w.o[r][t]);
      }
    }
    if (blk + WK < wend) load_v(blk + WK);
  }
  // the tail, in 16 bits: P is rounded to T here, as V is what it multiplies; slots past the last position hold anything
  if (blk == whole && blk < b_end) {
    const u16* tk = a.tk + bh * (BLK * D);
    const u16* tv = a.tv + bh * (BLK * D);
    const int left = (int)(total - whole * BLK);  // valid slots
    f32x4 s[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const u16* p = tk + (krow + 4 * t) * D + 16 * g;
      bf16x8_t kf[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) kf[h][e] = *reinterpret_cast<const bf16x8_t*>(p + 64 * h + 8 * e);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        s[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[r][t] = mfma_16x16x32<T>(kf[h][e], w.q[r][h][e], s[r][t]);
      }
    }
    const int key0 = (int)(whole * BLK - start) + 16 * g;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float mx = w.m[r];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[r][t][e] = key0 + 4 * t + e > qpos[r] ? -INFINITY : s[r][t][e] * a.scale2;
          mx = fmaxf(mx, s[r][t][e]);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float alpha = __builtin_amdgcn_exp2f(w.m[r] - mx);
      w.m[r] = mx;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[r][t][e] = __builtin_amdgcn_exp2f(s[r][t][e] - mx);
          sum += s[r][t][e];
        }
      w.l[r] = w.l[r] * alpha + sum;
      const float f = alpha * w.unit;  // O back to plain units: the tail's values are what they are
#pragma unroll
      for (int t = 0; t < 8; ++t) w.o[r][t] *= f;
    }
    w.unit = 1.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8_t p[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        i32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = (int)pack2<T>(s[r][2 * h + (e >> 1)][2 * (e & 1)], s[r][2 * h + (e >> 1)][2 * (e & 1) + 1]);
        p[r] = __builtin_bit_cast(bf16x8_t, x);
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        i32x4 v = *reinterpret_cast<const i32x4*>(tv + (16 * t + j) * BLK + 16 * g + 8 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int slot = 16 * g + 8 * h + 2 * e;
          if (slot >= left) v[e] = 0;
          else if (slot + 1 >= left) v[e] &= 0xffff;
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) w.o[r][t] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, v), p[r], w.o[r][t]);
      }
    }
  }
  // row sums over the lane groups, O in plain units
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    w.l[r] += __shfl_xor(w.l[r], 16, 64);
    w.l[r] += __shfl_xor(w.l[r], 32, 64);
#pragma unroll
    for (int t = 0; t < 8; ++t) w.o[r][t] *= w.unit;
  }
  // the waves of one set of rows joined in halves, in a fixed order
  if constexpr (WK > 1) {
    __shared__ f32x4 jo[WK / 2][RT][8][64];
    __shared__ float jm[WK / 2][RT][64], jl[WK / 2][RT][64];
#pragma unroll
    for (int half = WK / 2; half >= 1; half >>= 1) {
      if (wk >= half && wk < 2 * half) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          jm[wk - half][r][lane] = w.m[r];
          jl[wk - half][r][lane] = w.l[r];
#pragma unroll
          for (int t = 0; t < 8; ++t) jo[wk - half][r][t][lane] = w.o[r][t];
        }
      }
      __syncthreads();
      if (wk < half) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float m2 = jm[wk][r][lane], m = fmaxf(w.m[r], m2);
          const float f1 = __builtin_amdgcn_exp2f(w.m[r] - m), f2 = __builtin_amdgcn_exp2f(m2 - m);
          w.l[r] = w.l[r] * f1 + jl[wk][r][lane] * f2;
          w.m[r] = m;
#pragma unroll
          for (int t = 0; t < 8; ++t) w.o[r][t] = w.o[r][t] * f1 + jo[wk][r][t][lane] * f2;
        }
      }
      __syncthreads();
    }
    if (wk != 0) return;
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = row0 + 16 * r + j;
    if (row >= rows) continue;
    if (a.splits == 1) {
      const int64_t s = row / a.G, h = hk * a.G + (row - s * a.G);
      u16* op = a.o + b * a.ob + s * a.os + h * a.oh + 4 * g;
      const float inv = 1.f / w.l[r];
#pragma unroll
      for (int t = 0; t < 8; ++t)
        *reinterpret_cast<i32x2*>(op + 16 * t) = i32x2{(int)pack2<T>(w.o[r][t][0] * inv, w.o[r][t][1] * inv),
                                                       (int)pack2<T>(w.o[r][t][2] * inv, w.o[r][t][3] * inv)};
    } else {
      const int64_t pr = (bh * rows + row) * a.splits + split;
      if (g == 0) {
        a.pm[pr] = w.m[r];
        a.pl[pr] = w.l[r];
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) *reinterpret_cast<f32x4*>(a.po + pr * D + 16 * t + 4 * g) = w.o[r][t];
    }
  }
}

// out = sum_j 2^(m_j - M) o_j / sum_j 2^(m_j - M) l_j over a row's splits, in fixed order: a wave per row, 2 dims a lane.
template <typename T> __global__ __launch_bounds__(256) void kv8_merge_kernel(AttnArgs a) {
  const int64_t rows = a.S * a.G, i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t bh = blockIdx.y;
  if (i >= rows) return;
  const int64_t p0 = (bh * rows + i) * a.splits;
  float mx = kLow;
  for (int k = lane; k < a.splits; k += 64) mx = fmaxf(mx, a.pm[p0 + k]);
  mx = group_max<64>(mx);
  float l = 0.f, x = 0.f, y = 0.f;
  for (int k0 = 0; k0 < a.splits; k0 += 64) {
    const int n = min(64, a.splits - k0);
    const float wgt = lane < n ? __builtin_amdgcn_exp2f(a.pm[p0 + k0 + lane] - mx) : 0.f;
    l += lane < n ? wgt * a.pl[p0 + k0 + lane] : 0.f;
    for (int k = 0; k < n; ++k) {
      const float f = __shfl(wgt, k, 64);
      const float* o = a.po + (p0 + k0 + k) * D + 2 * lane;
      x += f * o[0];
      y += f * o[1];
    }
  }
  l = group_sum<64>(l);
  const int64_t s = i / a.G, h = (bh % a.Hkv) * a.G + (i - s * a.G);
  *reinterpret_cast<uint32_t*>(a.o + (bh / a.Hkv) * a.ob + s * a.os + h * a.oh + 2 * lane) = pack2<T>(x / l, y / l);
}

struct Plan {
  int wk, splits;
  int64_t row_blocks;
};

// Rows of one key/value head and the positions that a launch may span -> tiling.
Plan plan_for(int64_t B, int64_t Hkv, int64_t rows, int64_t span) {
  Plan p;
  p.wk = rows <= 16 ? 4 : 1;
  const int64_t per_wg = 16 * (4 / p.wk);
  p.row_blocks = (rows + per_wg - 1) / per_wg;
  const int64_t blocks = (span + BLK - 1) / BLK, groups = B * Hkv * p.row_blocks;
  // enough workgroups for two on every CU, but a block for each wave at least
  int64_t s = std::max<int64_t>(1, 512 / groups);
  s = std::min<int64_t>(s, (blocks + p.wk - 1) / p.wk);
  p.splits = (int)std::min<int64_t>(s, 1024);
  return p;
}

template <typename T> int launch(const Plan& p, const AttnArgs& a, dim3 g, hipStream_t s) {
  if (p.wk == 4) kv8_attn_kernel<T, 1, 4><<<g, 256, 0, s>>>(a);
  else kv8_attn_kernel<T, 1, 1><<<g, 256, 0, s>>>(a);
  if (p.splits > 1) {
    const dim3 mg((unsigned)((a.S * a.G + 3) / 4), g.z);
    kv8_merge_kernel<T><<<mg, 256, 0, s>>>(a);
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
  const int64_t rows = S * (Hq / Hkv);
  const Plan p = plan_for(B, Hkv, rows, start_dev ? capacity : start + S);
  Q3_REQUIRE(rows < (1ll << 31) - 128 && p.row_blocks < 65536);
  const int64_t parts = B * Hkv * rows * p.splits;
  if (p.splits > 1) Q3_REQUIRE(al16(workspace) && workspace_bytes >= (size_t)parts * (D + 2) * sizeof(float));
  float* ws = (float*)workspace;
  const AttnArgs a{(const u16*)q, qsb, qss, qsh, cache_k, cache_v, scale_k, scale_v, (const u16*)tail_k,
                   (const u16*)tail_v, (u16*)out, osb, oss, osh, ws, ws + parts * D, ws + parts * (D + 1), S, start,
                   capacity, start_dev, (int)Hkv, (int)(Hq / Hkv), p.splits, scale * 1.4426950408889634f};
  const dim3 g((unsigned)p.splits, (unsigned)p.row_blocks, (unsigned)(B * Hkv));
  return dtype == Q3_BF16 ? launch<BF16>(p, a, g, stream) : launch<F16>(p, a, g, stream);
}

}  // extern "C"
