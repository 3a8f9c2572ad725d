// Causal grouped-query attention of rows that continue shared prefixes: B rows in R groups of n = B / R; row b sees all P
// positions of prefix b / n (keys and values held once per group) and its own positions 0 .. start_b + s.  Head dim 128.
//
// A query row is one (row b, position s, head j of the G that share a key/value head).  The rows of all n continuations are one
// operand of the prefix's products, so a prefix is read once per 32 NW query rows, not once per continuation:
//   S^T = K Q^T and O^T += V^T P on v_mfma_f32_16x16x32, a wave holding 32 query rows (a lane two of them: its 16-row tiles'
//   rows lane % 16), 64 keys at a time.  The K row that feeds matrix row r is chosen so that P is the second product's operand
//   as it comes out of the exponentials; V^T comes from transpose reads of V's rows in LDS.  The running maximum moves only
//   when a score passes it by more than a factor 2^8; row sums are of the rounded P, by a product with ones.
// K and V go to LDS in direct loads, one 64-key block ahead.
//
// Work is cut into jobs (row tile, key/value head, range of 64-key blocks).  Few queries: jobs over ranges of the prefix with
// the rows of all continuations, and jobs over ranges of one row's own positions, each leaving unnormalised O, maximum and sum,
// which a second launch joins in a fixed order.  Many queries (enough row tiles of one row b to fill the chip): a job goes through
// the prefix and then its row's own positions, and writes the result.
#include <algorithm>

#include "common.h"

namespace {

constexpr int D = 128, BLK = 64;
constexpr float kLog2e = 1.4426950408889634f;
typedef __attribute__((address_space(3))) void* lds_vp;

struct Strides {
  int64_t b, h, s;  // elements between batch entries, heads, positions
};

struct Args {
  const u16* q;
  Strides ql;
  const u16 *pk, *pv;
  Strides pl;  // prefix, by group
  const u16 *ck, *cv;
  Strides cl;  // own positions, by row
  u16* o;
  Strides ol;
  float *po, *pm, *ps;  // partials [row (b, s, head)][slot]: O [128], maximum (base-2 score units), sum
  int R, n, Hkv, G, S, P, C;
  int64_t start;
  const int64_t* start_dev;
  int start_step;  // 0: one start for all rows
  float scale2;    // scale * log2(e)
  // plan
  int fused, pjobs, ptiles, psplits, pper, stiles, ssplits, max_splits, min_per, slots;
};

Q3_DEV float xmax4(float x) {  // over lanes {l, l ^ 16, l ^ 32, l ^ 48}
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}

// One wave load of 16 bytes a lane into LDS, zeros from `bytes` on.
Q3_DEV void buffer_to_lds(const u16* p, int bytes, uint32_t off, char* dst) {
  const auto d = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (lds_vp)dst, 16, off, 0, 0, 0);
}

// Own positions that row b's queries reach in all: start + S, within the capacity, and 0 for a negative end.
Q3_DEV int row_start(const Args& a, int b) {
  const int64_t s = a.start_dev ? a.start_dev[(int64_t)b * a.start_step] : a.start;
  return (int)min(max(s, (int64_t)-a.S), (int64_t)a.C);
}
Q3_DEV int own_end(const Args& a, int start, int s) { return min(max(start + s + 1, 0), a.C); }
// Blocks of own positions per split: from the number of positions alone, so that a captured step and an eager call of the same
// length form the same sums.
Q3_DEV int own_per(const Args& a, int blocks) { return max((blocks + a.max_splits - 1) / a.max_splits, a.min_per); }

// LDS: K rows of 256 bytes, 16-byte chunk c of row r at c ^ kswz(r); V in 16 slots of 4 rows (keys s, s + 16, s + 32, s + 48)
// at a pitch of 1056 bytes, which spreads a transpose read over all banks.
Q3_DEV int kswz(int r) { return (r & 7) | (((r >> 4) & 1) << 3); }
constexpr int kSlot = 1056, kKTile = BLK * D * 2, kVTile = 16 * kSlot, kStage = kKTile + kVTile;

// Whether both 16-bit halves are finite numbers of type T.
template <typename T> Q3_DEV bool finite2(uint32_t x) {
  constexpr uint32_t E = T::code == Q3_F16 ? 0x7c00u : 0x7f80u;
  return (x & E) != E && ((x >> 16) & E) != E;
}
template <typename T> Q3_DEV uint32_t only_finite2(uint32_t x) {
  constexpr uint32_t E = T::code == Q3_F16 ? 0x7c00u : 0x7f80u;
  return ((x & E) == E ? 0u : x & 0xffffu) | (((x >> 16) & E) == E ? 0u : x & 0xffff0000u);
}

template <typename T, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefix_attn_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];
  constexpr int RT = 32 * NW;  // query rows of a job
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int SG = a.S * a.G;

  // ---- the job
  int b0, hk, tile, slot = 0;       // first row b of the job's rows
  int rows;                         // query rows from b0's first on
  int pb = 0, pe = 0, sb = 0, se = 0;  // 64-key blocks of the prefix and of b0's own positions
  int own = 0, start = 0;           // own positions that the tile's last row sees
  const int pblocks = (a.P + BLK - 1) / BLK;
  if ((int)blockIdx.x < a.pjobs) {
    // each XCD (workgroup ids congruent mod 8) takes a contiguous range of jobs, row tiles innermost: the tiles that read the
    // same keys share an L2
    const int xcd = blockIdx.x & 7, per = a.pjobs >> 3, rem = a.pjobs & 7;
    int w = xcd * per + min(xcd, rem) + ((int)blockIdx.x >> 3);
    tile = w % a.ptiles;
    w /= a.ptiles;
    slot = w % a.psplits;
    w /= a.psplits;
    hk = w % a.Hkv;
    b0 = w / a.Hkv * a.n;
    rows = a.n * SG;
    pb = slot * a.pper;
    pe = min(pb + a.pper, pblocks);
  } else {
    int w = (int)blockIdx.x - a.pjobs;
    tile = w % a.stiles;
    w /= a.stiles;
    hk = w % a.Hkv;
    w /= a.Hkv;
    const int split = w % a.ssplits;
    b0 = w / a.ssplits;
    rows = SG;
    start = __builtin_amdgcn_readfirstlane(row_start(a, b0));
    const int all = (own_end(a, start, a.S - 1) + BLK - 1) / BLK;
    own = own_end(a, start, min(tile * RT + RT - 1, rows - 1) / a.G);
    const int blocks = (own + BLK - 1) / BLK;
    if (a.fused) {
      pe = pblocks;
      se = blocks;
    } else {
      const int per = own_per(a, all);
      sb = split * per;
      if (split > 0 && sb >= all) return;  // no such split: the joining launch knows
      se = min(sb + per, blocks);
      sb = min(sb, se);
      slot = a.psplits + split;
    }
  }
  const int npre = pe - pb, nblk = npre + (se - sb);
  const u16* pk = a.pk + b0 / a.n * a.pl.b + hk * a.pl.h;
  const u16* pv = a.pv + b0 / a.n * a.pl.b + hk * a.pl.h;
  const u16* ck = a.ck + b0 * a.cl.b + hk * a.cl.h;
  const u16* cv = a.cv + b0 * a.cl.b + hk * a.cl.h;

  // ---- this lane's query rows
  const int m0 = tile * RT + wave * 32;
  const bool work = m0 < rows;  // a wave without rows only loads
  int lim[2];                   // own positions that the row sees
  int64_t orow[2], ooff[2];     // its place among the partials, and in the output
  bf16x8_t qf[2][4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int m = min(m0 + 16 * u + r16, rows - 1), b = b0 + m / SG, x = m % SG, s = x / a.G, h = hk * a.G + x % a.G;
    lim[u] = own_end(a, start, s);
    const u16* qp = a.q + b * a.ql.b + h * a.ql.h + s * a.ql.s;
    ooff[u] = b * a.ol.b + h * a.ol.h + s * a.ol.s;
    orow[u] = ((int64_t)b * a.S + s) * (a.Hkv * a.G) + h;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
      qf[u][ks] = *reinterpret_cast<const bf16x8_t*>(qp + 32 * ks + 8 * g);
  }
  // the first own position that some row of the wave does not see
  const int lim_w = own_end(a, start, min(m0, rows - 1) / a.G);

  // ---- global -> LDS
  uint32_t krow[16 / NW], kchk[16 / NW], vrow[16 / NW];
#pragma unroll
  for (int i = 0; i < 16 / NW; ++i) {
    const int w = wave + NW * i, r = 4 * w + g;
    krow[i] = (uint32_t)r;
    kchk[i] = (uint32_t)((r16 ^ kswz(r)) * 16);
    vrow[i] = (uint32_t)(w + 16 * g);
  }
  auto issue = [&](int j) {
    if (j >= nblk) return;
    const bool pre = j < npre;
    const int key0 = (pre ? pb + j : sb + j - npre) * BLK, count = (pre ? a.P : own) - key0;
    const int64_t st = pre ? a.pl.s : a.cl.s;
    const int bytes = (min(count, BLK) - 1) * (int)st * 2 + 2 * D;
    const u16 *kp = (pre ? pk : ck) + key0 * st, *vp = (pre ? pv : cv) + key0 * st;
    char* base = lds + (j & 1) * kStage;
#pragma unroll
    for (int i = 0; i < 16 / NW; ++i)
      buffer_to_lds(kp, bytes, krow[i] * (uint32_t)(st * 2) + kchk[i], base + (wave + NW * i) * 1024);
#pragma unroll
    for (int i = 0; i < 16 / NW; ++i)
      buffer_to_lds(vp, bytes, vrow[i] * (uint32_t)(st * 2) + r16 * 16, base + kKTile + (wave + NW * i) * kSlot);
  };

  // ---- LDS -> fragments.  Matrix row r16 of key tile kt reads K row 32 (kt / 2) + 8 (kt % 2) + krow0; element i of that tile in
  // lane group g is then key 32 (kt / 2) + 8 (kt % 2) + kbase + i.
  const int krow0 = 4 * ((r16 >> 2) & 1) + 16 * (r16 >> 3) + (r16 & 3);
  const int kbase = 4 * (g & 1) + 16 * (g >> 1);
  int koff[4], voff[2];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) koff[ks] = krow0 * 256 + (((4 * ks + g) ^ r16) << 4);
#pragma unroll
  for (int kc = 0; kc < 2; ++kc) voff[kc] = (4 * (g & 1) + (r16 >> 2)) * kSlot + (g >> 1) * 256 + 8 * (r16 & 3) + kc * 512;
  constexpr int ktoff[4] = {0, 8 * 256, 32 * 256, 40 * 256};

  f32x4 oacc[8][2], lsum[2];
  float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    lsum[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) oacc[dt][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t one2 = pack2<T>(1.f, 1.f);
  const i32x4 ones = i32x4{(int)one2, (int)one2, (int)one2, (int)one2};
  const float thr = 8.f / a.scale2;

  issue(0);
  for (int j = 0; j < nblk; ++j) {
    __builtin_amdgcn_s_waitcnt((0 & 15) | (7 << 4) | (0 << 8));  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();  // block j is there, and every wave is done with block j - 1
    asm volatile("" ::: "memory");
    issue(j + 1);
    if (!work) continue;
    const char* kb = lds + (j & 1) * kStage;
    const char* vb = kb + kKTile;
    const bool pre = j < npre;
    const int key0 = (pre ? pb + j : sb + j - npre) * BLK;
    f32x4 S[4][2];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(kb + koff[ks] + ktoff[kt]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          S[kt][u] = mfma_16x16x32<T>(kf, qf[u][ks], ks == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : S[kt][u]);
      }
    const bool mask = key0 + BLK > (pre ? a.P : lim_w);
    if (mask) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int rel = (pre ? a.P : lim[u]) - key0 - kbase;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) S[kt][u][i] = 32 * (kt >> 1) + 8 * (kt & 1) + i < rel ? S[kt][u][i] : -INFINITY;
      }
    }
    // ---- online softmax
    bool need[2];
    float alpha[2], ms[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float x = S[0][u][0];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) x = __builtin_fmaxf(x, S[kt][u][i]);
      x = xmax4(x);
      need[u] = x > m[u] + thr || m[u] == -INFINITY;
      const float mn = need[u] ? x : m[u];
      alpha[u] = m[u] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[u] - mn) * a.scale2);
      m[u] = mn;
      ms[u] = mn == -INFINITY ? 0.f : mn * a.scale2;
    }
    if (__any(need[0] || need[1])) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        lsum[u] *= alpha[u];
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) oacc[dt][u] *= alpha[u];
      }
    }
    i32x4 P[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          S[kt][u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kt][u][i], a.scale2, -ms[u]));
        P[u][kt >> 1][2 * (kt & 1)] = (int)pack2<T>(S[kt][u][0], S[kt][u][1]);
        P[u][kt >> 1][2 * (kt & 1) + 1] = (int)pack2<T>(S[kt][u][2], S[kt][u][3]);
      }
    // ---- O^T += V^T P.  A value that is not finite would spoil the rows that do not see its position too (0 times it is NaN):
    // blocks that some row sees in part are looked through first, and then such values are kept out of the product and added
    // to the rows that do see them.
    bool clean = true;
    if (mask && !pre && a.S > 1) {
      uint32_t ok = 1;
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const i32x4 x = *reinterpret_cast<const i32x4*>(vb + i * kSlot + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) ok &= finite2<T>((uint32_t)x[e]) ? 1u : 0u;
      }
      clean = !__any(ok == 0);
    }
    if (clean) {
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
          const i32x4 v = lds_frag_tr(vb + voff[kc] + dt * 32, 8 * kSlot);
#pragma unroll
          for (int u = 0; u < 2; ++u)
            oacc[dt][u] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, P[u][kc]), oacc[dt][u]);
        }
    } else {
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
          i32x4 v = lds_frag_tr(vb + voff[kc] + dt * 32, 8 * kSlot);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (int)only_finite2<T>((uint32_t)v[e]);
#pragma unroll
          for (int u = 0; u < 2; ++u)
            oacc[dt][u] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, P[u][kc]), oacc[dt][u]);
        }
      for (int key = 0; key < BLK; ++key) {
        const char* row = vb + (key & 15) * kSlot + (key >> 4) * 256 + 8 * g;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
          const i32x2 x = *reinterpret_cast<const i32x2*>(row + dt * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bits = ((uint32_t)x[i >> 1] >> (16 * (i & 1))) & 0xffffu;
            if (finite2<T>(bits)) continue;
#pragma unroll
            for (int u = 0; u < 2; ++u)
              if (key0 + key < lim[u]) oacc[dt][u][i] += to_f32<T>((u16)bits);
          }
        }
      }
    }
#pragma unroll
    for (int kc = 0; kc < 2; ++kc)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        lsum[u] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, ones), __builtin_bit_cast(bf16x8_t, P[u][kc]), lsum[u]);
  }

  // ---- out: lane holds O[row 16 u + r16][16 dt + 4 g + i]
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (m0 + 16 * u + r16 >= rows) continue;
    if (a.slots == 1) {
      const float inv = a.P == 0 && lim[u] == 0 ? 0.f : 1.f / lsum[u][0];  // no position to see: zeros
      u16* out = a.o + ooff[u];
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
        *reinterpret_cast<i32x2*>(out + 16 * dt + 4 * g) =
            i32x2{(int)pack2<T>(oacc[dt][u][0] * inv, oacc[dt][u][1] * inv),
                  (int)pack2<T>(oacc[dt][u][2] * inv, oacc[dt][u][3] * inv)};
    } else {
      const int64_t at = orow[u] * a.slots + slot;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(a.po + at * D + 16 * dt + 4 * g) = oacc[dt][u];
      if (g == 0) {
        a.pm[at] = m[u] == -INFINITY ? -INFINITY : m[u] * a.scale2;
        a.ps[at] = lsum[u][0];
      }
    }
  }
}

// o = sum_j 2^(m_j - M) O_j / sum_j 2^(m_j - M) s_j over a query row's slots, in slot order: the prefix's splits, then those of
// its own positions.  32 lanes a row, 4 dims each.
template <typename T> __global__ __launch_bounds__(256) void prefix_join_kernel(Args a, int64_t rows) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int l = threadIdx.x & 31, Hq = a.Hkv * a.G;
  const int64_t bs = row / Hq;
  const int h = (int)(row - bs * Hq), b = (int)(bs / a.S), s = (int)(bs - (int64_t)b * a.S);
  const int start = row_start(a, b), all = (own_end(a, start, a.S - 1) + BLK - 1) / BLK;
  const int per = own_per(a, all);
  const int used = a.psplits + max((all + per - 1) / per, 1);
  const float *pm = a.pm + row * a.slots, *ps = a.ps + row * a.slots, *po = a.po + row * a.slots * D + 4 * l;
  float M = -INFINITY;
  for (int j = 0; j < used; ++j) M = __builtin_fmaxf(M, pm[j]);
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < used; ++j) {
    const float w = pm[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(pm[j] - M);
    sum = __builtin_fmaf(w, ps[j], sum);
    o += w * *reinterpret_cast<const f32x4*>(po + (int64_t)j * D);
  }
  const float inv = a.P == 0 && own_end(a, start, s) == 0 ? 0.f : 1.f / sum;
  u16* out = a.o + b * a.ol.b + s * a.ol.s + h * a.ol.h + 4 * l;
  *reinterpret_cast<i32x2*>(out) = i32x2{(int)pack2<T>(o[0] * inv, o[1] * inv), (int)pack2<T>(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------- host
int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }
bool al(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }
bool lay_ok(const void* p, const Strides& l) { return p && al(p, 16) && l.b % 8 == 0 && l.h % 8 == 0 && l.s % 8 == 0; }

constexpr int kMinPer = 4;  // own blocks of a split at least

// The jobs of a call; span: own positions that the launch has to cover.
struct Plan {
  int nw, fused, ptiles, psplits, pper, stiles, ssplits, max_splits, slots;
  int64_t pjobs, sjobs;
};
Plan plan_for(int64_t R, int64_t n, int64_t S, int64_t Hkv, int64_t G, int64_t P, int64_t span) {
  Plan p{};
  const int64_t B = R * n, SG = S * G, pblocks = cdiv(P, BLK);
  auto waves = [](int64_t rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8; };
  // one pass over everything where a row's own queries fill tiles and the tiles fill the chip
  if (SG >= 128 && B * Hkv * cdiv(SG, 256) >= 192) {
    p.nw = 8;
    p.fused = 1;
    p.stiles = (int)cdiv(SG, 256);
    p.ssplits = p.max_splits = p.slots = 1;
    p.sjobs = B * Hkv * p.stiles;
    return p;
  }
  p.nw = waves(P > 0 ? n * SG : SG);
  const int64_t rt = 32 * p.nw, target = p.nw == 8 ? 256 : 512;
  if (P > 0) {
    p.ptiles = (int)cdiv(n * SG, rt);
    const int64_t want = std::max<int64_t>(1, target / (R * Hkv * p.ptiles));
    p.pper = (int)std::max<int64_t>(cdiv(pblocks, want), 2);
    p.psplits = (int)cdiv(pblocks, p.pper);
    p.pjobs = R * Hkv * p.ptiles * p.psplits;
  }
  p.stiles = (int)cdiv(SG, rt);
  p.max_splits = (int)std::max<int64_t>(1, target / (B * Hkv * p.stiles));
  p.ssplits = (int)std::max<int64_t>(1, std::min<int64_t>(p.max_splits, cdiv(cdiv(span, BLK), kMinPer)));
  p.sjobs = B * Hkv * p.stiles * p.ssplits;
  p.slots = p.psplits + p.ssplits;
  return p;
}
bool sizes_ok(int64_t B, int64_t R, int64_t S, int64_t Hq, int64_t Hkv, int64_t P, int64_t C) {
  return B > 0 && R > 0 && B % R == 0 && S > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && P >= 0 && C > 0 && P < (1 << 30) &&
         C < (1 << 30) && S < (1 << 30) && B < (1 << 24) && Hq < (1 << 16) && B * S * Hq < (1ll << 31) &&
         S <= C;
}
size_t bytes_for(const Plan& p, int64_t rows) {
  return p.slots == 1 ? 0 : (size_t)rows * p.slots * (D + 2) * sizeof(float);
}

template <typename T> int run(const Plan& p, const Args& a, int64_t rows, hipStream_t s) {
  const unsigned grid = (unsigned)(p.pjobs + p.sjobs);
  switch (p.nw) {
    case 1: prefix_attn_kernel<T, 1><<<grid, 64, 0, s>>>(a); break;
    case 2: prefix_attn_kernel<T, 2><<<grid, 128, 0, s>>>(a); break;
    case 4: prefix_attn_kernel<T, 4><<<grid, 256, 0, s>>>(a); break;
    default: prefix_attn_kernel<T, 8><<<grid, 512, 0, s>>>(a); break;
  }
  const int rc = (int)hipGetLastError();
  if (rc != 0 || p.slots == 1) return rc;
  prefix_join_kernel<T><<<(unsigned)cdiv(rows, 8), 256, 0, s>>>(a, rows);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t q3_prefix_attention_workspace_bytes(int64_t B, int64_t R, int64_t S, int64_t Hq, int64_t Hkv, int64_t P, int64_t span) {
  if (!sizes_ok(B, R, S, Hq, Hkv, P, std::max<int64_t>(span, S)) || span < 0) return 0;
  return bytes_for(plan_for(R, B / R, S, Hkv, Hq / Hkv, P, span), B * S * Hq);
}

int q3_prefix_attention(int dtype, const void* q, int64_t qsb, int64_t qss, int64_t qsh, const void* prefix_k, const void* prefix_v,
                        int64_t psb, int64_t psh, int64_t pss, const void* cache_k, const void* cache_v, int64_t csb, int64_t csh,
                        int64_t css, void* out, int64_t osb, int64_t oss, int64_t osh, void* workspace, size_t workspace_bytes,
                        int64_t B, int64_t R, int64_t S, int64_t Hq, int64_t Hkv, int64_t d, int64_t P, int64_t C, int64_t start,
                        const int64_t* start_dev, int64_t starts, float scale, hipStream_t stream) {
  Q3_REQUIRE((dtype == Q3_BF16 || dtype == Q3_F16) && d == D && sizes_ok(B, R, S, Hq, Hkv, P, C) && scale > 0.f && scale < 1e30f);
  const Strides ql{qsb, qsh, qss}, pl{psb, psh, pss}, cl{csb, csh, css}, ol{osb, osh, oss};
  Q3_REQUIRE(lay_ok(q, ql) && lay_ok(cache_k, cl) && lay_ok(cache_v, cl) && css >= D && css < (1 << 24));
  Q3_REQUIRE(P == 0 || (lay_ok(prefix_k, pl) && lay_ok(prefix_v, pl) && pss >= D && pss < (1 << 24)));
  Q3_REQUIRE(out && al(out, 8) && osb % 4 == 0 && oss % 4 == 0 && osh % 4 == 0);
  Q3_REQUIRE(start_dev ? (starts == 1 || starts == B) : (start >= 0 && start + S <= C));
  const int64_t n = B / R, span = start_dev ? C : start + S, rows = B * S * Hq;
  const Plan p = plan_for(R, n, S, Hkv, Hq / Hkv, P, span);
  const size_t need = bytes_for(p, rows);
  Q3_REQUIRE(p.pjobs + p.sjobs < (1ll << 31) && (need == 0 || (workspace && al(workspace, 16) && workspace_bytes >= need)));
  Args a{};
  a.q = (const u16*)q;
  a.ql = ql;
  a.pk = (const u16*)prefix_k;
  a.pv = (const u16*)prefix_v;
  a.pl = pl;
  a.ck = (const u16*)cache_k;
  a.cv = (const u16*)cache_v;
  a.cl = cl;
  a.o = (u16*)out;
  a.ol = ol;
  a.po = (float*)workspace;
  a.pm = a.po ? a.po + (size_t)rows * p.slots * D : nullptr;
  a.ps = a.po ? a.pm + (size_t)rows * p.slots : nullptr;
  a.R = (int)R;
  a.n = (int)n;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.S = (int)S;
  a.P = (int)P;
  a.C = (int)C;
  a.start = start;
  a.start_dev = start_dev;
  a.start_step = start_dev && starts == B && B > 1 ? 1 : 0;
  a.scale2 = scale * kLog2e;
  a.fused = p.fused;
  a.pjobs = (int)p.pjobs;
  a.ptiles = p.ptiles;
  a.psplits = p.psplits;
  a.pper = p.pper;
  a.stiles = p.stiles;
  a.ssplits = p.ssplits;
  a.max_splits = p.max_splits;
  a.min_per = kMinPer;
  a.slots = p.slots;
  return dtype == Q3_BF16 ? run<BF16>(p, a, rows, stream) : run<F16>(p, a, rows, stream);
}

}  // extern "C"
