// Causal grouped-query attention of rows that continue shared prefixes: B rows in R groups of n = B / R; row b sees all P
// positions of prefix b / n (keys and values held once per group) and its own positions 0 .. start_b + s.  Head dim 128.
//
// A query row is one (row b, position s, head j of the G that share a key/value head).  The rows of all n continuations are one
// operand of the prefix's products, so a prefix is read once per 128 query rows, not once per continuation:
//   S^T = K Q^T and O^T += V^T P on v_mfma_f32_16x16x32, a wave holding 16 or 32 query rows (a lane one of each 16: its rows
//   lane % 16), 64 keys at a time.  The K row that feeds matrix row r is chosen so that P is the second product's operand
//   as it comes out of the exponentials; V^T comes from transpose reads of V's rows in LDS.  The running maximum moves only
//   when a score passes it by more than a factor 2^8; row sums are of the rounded P, by a product with ones.
//
// Work is cut into jobs (query rows, key/value head, range of 64-key blocks), a workgroup each:
//  * more than 32 query rows (16 of chunks): waves take 32 rows each and share K and V tiles in LDS, loaded a block ahead;
//  * fewer: waves take every fourth block of the range each (K straight into the operand's registers, V into a tile of the
//    wave's own), without waiting for each other, and their sums are joined in LDS.  A decode step's own positions are such jobs:
//    they wait for memory beside the prefix's jobs, which are bound by the matrix cores.
// Jobs leave unnormalised O, maximum and sum, which a second launch joins in a fixed order.  Where the queries of single rows fill
// tiles and the tiles the chip, and where there are few positions in all, a job goes through the prefix and then its row's own
// positions, and writes the result.
#include <algorithm>
#include <type_traits>

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
  int fused, pjobs, sjobs, ptiles, psplits, pper, sfew, stiles, ssplits, max_splits, min_per, slots;
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
Q3_DEV int own_per(const Args& a, int blocks) {
  const int per = max((blocks + a.max_splits - 1) / a.max_splits, a.min_per);
  return a.sfew ? (per + 3) & ~3 : per;  // as many for each wave
}

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

// A lane's offset in a V tile of the fragments of key half kc.
Q3_DEV int value_offset(int g, int r16, int kc) {
  return (4 * (g & 1) + (r16 >> 2)) * kSlot + (g >> 1) * 256 + 8 * (r16 & 3) + kc * 512;
}

// A wave's 16 U query rows: operands, O^T (lane: dims 16 dt + 4 g + i of rows 16 u + r16), maxima and sums.
template <int U> struct Rows {
  bf16x8_t qf[U][4];
  f32x4 o[8][U], l[U];
  float m[U];
  int lim[U];  // own positions that the row sees
};

// Where in a key block an element of S^T stands: matrix row r16 of key tile kt is key tile_key(kt) + row_key(r16), element i of
// that tile in lane group g is key tile_key(kt) + group_key(g) + i.
Q3_DEV constexpr int tile_key(int kt) { return 32 * (kt >> 1) + 8 * (kt & 1); }
Q3_DEV int row_key(int r16) { return 4 * ((r16 >> 2) & 1) + 16 * (r16 >> 3) + (r16 & 3); }
Q3_DEV int group_key(int g) { return 4 * (g & 1) + 16 * (g >> 1); }

// Query rows m0 .. of the job's `rows`, which start at row b0's first; rows past the last are copies of it.
template <int U> Q3_DEV void load_rows(const Args& a, Rows<U>& w, int m0, int rows, int b0, int hk, int start, int g, int r16) {
  const int SG = a.S * a.G;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int m = min(m0 + 16 * u + r16, rows - 1), b = b0 + m / SG, x = m % SG, s = x / a.G, h = hk * a.G + x % a.G;
    w.lim[u] = own_end(a, start, s);
    const u16* qp = a.q + b * a.ql.b + h * a.ql.h + s * a.ql.s + 8 * g;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) w.qf[u][ks] = *reinterpret_cast<const bf16x8_t*>(qp + 32 * ks);
    w.l[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    w.m[u] = -INFINITY;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) w.o[dt][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// keys from `end` on (the prefix) or from the row's own limit on (end < 0) are hidden
template <int U> Q3_DEV void mask_block(const Rows<U>& w, f32x4 (&S)[4][U], int key0, int end, int g) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int rel = (end >= 0 ? end : w.lim[u]) - key0 - group_key(g);
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[kt][u][i] = tile_key(kt) + i < rel ? S[kt][u][i] : -INFINITY;
  }
}
template <int U> Q3_DEV float row_max(const f32x4 (&S)[4][U], int u) {
  float x = __builtin_fmaxf(__builtin_fmaxf(S[0][u][0], S[0][u][1]), __builtin_fmaxf(S[0][u][2], S[0][u][3]));
#pragma unroll
  for (int kt = 1; kt < 4; ++kt)
    x = __builtin_fmaxf(__builtin_fmaxf(x, __builtin_fmaxf(S[kt][u][0], S[kt][u][1])), __builtin_fmaxf(S[kt][u][2], S[kt][u][3]));
  return xmax4(x);
}
// The maxima moved where a block's pass them by more than 2^8; O and the sums are to be multiplied by alpha if some row's did.
template <int U> struct Step {
  float alpha[U], ms[U];
  bool moved;
};
template <int U> Q3_DEV void move_max(Rows<U>& w, Step<U>& t, const float (&x)[U], float scale2, float thr) {
  bool any = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool need = x[u] > w.m[u] + thr || w.m[u] == -INFINITY;
    const float mn = need ? x[u] : w.m[u];
    t.alpha[u] = w.m[u] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((w.m[u] - mn) * scale2);
    w.m[u] = mn;
    t.ms[u] = mn == -INFINITY ? 0.f : mn * scale2;
    any = any || need;
  }
  t.moved = __any(any);
}
template <int U> Q3_DEV void rescale(Rows<U>& w, const Step<U>& t) {
  if (!t.moved) return;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    w.l[u] *= t.alpha[u];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) w.o[dt][u] *= t.alpha[u];
  }
}
template <int U> Q3_DEV void exp_tile(f32x4 (&S)[4][U], const Step<U>& t, float scale2, int u, int kt) {
#pragma unroll
  for (int i = 0; i < 4; ++i) S[kt][u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kt][u][i], scale2, -t.ms[u]));
}
template <typename T, int U> Q3_DEV void pack_block(const f32x4 (&S)[4][U], i32x4 (&P)[U][2]) {
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      P[u][kt >> 1][2 * (kt & 1)] = (int)pack2<T>(S[kt][u][0], S[kt][u][1]);
      P[u][kt >> 1][2 * (kt & 1) + 1] = (int)pack2<T>(S[kt][u][2], S[kt][u][3]);
    }
}
// Scores of a block -> P and the step that O has to take before it.
template <typename T, int U>
Q3_DEV void softmax_block(Rows<U>& w, Step<U>& t, f32x4 (&S)[4][U], i32x4 (&P)[U][2], float scale2, float thr) {
  float x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) x[u] = row_max<U>(S, u);
  move_max(w, t, x, scale2, thr);
  // A product of the maximum and the scale that passes 2^24 is off by more than 1: differences first there.
  bool far = false;
#pragma unroll
  for (int u = 0; u < U; ++u) far = far || fabsf(t.ms[u]) > 0x1p24f;
  if (__builtin_expect(__any(far), 0)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float m = w.m[u] == -INFINITY ? 0.f : w.m[u];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) S[kt][u] -= m;
      t.ms[u] = 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) exp_tile<U>(S, t, scale2, u, kt);
  pack_block<T, U>(S, P);
}

// O^T += V^T P and the sums of P, V's tile at vb.  A value that is not finite would spoil the rows that do not see its position too
// (0 times it is NaN): blocks that some row sees in part (LOOK; the last of a job, in a loop of their own, since the second way
// through the product costs copies of O) are looked through first, and then such values are kept out of the product and
// added to the rows that do see them: all rows see a block of the prefix (pre), whose rows behind its end are zeros here.
template <typename T, int U, bool LOOK>
Q3_DEV void value_block(Rows<U>& w, const i32x4 (&P)[U][2], const char* vb, bool pre, int key0, int g, int r16) {
  const int lane = 16 * g + r16;
  const int voff[2] = {value_offset(g, r16, 0), value_offset(g, r16, 1)};
  bool clean = true;
  if constexpr (LOOK) {
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
        for (int u = 0; u < U; ++u)
          w.o[dt][u] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, P[u][kc]), w.o[dt][u]);
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
        for (int u = 0; u < U; ++u)
          w.o[dt][u] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, P[u][kc]), w.o[dt][u]);
      }
#pragma unroll 1
    for (int key = 0; key < BLK; ++key) {
      const char* row = vb + (key & 15) * kSlot + (key >> 4) * 256 + 8 * g;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const i32x2 x = *reinterpret_cast<const i32x2*>(row + dt * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t bits = ((uint32_t)x[i >> 1] >> (16 * (i & 1))) & 0xffffu;
          const float bad = finite2<T>(bits) ? 0.f : to_f32<T>((u16)bits);
#pragma unroll
          for (int u = 0; u < U; ++u) w.o[dt][u][i] += pre || key0 + key < w.lim[u] ? bad : 0.f;
        }
      }
    }
  }
  const uint32_t one2 = pack2<T>(1.f, 1.f);
  const i32x4 ones = i32x4{(int)one2, (int)one2, (int)one2, (int)one2};
#pragma unroll
  for (int kc = 0; kc < 2; ++kc)
#pragma unroll
    for (int u = 0; u < U; ++u)
      w.l[u] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, ones), __builtin_bit_cast(bf16x8_t, P[u][kc]), w.l[u]);
}

// The range of a job: blocks of the prefix, then of b0's own positions.
struct Job {
  int b0, hk, tile, slot;  // first row b of the job's query rows
  int rows;                // query rows from b0's first on
  int pb, npre, sb, nblk;
  int own, start;          // own positions that the job's last query row sees
  const u16 *pk, *pv, *ck, *cv;
};
struct Block {  // one of them: 64 positions from key0 on, `count` of them there
  int key0, count;
  int64_t st;
  const u16 *k, *v;
};
// The prefix's blocks come last first: its unfinished block is the job's first, so blocks with hidden keys are the first and the last ones.
Q3_DEV int block_key(const Job& job, int j) { return (j < job.npre ? job.pb + job.npre - 1 - j : job.sb + j - job.npre) * BLK; }
Q3_DEV Block block_of(const Args& a, const Job& job, int j) {
  const bool pre = j < job.npre;
  Block x;
  x.key0 = block_key(job, j);
  x.count = min((pre ? a.P : job.own) - x.key0, BLK);
  x.st = pre ? a.pl.s : a.cl.s;
  x.k = (pre ? job.pk : job.ck) + x.key0 * x.st;
  x.v = (pre ? job.pv : job.cv) + x.key0 * x.st;
  return x;
}
Q3_DEV int block_bytes(const Block& x) { return (x.count - 1) * (int)x.st * 2 + 2 * D; }
// The first of a job's blocks that queries of a wave see in part while others of it see it whole; lim: own positions that its first
// row sees.  One query a row sees all that is there.
Q3_DEV int first_partial(const Args& a, const Job& job, int lim) {
  return a.S == 1 ? job.nblk : min(max(lim / BLK - job.sb, 0) + job.npre, job.nblk);
}

// The launch's arguments read again where a job ends: kept from its start, they would crowd its loop's scalars out of registers.
Q3_DEV const Args& args_again() {
  auto p = (const __attribute__((address_space(4))) Args*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args*)p;
}

// A query row's place among the partials, and in the output.
Q3_DEV void row_place(const Args& a, const Job& job, int m, int64_t& part, int64_t& out) {
  const int SG = a.S * a.G, b = job.b0 + m / SG, x = m % SG, s = x / a.G, h = job.hk * a.G + x % a.G;
  part = (((int64_t)b * a.S + s) * (a.Hkv * a.G) + h) * a.slots + job.slot;
  out = b * a.ol.b + h * a.ol.h + s * a.ol.s;
}
template <typename T> Q3_DEV void store4(const Args& a, int64_t part, int64_t out, int d, f32x4 o, float l, bool none) {
  if (a.slots == 1) {
    const float inv = none ? 0.f : 1.f / l;  // no position to see: zeros
    *reinterpret_cast<i32x2*>(a.o + out + d) =
        i32x2{(int)pack2<T>(o[0] * inv, o[1] * inv), (int)pack2<T>(o[2] * inv, o[3] * inv)};
  } else {
    *reinterpret_cast<f32x4*>(a.po + part * D + d) = o;
  }
}

// More query rows: 32 a wave.  Bound by the matrix cores and the softmax between them: 8 x 200 queries of 32 heads behind 4001 (256
// tiles, 78 % full) 131 us, 0.82 PFLOP/s; 64 single queries behind 32768, with up to 1000 positions of the rows' own in jobs beside,
// 67 us (265 MB, 4.0 TB/s).  A third K and V tile in flight, or the softmax of one block beside the products of the next, gave
// nothing more (138 and 134 us where this took 134).
template <typename T, int NW> Q3_DEV void tile_job(const Args& a, const Job& job, char* lds, int wave, int g, int r16) {
  constexpr int RT = 32 * NW, L = 16 / NW;  // L: a wave's loads of a tile
  const int m0 = job.tile * RT + wave * 32, nblk = job.nblk;
  const bool work = m0 < job.rows;  // a wave without rows only loads
  Rows<2> w;
  load_rows(a, w, m0, job.rows, job.b0, job.hk, job.start, g, r16);
  const int lim_w = own_end(a, job.start, min(m0, job.rows - 1) / a.G);  // of the wave's first row, the lowest

  uint32_t krow[L], kchk[L], vrow[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int x = wave + NW * i, r = 4 * x + g;
    krow[i] = (uint32_t)r;
    kchk[i] = (uint32_t)((r16 ^ kswz(r)) * 16);
    vrow[i] = (uint32_t)(x + 16 * g);
  }
  auto issue = [&](int j) {
    if (j >= nblk) return;
    const Block x = block_of(a, job, j);
    const int bytes = block_bytes(x);
    char* base = lds + (j & 1) * kStage;
#pragma unroll
    for (int i = 0; i < L; ++i)
      buffer_to_lds(x.k, bytes, krow[i] * (uint32_t)(x.st * 2) + kchk[i], base + (wave + NW * i) * 1024);
#pragma unroll
    for (int i = 0; i < L; ++i)
      buffer_to_lds(x.v, bytes, vrow[i] * (uint32_t)(x.st * 2) + r16 * 16, base + kKTile + (wave + NW * i) * kSlot);
  };
  int koff[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) koff[ks] = row_key(r16) * 256 + (((4 * ks + g) ^ r16) << 4);
  const float thr = 8.f / a.scale2;

  auto block = [&](int j, auto look) {
    __builtin_amdgcn_s_waitcnt((0 & 15) | (7 << 4) | (0 << 8));  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();  // block j is there, and every wave is done with block j - 1
    asm volatile("" ::: "memory");
    issue(j + 1);
    if (!work) return;
    const char* kb = lds + (j & 1) * kStage;
    f32x4 S[4][2];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(kb + koff[ks] + tile_key(kt) * 256);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          S[kt][u] = mfma_16x16x32<T>(kf, w.qf[u][ks], ks == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : S[kt][u]);
      }
    const bool pre = j < job.npre;
    const int key0 = block_key(job, j);
    const bool mask = key0 + BLK > (pre ? a.P : lim_w);
    if (mask) mask_block<2>(w, S, key0, pre ? a.P : -1, g);
    i32x4 P[2][2];
    Step<2> step;
    softmax_block<T, 2>(w, step, S, P, a.scale2, thr);
    rescale(w, step);
    value_block<T, 2, decltype(look)::value>(w, P, kb + kKTile, pre, key0, g, r16);
  };
  issue(0);
  const int seen = first_partial(a, job, lim_w);
  for (int j = 0; j < seen; ++j) block(j, std::false_type{});
  for (int j = seen; j < nblk; ++j) block(j, std::true_type{});

  const Args& e = args_again();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int m = m0 + 16 * u + r16;
    if (m >= job.rows) continue;
    int64_t part, out;
    row_place(e, job, m, part, out);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
      store4<T>(e, part, out, 16 * dt + 4 * g, w.o[dt][u], w.l[u][0], e.P == 0 && w.lim[u] == 0);
    if (e.slots > 1 && g == 0) {
      e.pm[part] = w.m[u] == -INFINITY ? -INFINITY : w.m[u] * e.scale2;
      e.ps[part] = w.l[u][0];
    }
  }
}

// Up to 16 U query rows: each wave takes every fourth block.  Bound by the loads' latency until many jobs share a CU: 32 single queries
// behind 8192 and 511 of their own 21 us (4.8 TB/s), 4 x 8 behind 2047 20.8 (3.9 TB/s), 4 behind 200 6.9.
template <typename T, int U, bool LOOK> Q3_DEV void few_job(const Args& a, const Job& job, char* lds, int wave, int g, int r16) {
  // 16 rows: the next K on its way beside the softmax and V's product; 32 have no registers for it.
  constexpr bool EARLY = U == 1;
  constexpr int NW = 4, R = 16 * U;
  char* const vt = lds + wave * kVTile;
  const int lim_w = own_end(a, job.start, 0);
  Rows<U> w;
  i32x4 kf[4][4];
  auto load_k = [&](int j) {
    const Block x = block_of(a, job, j);
    const auto d = __builtin_amdgcn_make_buffer_rsrc((void*)x.k, 0, block_bytes(x), 0x00027000);
    const uint32_t off = (uint32_t)row_key(r16) * (uint32_t)(x.st * 2) + 16 * g;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        kf[kt][ks] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(d, off + (uint32_t)tile_key(kt) * (uint32_t)(x.st * 2) + 64 * ks, 0, 0));
  };
  auto load_v = [&](int j) {
    const Block x = block_of(a, job, j);
    const int bytes = block_bytes(x);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      buffer_to_lds(x.v, bytes, (uint32_t)(i + 16 * g) * (uint32_t)(x.st * 2) + r16 * 16, vt + i * kSlot);
  };
  auto fence = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto block = [&](int j) {
    const Block x = block_of(a, job, j);
    f32x4 S[4][U];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int u = 0; u < U; ++u)
          S[kt][u] = mfma_16x16x32<T>(__builtin_bit_cast(bf16x8_t, kf[kt][ks]), w.qf[u][ks], ks == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : S[kt][u]);
    const bool more = j + NW < job.nblk;
    fence();
    if (EARLY && more) load_k(j + NW);
    fence();
    const bool pre = j < job.npre, mask = x.key0 + BLK > (pre ? a.P : lim_w);
    i32x4 P[U][2];
    Step<U> step;
    if (mask) mask_block<U>(w, S, x.key0, pre ? a.P : -1, g);
    softmax_block<T, U>(w, step, S, P, a.scale2, 8.f / a.scale2);
    rescale(w, step);
    // this block's V: everything older than the next K's 16 loads
    fence();
    if (EARLY && more) __builtin_amdgcn_s_waitcnt((16 & 15) | ((16 >> 4) << 14) | (7 << 4) | (15 << 8));
    else __builtin_amdgcn_s_waitcnt((0 & 15) | (7 << 4) | (15 << 8));
    fence();
    value_block<T, U, LOOK>(w, P, vt, pre, x.key0, g, r16);
    if (more) {
      __builtin_amdgcn_s_waitcnt((15) | (3 << 14) | (7 << 4) | (0 << 8));  // the tile is read
      fence();
      if (!EARLY) load_k(j + NW);
      load_v(j + NW);
    }
  };
  if (wave < job.nblk) {
    load_k(wave);
    load_v(wave);
  }
  load_rows(a, w, 0, job.rows, job.b0, job.hk, job.start, g, r16);
  for (int j = wave; j < job.nblk; j += NW) block(j);
  // The waves' sums joined: wave i's O [R][128], maxima and sums at its tile.  What is left there is read by the wave itself.
  __builtin_amdgcn_s_waitcnt((15) | (3 << 14) | (7 << 4) | (0 << 8));
  fence();
  constexpr int kRow = D * 4 + 16;  // 16 bytes of padding a row
  static_assert(R * kRow <= kVTile, "fits the wave's tile");
  float* const stat = (float*)(lds + NW * kVTile);  // [wave][2][R]
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
      *reinterpret_cast<f32x4*>(vt + (16 * u + r16) * kRow + (16 * dt + 4 * g) * 4) = w.o[dt][u];
    if (g == 0) {
      stat[(wave * 2 + 0) * R + 16 * u + r16] = w.m[u] == -INFINITY ? -INFINITY : w.m[u] * a.scale2;
      stat[(wave * 2 + 1) * R + 16 * u + r16] = w.l[u][0];
    }
  }
  __syncthreads();
  // 32 lanes a row, 4 dims each
  const Args& out_args = args_again();
  const int t = wave * 64 + 16 * g + r16, l = t & 31;
  for (int m = t >> 5; m < job.rows; m += 8) {
    float M = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) M = __builtin_fmaxf(M, stat[(i * 2) * R + m]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float mi = stat[(i * 2) * R + m], e = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - M);
      sum = __builtin_fmaf(e, stat[(i * 2 + 1) * R + m], sum);
      o += e * *reinterpret_cast<const f32x4*>(lds + i * kVTile + m * kRow + l * 16);
    }
    int64_t part, out;
    row_place(out_args, job, m, part, out);
    store4<T>(out_args, part, out, 4 * l, o, sum, out_args.P == 0 && own_end(out_args, job.start, m / out_args.G) == 0);
    if (out_args.slots > 1 && l == 0) {
      out_args.pm[part] = M;
      out_args.ps[part] = sum;
    }
  }
}

// Pointers to a job's keys and values.
Q3_DEV void job_pointers(const Args& a, Job& job) {
  // in scalar registers, whatever way they came: the tiles' descriptors are formed from them
  for (int* x : {&job.b0, &job.hk, &job.tile, &job.slot, &job.rows, &job.pb, &job.npre, &job.sb, &job.nblk, &job.own, &job.start})
    *x = __builtin_amdgcn_readfirstlane(*x);
  job.pk = a.pk + job.b0 / a.n * a.pl.b + job.hk * a.pl.h;
  job.pv = a.pv + job.b0 / a.n * a.pl.b + job.hk * a.pl.h;
  job.ck = a.ck + job.b0 * a.cl.b + job.hk * a.cl.h;
  job.cv = a.cv + job.b0 * a.cl.b + job.hk * a.cl.h;
}
// Job w of the prefix: row tiles innermost.
Q3_DEV void prefix_job(const Args& a, Job& job, int w) {
  job.tile = w % a.ptiles;
  w /= a.ptiles;
  job.slot = w % a.psplits;
  w /= a.psplits;
  job.hk = w % a.Hkv;
  job.b0 = w / a.Hkv * a.n;
  job.rows = a.n * a.S * a.G;
  job.pb = job.slot * a.pper;
  job.npre = job.nblk = min(a.pper, (a.P + BLK - 1) / BLK - job.pb);
}
// Job w of the rows' own positions, with tiles of RT query rows; false: there is no such split (the joining launch knows).
Q3_DEV bool own_job(const Args& a, Job& job, int w, int RT) {
  const int SG = a.S * a.G;
  job.tile = w % a.stiles;
  w /= a.stiles;
  job.hk = w % a.Hkv;
  w /= a.Hkv;
  const int split = w % a.ssplits;
  job.b0 = w / a.ssplits;
  job.rows = SG;
  job.start = __builtin_amdgcn_readfirstlane(row_start(a, job.b0));
  const int all = (own_end(a, job.start, a.S - 1) + BLK - 1) / BLK;
  job.own = own_end(a, job.start, min(job.tile * RT + RT - 1, SG - 1) / a.G);
  const int blocks = (job.own + BLK - 1) / BLK, per = own_per(a, all);
  const int pre = a.fused ? (a.P + BLK - 1) / BLK : 0;
  job.sb = a.fused ? 0 : split * per;
  job.npre = pre;
  job.nblk = pre + (a.fused ? blocks : max(min(per, blocks - job.sb), 0));
  job.slot = a.psplits + split;
  return split == 0 || job.sb < all;
}

// A workgroup's job.  The launch has pjobs jobs of the prefix and sjobs of the rows' own positions, 256 of each in turn as long as
// there are such: workgroups that many apart share a CU, and the first kind keeps the matrix cores busy, the second the memory.
// Jobs of the prefix: each XCD (workgroup ids congruent mod 8) takes a contiguous range, so that row tiles that read the same keys share
// an L2.  false: nothing to do.
Q3_DEV bool find_job(const Args& a, Job& job, int RT, bool& own) {
  const int id = blockIdx.x, both = min(a.pjobs, a.sjobs) & ~255;
  int w;
  if (id < 2 * both) {
    own = (id >> 8) & 1;
    w = (id >> 9) * 256 + (id & 255);
  } else {
    w = id - both;  // the rest of the prefix's jobs, then of the others
    own = w >= a.pjobs;
    if (own) w = id - a.pjobs;
  }
  if (own) {
    if (!own_job(a, job, w, RT)) return false;
  } else {
    const int xcd = w & 7, per = a.pjobs >> 3, rem = a.pjobs & 7;
    prefix_job(a, job, xcd * per + min(xcd, rem) + (w >> 3));
  }
  job_pointers(a, job);
  return true;
}

template <typename T, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefix_tile_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Job job{};
  bool own;
  if (!find_job(a, job, 32 * NW, own)) return;
  tile_job<T, NW>(a, job, lds, wave, (tid & 63) >> 4, tid & 15);
}

// Jobs of up to 16 U rows, and with TILES the prefix's of more.  LOOK: several queries a row.
template <typename T, int U, bool TILES, bool LOOK>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefix_few_kernel(Args a) {
  constexpr int kFew = 4 * kVTile + 4 * 2 * 16 * U * 4, kTiles = 2 * kStage;
  __shared__ __attribute__((aligned(1024))) char lds[TILES && kTiles > kFew ? kTiles : kFew];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Job job{};
  bool own;
  if (!find_job(a, job, 32, own)) return;
  if constexpr (TILES) {
    if (!own) {
      tile_job<T, 4>(a, job, lds, wave, (tid & 63) >> 4, tid & 15);
      return;
    }
  }
  few_job<T, U, LOOK>(a, job, lds, wave, (tid & 63) >> 4, tid & 15);
}

// o = sum_j 2^(m_j - M) O_j / sum_j 2^(m_j - M) s_j over a query row's slots: the prefix's splits, then those of its own positions.
// GR groups of 32 lanes (4 dims a lane) take every GR-th slot each, four loads in flight, and are added in order.  Bound by its
// launch and one trip to the caches: 4 x 32 query rows of 2 slots 2.6 us, 64 x 32 of 17 6.8.
template <typename T, int GR> __global__ __launch_bounds__(256) void prefix_join_kernel(Args a, int64_t rows) {
  constexpr int RB = 8 / GR;  // rows a workgroup
  __shared__ f32x4 part[RB][GR][32];
  __shared__ float psum[RB][GR];
  const int l = threadIdx.x & 31, grp = (threadIdx.x >> 5) % GR, rb = (threadIdx.x >> 5) / GR, Hq = a.Hkv * a.G;
  const int64_t row = min((int64_t)blockIdx.x * RB + rb, rows - 1);
  const float *pm = a.pm + row * a.slots, *ps = a.ps + row * a.slots, *po = a.po + row * a.slots * D + 4 * l;
  f32x4 x[4];
  float m[4], sj[4];
  auto load = [&](int j0) {  // slots that the row has not are loaded too (they are there), and not used
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = min(j0 + k * GR, a.slots - 1);
      x[k] = *reinterpret_cast<const f32x4*>(po + (int64_t)j * D);
      m[k] = pm[j];
      sj[k] = ps[j];
    }
  };
  load(grp);
  const float m0 = pm[min(l, a.slots - 1)];
  const int64_t bs = row / Hq;
  const int h = (int)(row - bs * Hq), b = (int)(bs / a.S), s = (int)(bs - (int64_t)b * a.S);
  const int start = row_start(a, b), all = (own_end(a, start, a.S - 1) + BLK - 1) / BLK;
  const int per = own_per(a, all);
  const int used = a.psplits + max((all + per - 1) / per, 1);
  float M = l < used ? m0 : -INFINITY;
  for (int j = l + 32; j < used; j += 32) M = __builtin_fmaxf(M, pm[j]);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) M = __builtin_fmaxf(M, __shfl_xor(M, o, 64));
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = grp; j0 < used; j0 += 4 * GR) {
    if (j0 != grp) load(j0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (j0 + k * GR >= used) continue;
      // a slot without a maximum may hold a sum that is not a number (scores that are none beside hidden ones): times 0 it stays one
      const float w = m[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[k] - M);
      sum = __builtin_fmaf(w, sj[k], sum);
      o += w * x[k];
    }
  }
  part[rb][grp][l] = o;
  if (l == 0) psum[rb][grp] = sum;
  __syncthreads();
  if (grp != 0 || (int64_t)blockIdx.x * RB + rb >= rows) return;
#pragma unroll
  for (int k = 1; k < GR; ++k) {
    o += part[rb][k][l];
    sum += psum[rb][k];
  }
  const float inv = a.P == 0 && own_end(a, start, s) == 0 ? 0.f : 1.f / sum;
  u16* out = a.o + b * a.ol.b + s * a.ol.s + h * a.ol.h + 4 * l;
  *reinterpret_cast<i32x2*>(out) = i32x2{(int)pack2<T>(o[0] * inv, o[1] * inv), (int)pack2<T>(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------- host
int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }
bool al(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }
bool lay_ok(const void* p, const Strides& l) { return p && al(p, 16) && l.b % 8 == 0 && l.h % 8 == 0 && l.s % 8 == 0; }

// The jobs of a call; span: own positions that the launches have to cover.
struct Plan {
  int fused, pfew, sfew, nw, ptiles, psplits, pper, stiles, ssplits, max_splits, slots;
  int64_t pjobs, sjobs;
};
constexpr int kMinPer = 4;  // blocks of a split at least
Plan plan_for(int64_t R, int64_t n, int64_t S, int64_t Hkv, int64_t G, int64_t P, int64_t C, int64_t span) {
  Plan p{};
  const int64_t B = R * n, SG = S * G, pblocks = cdiv(P, BLK);
  // One pass over everything, a row's own queries in tiles of 256, a tile a CU: where the queries fill more than 11 / 20 of the
  // CUs' tiles in its rounds.  No partial sums are written, but a CU without a tile and a tile's missing rows are lost: 8 heads of
  // 4 queries, 100 own positions, behind 4001: 8 x 200 (0.78) 136 against 162 us in jobs, 6 x 200 (0.59) 133 against 154,
  // 5 x 200 (0.49) 133 against 113; behind 3000: 24 x 64 (0.75) 103 against 130, 40 x 40 (0.39) 185 against 132.
  const int64_t tiles = B * Hkv * cdiv(SG, 256);
  if (20 * B * Hkv * SG > 11 * 256 * 256 * cdiv(tiles, 256)) {
    p.fused = p.ptiles = 1;
    p.nw = 8;
    p.stiles = (int)cdiv(SG, 256);
    p.ssplits = p.max_splits = p.slots = 1;
    p.sjobs = B * Hkv * p.stiles;
    return p;
  }
  // About a workgroup a CU for each kind of position, two in all, if that leaves kMinPer blocks a job.  More would fill the CUs in
  // finer pieces, but every one writes its rows' O for the second launch (64 rows behind 32768: 256 jobs 80 us, 512 85, 1024 100).
  constexpr int64_t kJobs = 256;
  // Few rows to a job: 32 of single queries (8 x 4 behind 8192 22.9 us and 22.2 in tiles, 5 x 4 behind 32768 34.5 and 36.8, 7 x 4
  // behind 1000 17.1 and 18.1), 16 of longer chunks, whose products look at values (4 x 8 behind 8192 24.6 and 22.3 in tiles, 1 x 32
  // 23.6 and 20.4).
  const int64_t few = S == 1 ? 32 : 16;
  p.pfew = P > 0 && n * SG <= few;
  p.sfew = SG <= few;
  p.nw = 4;
  p.ptiles = 1;
  // One pass a row and head over its prefix and its own positions where few blocks of both fit (counted by the capacity, so that a captured
  // step goes the way of an eager call): no second launch and no partial sums, but a prefix is read once a row.  By the rounds of a
  // job's four waves (2.2 us each) against the two launches (us, single queries behind 200 and 500 positions, a position block of
  // their own): 1 row 7.1 and 8.7, 9.5 and 9.0; 8 rows of 8 heads 7.3 and 10.9, 9.6 and 11.3; 32 7.4 and 14.1, 9.7 and 14.3; 64 9.8
  // and 14.5, 14.9 and 14.8.  Four rounds: 8 rows 11.8 and 11.3, 32 14.5 and 17.9, 64 23.7 and 23.7.
  const int64_t rounds = cdiv(pblocks + cdiv(C, BLK), 4), jobs = B * Hkv;
  if (p.sfew && jobs <= 512 && rounds <= (jobs > 256 ? 2 : jobs >= 64 ? 4 : 3)) {
    p.fused = 1;
    p.stiles = p.ssplits = p.max_splits = p.slots = 1;
    p.sjobs = jobs;
    p.pfew = 0;
    return p;
  }
  if (P > 0) {
    p.ptiles = p.pfew ? 1 : (int)cdiv(n * SG, 128);
    const int64_t want = std::max<int64_t>(1, kJobs / (R * Hkv * p.ptiles));
    p.pper = (int)std::max<int64_t>(cdiv(pblocks, want), kMinPer);
    if (p.pfew) p.pper = (p.pper + 3) & ~3;
    p.psplits = (int)cdiv(pblocks, p.pper);
    p.pjobs = R * Hkv * p.ptiles * p.psplits;
  }
  p.stiles = p.sfew ? 1 : (int)cdiv(SG, 128);
  p.max_splits = (int)std::max<int64_t>(1, kJobs / (B * Hkv * p.stiles));
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
  const bool one = a.S * a.G * (p.pfew ? a.n : 1) <= 16;  // 16 rows a job at most
  auto few = [&](auto tiles) {
    constexpr bool TILES = decltype(tiles)::value;
    if (a.S == 1)
      one ? prefix_few_kernel<T, 1, TILES, false><<<grid, 256, 0, s>>>(a) : prefix_few_kernel<T, 2, TILES, false><<<grid, 256, 0, s>>>(a);
    else
      prefix_few_kernel<T, 1, TILES, true><<<grid, 256, 0, s>>>(a);
  };
  if (p.nw == 8) prefix_tile_kernel<T, 8><<<grid, 512, 0, s>>>(a);
  else if (!p.sfew) prefix_tile_kernel<T, 4><<<grid, 256, 0, s>>>(a);
  else if (p.pfew || p.fused || a.P == 0) few(std::false_type{});
  else few(std::true_type{});
  const int rc = (int)hipGetLastError();
  if (p.slots == 1) return rc;
  // many slots: a workgroup a row (by what the sizes allow, not by the span: the order of the sums)
  if (p.psplits + p.max_splits > 8) prefix_join_kernel<T, 8><<<(unsigned)rows, 256, 0, s>>>(a, rows);
  else prefix_join_kernel<T, 2><<<(unsigned)cdiv(rows, 4), 256, 0, s>>>(a, rows);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t q3_prefix_attention_workspace_bytes(int64_t B, int64_t R, int64_t S, int64_t Hq, int64_t Hkv, int64_t P, int64_t C,
                                           int64_t span) {
  if (!sizes_ok(B, R, S, Hq, Hkv, P, C) || span < 0 || span > C) return 0;
  return bytes_for(plan_for(R, B / R, S, Hkv, Hq / Hkv, P, C, span), B * S * Hq);
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
  const Plan p = plan_for(R, n, S, Hkv, Hq / Hkv, P, C, span);
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
  a.sjobs = (int)p.sjobs;
  a.sfew = p.sfew;
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
