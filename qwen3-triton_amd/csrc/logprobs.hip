// Log probabilities of given tokens, with the entropy and the most likely alternatives, from rows of logits; and their gradient.
//
// For a row z of V logits at temperature 1 / c:  M = max z, d_i = c (z_i - M), rest = the sum of e^d_i over all but one element
// that is M, total = 1 + rest:
//   log p_i = d_i - log1p(rest),   entropy = log1p(rest) - (sum e^d_i d_i) / total
// Both terms of the entropy are >= 0 and log1p sees the small part of the sum by itself, so a row that is almost certain keeps
// its digits (1 + rest as one number holds nothing of a rest below 2^-24).  Statistics (M, rest, sum e^d (z - M)) of parts of a
// row join exactly like those of an online softmax.
//   dz_i = c (sum_j g_j [i = token_j] - p_i (sum_j g_j + h (log p_i + entropy)))
// over the given token and the alternatives (upstream gradients g_j) and the entropy (h); at i = token_j, 1 - p_i is formed as
// -expm1(log p_i).
//
// Bound by the logits, read once (forward) or read and written once (backward).  A workgroup holds its slice of a row in
// registers: the slice's maximum, then the sums, then the alternatives are taken from them.  Many rows take slices of 32 values (fp32: 16) a
// thread; few rows small ones, so that one row's latency is spread over many CUs.  A second launch joins a
// row's slices, unless one workgroup goes through all of them (short rows; very many rows).
// On MI355X (kernels alone, 151936 logits a row): 4096 rows of bf16 196 us (6.4 TB/s), 777 of fp32 with 5 alternatives 75 + 7 (6.2 TB/s),
// one row with 20 alternatives 7.3 + 6.3; the gradient of 2048 bf16 rows 260 us (4.8 TB/s).
#include <algorithm>

#include "logprobs.h"

namespace {

using namespace q3lp;

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;
constexpr int kGradVectors = 4;  // 16-byte vectors of logits a thread

// ---------------------------------------------------------------- the largest k
// Values as whole numbers in their order, NaN above all, 0 below all; keys: the value's order, then the lower index first.
Q3_DEV uint32_t order32(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as +0
  return x != x ? 0xffffffffu : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
Q3_DEV float unorder32(uint32_t k) {
  return k == 0xffffffffu ? NAN : __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
Q3_DEV uint64_t key_of(uint32_t order, uint32_t index) { return ((uint64_t)order << 32) | (uint32_t)~index; }
Q3_DEV uint64_t key_xor(uint64_t x, int mask) {
  return ((uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), mask, 64) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)x, mask, 64);
}

// The k largest (k <= kMaxTop) of a workgroup's values in order, to emit(rank, key) by some thread each; ranks that no value
// takes get key 0.  most: the order of the thread's largest value (0: it has none), and no higher, or ranks would stay empty;
// scan(f) calls f(order, index) for each of its values, order 0 for none, and may read them again; collect(reaches, f), called by
// all threads, does so for at least the values of the threads for which `reaches`.
//  * The 64 maxima of groups of 4 threads: the k-th largest of those is a bound that at least k values reach.  Of random
//    values about 1.3 k do; they are collected and ranked by counting the larger ones.
//  * More than kCand may reach it (ties, a row that rises, few values that are not -inf): then k rounds, each the largest key
//    left, whose thread looks for its next one.
constexpr int kCand = 2 * kThreads;
struct TopScratch {
  alignas(16) uint64_t cand[kCand];
  alignas(16) uint32_t group[64];
  uint64_t wave[kThreads / 64];
  uint32_t bound;
  int count;
};
template <typename Collect, typename Scan, typename Emit>
Q3_DEV void block_top(TopScratch& sc, int k, uint32_t most, Collect&& collect, Scan&& scan, Emit&& emit) {
  const int tid = threadIdx.x;
  uint32_t g = max(most, (uint32_t)__shfl_xor((int)most, 1, 64));
  g = max(g, (uint32_t)__shfl_xor((int)g, 2, 64));
  if ((tid & 3) == 0) sc.group[tid >> 2] = g;
  if (tid == 0) sc.count = 0;
  __syncthreads();
  if (tid < 64) {
    const uint32_t mine = sc.group[tid];
    int larger = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      const uint32_t o = sc.group[i];
      larger += (o > mine || (o == mine && i < tid)) ? 1 : 0;
    }
    if (larger == k - 1) sc.bound = mine;
  }
  __syncthreads();
  const uint32_t bound = sc.bound;
  collect(most >= bound && most != 0, [&](uint32_t o, uint32_t i) {
    if (o >= bound && o != 0) {
      const int at = atomicAdd(&sc.count, 1);
      if (at < kCand) sc.cand[at] = key_of(o, i);
    }
  });
  __syncthreads();
  const int n = sc.count;
  if (n <= kCand) {
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t mine = sc.cand[i];
      int larger = 0, j = 0;
      for (; j + 16 <= n; j += 16)  // 16 reads in flight together
#pragma unroll
        for (int e = 0; e < 16; ++e) larger += sc.cand[j + e] > mine ? 1 : 0;
#pragma unroll 4
      for (; j < n; ++j) larger += sc.cand[j] > mine ? 1 : 0;
      if (larger < k) emit(larger, mine);
    }
    if (tid >= n && tid < k) emit(tid, (uint64_t)0);
    return;
  }
  uint64_t best = 0, below = ~0ull;
  for (int r = 0; r < k; ++r) {
    if (most != 0 && (r == 0 || best == 0)) {  // look for the thread's largest key below its last one
      scan([&](uint32_t o, uint32_t i) {
        const uint64_t x = o ? key_of(o, i) : 0;
        best = x > best && x < below ? x : best;
      });
      if (best == 0) most = 0;  // it has no more
    }
    uint64_t w = best;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t y = key_xor(w, o);
      w = y > w ? y : w;
    }
    __syncthreads();  // the last round's maxima are read
    if ((tid & 63) == 0) sc.wave[tid >> 6] = w;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) w = sc.wave[i] > w ? sc.wave[i] : w;
    if (w == 0 ? tid == 0 : w == best) {
      emit(r, w);
      below = best;
      best = 0;
    }
  }
}

// ---------------------------------------------------------------- one slice of a row
struct Fwd {
  const void* z;
  int64_t ld, rows, vocab;
  const int64_t* tok;
  int64_t ignore;
  float c;      // 1 / temperature
  int top, slices, span, per, parts;  // slices of a row, their elements, slices of a workgroup, workgroups of a row
  Part* part;   // [rows][parts]
  uint64_t* key;  // [rows][parts][top]
  float *logprob, *entropy, *m, *ls;  // ls: log1p(rest); m and ls: for the gradient, or null
  float* top_logprob;
  int64_t* top_token;
};

// Elements between the 16-byte boundary before a row and its start.
template <typename T> Q3_DEV int misaligned(const typename T::storage* row) {
  return (int)(((uintptr_t)row & 15) / sizeof(typename T::storage));
}
template <typename T> constexpr uint32_t kLowest = T::code == Q3_F32 ? 0xff800000u : T::code == Q3_F16 ? 0xfc00fc00u : 0xff80ff80u;

// 16 bytes from element i0 of a row of n on: i0 counts from a 16-byte boundary at or before the row, so only a row's first and
// last vectors are not whole; elements outside the row are -inf.
template <typename T> Q3_DEV i32x4 load_edge(const typename T::storage* row, int64_t i0, int64_t n) {
  if (i0 >= 0 && i0 + T::vec <= n) return *reinterpret_cast<const i32x4*>(row + i0);
  i32x4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t x = kLowest<T>;
    if constexpr (T::vec == 4) {
      if (i0 + w >= 0 && i0 + w < n) x = __float_as_uint(row[i0 + w]);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t i = i0 + 2 * w + e;
        if (i >= 0 && i < n) x = (x & ~(0xffffu << (16 * e))) | ((uint32_t)row[i] << (16 * e));
      }
    }
    v[w] = (int)x;
  }
  return v;
}
// C vectors a thread of the slice that starts at element `base`, 256 threads side by side; past the caches, since each is read once
// (4096 x 151936 bf16 206 us and 226 without, 1000 x 32000 19.5 either way; alternatives' second look takes as long).
template <typename T, int C> Q3_DEV void load_slice(i32x4 (&v)[C], const typename T::storage* row, int64_t base, int64_t n) {
  constexpr int V = T::vec;
  if (base >= 0 && base + kThreads * V * C <= n) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = ld_nt(row + base + (i * kThreads + (int)threadIdx.x) * V);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = load_edge<T>(row, base + (i * kThreads + (int)threadIdx.x) * V, n);
  }
}
template <typename T, int C> Q3_DEV void unpack(float (&x)[C * T::vec], const i32x4 (&v)[C]) {
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const Vec<T> f = unpack_vec<T>(v[i]);
#pragma unroll
    for (int e = 0; e < T::vec; ++e) x[i * T::vec + e] = f.v[e];
  }
}

// A row's results from its statistics.
Q3_DEV void finish_row(const Fwd& a, int64_t r, const Part& p, float picked, bool valid) {
  const float ls = log1pf(p.rest), d = picked - p.m;
  const bool none = p.m == -INFINITY;
  a.logprob[r] = valid ? fmaf(d, a.c, -ls) : NAN;
  a.entropy[r] = none ? NAN : fmaf(-kLn2, p.u / (1.f + p.rest), ls);
  if (!a.m) return;
  a.m[r] = p.m;
  a.ls[r] = none ? NAN : ls;
}

// The alternative of a rank, from its key.
Q3_DEV void finish_top(const Fwd& a, int64_t r, int rank, uint64_t k, const Part& p) {
  a.top_token[r * a.top + rank] = (int64_t)(uint32_t)~(uint32_t)k;
  const float x = unorder32((uint32_t)(k >> 32));
  a.top_logprob[r * a.top + rank] = p.m == -INFINITY ? NAN : fmaf(x - p.m, a.c, -log1pf(p.rest));
}

// Called by the row's threads 0 .. kMaxTop - 1 at least.
Q3_DEV void left_out(const Fwd& a, int64_t r, int tid) {
  if (tid == 0) a.logprob[r] = a.entropy[r] = 0.f;
  if (tid == 0 && a.m) a.m[r] = a.ls[r] = 0.f;
  if (tid < a.top) {
    a.top_logprob[r * a.top + tid] = 0.f;
    a.top_token[r * a.top + tid] = 0;
  }
}

// Bound by the logits where rows are many (the next slice is on its way beside the sums: with part_of's four chains of 32 values
// these take about as long as the loads), by one trip to memory and the reductions where they are few.
// ONE: the workgroup's slices are the whole row, whose results it writes.
template <typename T, int C, bool TOP, bool ONE>
__global__ __launch_bounds__(kThreads) void slice_kernel(Fwd a) {
  typedef typename T::storage S;
  constexpr int V = T::vec;
  const int N = a.span;
  const int64_t r = ONE ? blockIdx.x : blockIdx.x / (unsigned)a.parts;
  const int part = ONE ? 0 : (int)(blockIdx.x - (unsigned)(r * a.parts)), tid = threadIdx.x;
  const int64_t t = a.tok[r];
  if (t == a.ignore) {  // the whole workgroup: nothing of the row is read
    if (ONE) left_out(a, r, tid);
    return;
  }
  const S* row = (const S*)a.z + r * a.ld;
  const int mis = misaligned<T>(row);
  const float c2 = a.c * kLog2e;
  const int first = part * a.per, last = ONE ? a.slices : min(first + a.per, a.slices);
  const bool valid = t >= 0 && t < a.vocab;
  [[maybe_unused]] const float picked = ONE && tid == 0 && valid ? to_f32<T>(row[t]) : 0.f;
  Part p{-INFINITY, 0.f, 0.f};
  [[maybe_unused]] bool nan = false;  // among the thread's values (p.rest is NaN for +inf too)
  i32x4 raw[C];
  auto load = [&](int sl) {
    const int64_t base = (int64_t)sl * N - mis;
    load_slice<T, C>(raw, row, base, min(a.vocab, base + N));
  };
  load(first);
  for (int sl = first; sl < last; ++sl) {
    float x[C * V];
    unpack<T, C>(x, raw);
    if (sl + 1 < last) load(sl + 1);  // in flight meanwhile
    const Part q = part_of(x, c2);
    if constexpr (TOP) nan = nan || (q.m == -INFINITY && q.rest != q.rest);
    p = sl == first ? q : join(p, q, c2);
  }
  [[maybe_unused]] uint32_t most = 0;  // the order of the thread's largest value
  if constexpr (TOP) {
    const int64_t begin = (int64_t)first * N - mis + tid * V;  // of the thread's first vector
    const bool any = begin < a.vocab && begin + V > 0 && tid * V < N;
    most = !any ? 0 : nan ? order32(NAN) : order32(p.m);
  }
  // over the wave: one lane that holds the maximum gives its rest, the others their totals
  const float wm = group_max<64>(p.m);
  {
    const uint64_t at = __ballot(p.m == wm);
    const bool one = (threadIdx.x & 63) == (unsigned)__builtin_ctzll(at | (1ull << 63));
    const float d = (p.m - wm) * c2, w = p.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(d);
    const float full = part_total(p), t = one ? p.rest : full;
    p.u = group_sum<64>(p.m == -INFINITY ? 0.f : w * fmaf(full, fmaxf(d, kDeep), p.u));
    p.rest = group_sum<64>(t * w);
    p.m = wm;
  }
  __shared__ Part wave_part[kThreads / 64];
  if ((tid & 63) == 0) wave_part[tid >> 6] = p;
  __syncthreads();
  [[maybe_unused]] __shared__ Part row_part;
  if (tid == 0) {
    p = wave_part[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) p = join(p, wave_part[w], c2);
    if constexpr (ONE) {
      finish_row(a, r, p, picked, valid);
      row_part = p;
    } else {
      a.part[r * a.parts + part] = p;
    }
  }
  if constexpr (TOP) {
    __shared__ TopScratch sc;
    __shared__ int who[kThreads], whos;
    [[maybe_unused]] uint64_t* out = a.key + (r * a.parts + part) * a.top;
    if (tid == 0) whos = 0;
    const int each = (last - first) * C;  // vectors of a thread
    auto look = [&](int thread, int v, auto&& f) {
      const int64_t base = (int64_t)(first + v / C) * N - mis, i0 = base + (v % C * kThreads + thread) * V, end = min(a.vocab, base + N);
      const Vec<T> x = unpack_vec<T>(load_edge<T>(row, i0, end));
#pragma unroll
      for (int e = 0; e < V; ++e) f(i0 + e >= 0 && i0 + e < end ? order32(x.v[e]) : 0, (uint32_t)(i0 + e));
    };
    // The threads whose maximum reaches the bound are few, but one in most waves: all threads look at a vector of theirs each (5 of 777 bf16
    // rows 66 us, 10 of 2000 133; each such thread at its own, one after the other, 100 and 225).
    block_top(sc, a.top, most, [&](bool reaches, auto&& f) {
      if (reaches) who[atomicAdd(&whos, 1)] = tid;
      __syncthreads();
      const int n = whos * each;
      for (int i = tid; i < n; i += kThreads) look(who[i / each], i % each, f);
    }, [&](auto&& f) {
#pragma unroll 1
      for (int v = 0; v < each; ++v) look(tid, v, f);
    }, [&](int rank, uint64_t k) {  // behind barriers: row_part is there
      if constexpr (ONE) finish_top(a, r, rank, k, row_part);
      else out[rank] = k;
    });
  }
}

// ---------------------------------------------------------------- a row's slices joined
// One wave a row, no alternatives (2048 rows of three parts 4 us: a launch).
template <typename T> __global__ __launch_bounds__(kThreads) void finish_kernel(Fwd a) {
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (r >= a.rows) return;
  const int64_t t = a.tok[r];
  if (t == a.ignore) {
    left_out(a, r, lane);
    return;
  }
  const bool valid = t >= 0 && t < a.vocab;
  const float picked = valid ? to_f32<T>(((const typename T::storage*)a.z)[r * a.ld + t]) : 0.f;
  const float c2 = a.c * kLog2e;
  Part p{-INFINITY, 0.f, 0.f};
  for (int i = lane; i < a.parts; i += 64) p = join(p, a.part[r * a.parts + i], c2);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
    p = join(p, Part{__shfl_xor(p.m, o, 64), __shfl_xor(p.rest, o, 64), __shfl_xor(p.u, o, 64)}, c2);
  if (lane == 0) finish_row(a, r, p, picked, valid);
}

// One workgroup a row: the alternatives are the largest of its slices' largest.  Bound by latencies: a load of the keys, the bound, the
// ranks, 6.3 us for one row's 75 slices of 20.
template <typename T> __global__ __launch_bounds__(kThreads) void finish_top_kernel(Fwd a) {
  __shared__ TopScratch sc;
  __shared__ Part row_part;
  constexpr int R = 8;  // keys of a thread in registers
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, n = a.parts * a.top;
  const int64_t t = a.tok[r];
  const uint64_t* key = a.key + r * n;
  uint64_t mine[R];
  if (t != a.ignore) {
#pragma unroll
    for (int i = 0; i < R; ++i) mine[i] = tid + i * kThreads < n ? key[tid + i * kThreads] : 0;
  }
  if (t == a.ignore) {
    left_out(a, r, tid);
    return;
  }
  if (tid < 64) {
    const bool valid = t >= 0 && t < a.vocab;
    const float picked = valid ? to_f32<T>(((const typename T::storage*)a.z)[r * a.ld + t]) : 0.f;
    const float c2 = a.c * kLog2e;
    Part p{-INFINITY, 0.f, 0.f};
    for (int i = tid; i < a.parts; i += 64) p = join(p, a.part[r * a.parts + i], c2);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
      p = join(p, Part{__shfl_xor(p.m, o, 64), __shfl_xor(p.rest, o, 64), __shfl_xor(p.u, o, 64)}, c2);
    if (tid == 0) {
      finish_row(a, r, p, picked, valid);
      row_part = p;
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) most = max(most, (uint32_t)(mine[i] >> 32));
  for (int i = tid + R * kThreads; i < n; i += kThreads) most = max(most, (uint32_t)(key[i] >> 32));
  auto scan = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < R; ++i) f((uint32_t)(mine[i] >> 32), ~(uint32_t)mine[i]);
    for (int i = tid + R * kThreads; i < n; i += kThreads) f((uint32_t)(key[i] >> 32), ~(uint32_t)key[i]);
  };
  block_top(sc, a.top, most, [&](bool reaches, auto&& f) {
    if (reaches) scan(f);
  }, scan, [&](int rank, uint64_t k) { finish_top(a, r, rank, k, row_part); });  // behind barriers: row_part is there
}

// ---------------------------------------------------------------- gradient
// N values as one store of N elements; FAR: past the caches.
template <typename O, int N, bool FAR> Q3_DEV void store_values(typename O::storage* p, const float (&v)[N]) {
  if constexpr (N == O::vec) {
    Vec<O> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = v[e];
    if constexpr (FAR) st_nt<O>(p, o);
    else store_vec<O>(p, o);
  } else {
    static_assert(N == 4 && O::vec == 8, "fp32 logits, 16-bit gradient");
    const i32x2 o = {(int)pack2<O>(v[0], v[1]), (int)pack2<O>(v[2], v[3])};
    if constexpr (FAR) __builtin_nontemporal_store(o, reinterpret_cast<i32x2*>(p));
    else *reinterpret_cast<i32x2*>(p) = o;
  }
}

struct Bwd {
  const void* z;
  int64_t ld, rows, vocab;
  const int64_t* tok;
  int64_t ignore;
  float c;
  int top;
  const int64_t* top_token;
  const float *m, *ls, *entropy, *g, *gh, *gtop;
  void* dz;
  int64_t ldo;
  const float* scale;  // fp16 gradients: a power of two that they are multiplied with (scale_kernel), or null
};
Q3_DEV float scale_of(const Bwd& a) { return a.scale ? *a.scale : 1.f; }

// A gradient in fp16 that products are formed from is scaled into the type's range, and the products take the scale back before they
// round: with a mean of 4096 rows and 151936 tokens, single values (1e-9) would be below its smallest number and add up to nothing.
// scale[0] = 2^e such that no value passes 2^14, scale[1] = 2^-e: what |dz| is at most, c (|g| + sum |g_j| + |h| (1 + log V)), from all
// rows that are not left out and have a number for it (p |log p| <= 1 / e, p entropy <= log V).  One value for all rows, since dW sums over
// them.  One workgroup (4096 rows 7.6 us).
constexpr int kScaleThreads = 1024;
__global__ __launch_bounds__(kScaleThreads) void scale_kernel(Bwd a, float log_v, float* __restrict__ scale) {
  __shared__ float wave_most[kScaleThreads / 64];
  float most = 0.f;
  for (int64_t r = threadIdx.x; r < a.rows; r += kScaleThreads) {
    float x = (a.g ? fabsf(a.g[r]) : 0.f) + (a.gh ? fabsf(a.gh[r]) * (1.f + log_v) : 0.f);
    if (a.gtop)
      for (int j = 0; j < a.top; ++j) x += fabsf(a.gtop[r * a.top + j]);
    x *= a.c;
    if (a.tok[r] != a.ignore && x < INFINITY) most = fmaxf(most, x);
  }
  most = group_max<64>(most);
  if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kScaleThreads / 64; ++w) most = fmaxf(most, wave_most[w]);
  int x = 14;
  if (most > 0.f) frexpf(most, &x);  // most <= 2^x
  const int e = max(-110, min(14 - x, 110));
  scale[0] = ldexpf(1.f, e);
  scale[1] = ldexpf(1.f, -e);
}

// 16-bit results of sums in fp32, times scale[1].
__global__ __launch_bounds__(kThreads) void unscale_kernel(const float* __restrict__ x, u16* __restrict__ y, int64_t n, const float* __restrict__ scale) {
  const float s = scale[1];
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) y[i] = from_f32<F16>(x[i] * s);
}

// 32 (fp32: 16) values a thread, all loads before the first use; bound by the logits' read and the gradient's write (2048 x 151936
// bf16: 1.24 GB in 260 us).  Rows left out are zeros, and nothing of them is read.
template <typename T, typename O, bool FAR> __global__ __launch_bounds__(kThreads) void grad_kernel(Bwd a, int slices) {
  typedef typename T::storage S;
  typedef typename O::storage SO;
  constexpr int V = T::vec, C = kGradVectors, N = kThreads * V * C;
  const int64_t r = blockIdx.x / (unsigned)slices;
  const int sl = (int)(blockIdx.x - (unsigned)(r * slices)), tid = threadIdx.x;
  const int64_t t = a.tok[r];
  const bool live = t != a.ignore;
  const S* row = (const S*)a.z + r * a.ld;
  SO* out = (SO*)a.dz + r * a.ldo;
  const int mis = (int)(((uintptr_t)out & (V * sizeof(SO) - 1)) / sizeof(SO));
  const int64_t base = (int64_t)sl * N - mis;
  const bool whole = base >= 0 && base + N <= a.vocab;
  i32x4 raw[C];
  if (live) {
    if (misaligned<T>(row) == mis) {
      load_slice<T, C>(raw, row, base, a.vocab);
    } else {  // the gradient's rows begin elsewhere between 16-byte boundaries
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t i0 = base + (i * kThreads + tid) * V;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t x = kLowest<T>;
#pragma unroll
          for (int e = 0; e < V / 4; ++e) {
            const int64_t j = i0 + w * (V / 4) + e;
            if (j < 0 || j >= a.vocab) continue;
            if constexpr (V == 4) x = __float_as_uint(row[j]);
            else x = (x & ~(0xffffu << (16 * e))) | ((uint32_t)row[j] << (16 * e));
          }
          raw[i][w] = (int)x;
        }
      }
    }
  }
  float m = 0.f, ls = 0.f, g = 0.f, gh = 0.f, ent = 0.f, all = 0.f;
  const float by = O::code == Q3_F16 && T::code == Q3_F32 ? scale_of(a) : 1.f;
  if (live) {
    m = a.m[r];
    ls = a.ls[r];
    ent = a.entropy[r];
    g = a.g ? (t >= 0 && t < a.vocab ? a.g[r] * by : NAN) : 0.f;
    gh = a.gh ? a.gh[r] * by : 0.f;
    all = g;
    if (a.gtop)
      for (int j = 0; j < a.top; ++j) all += a.gtop[r * a.top + j] * by;
  }
  const float c2 = a.c * kLog2e, l2 = ls * kLog2e;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int64_t i0 = base + (i * kThreads + tid) * V;
    float o[V];
    if (live) {
      const Vec<T> x = unpack_vec<T>(raw[i]);
      // -c p (all + h (log p + entropy)), log p = d c - ls
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = x.v[e] - m;
        const float p = __builtin_amdgcn_exp2f(fmaf(d, c2, -l2));
        const float lp = fmaxf(fmaf(d, a.c, -ls), kDeep);
        o[e] = -a.c * p * fmaf(gh, lp + ent, all);
      }
      // the given token, and the alternatives
      for (int j = -1; j < (a.gtop ? a.top : 0); ++j) {
        const int64_t at = (j < 0 ? t : a.top_token[r * a.top + j]) - i0;
        if (at < 0 || at >= V) continue;
        float mine = i0 + at == t ? g : 0.f;
        if (a.gtop)
          for (int k = 0; k < a.top; ++k) mine += a.top_token[r * a.top + k] == i0 + at ? a.gtop[r * a.top + k] * by : 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (e != at) continue;
          const float lp = fmaf(x.v[e] - m, a.c, -ls), p = __builtin_amdgcn_exp2f(fmaf(x.v[e] - m, c2, -l2));
          o[e] = a.c * (-expm1f(lp) * mine - p * fmaf(gh, fmaxf(lp, kDeep) + ent, all - mine));
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = 0.f;
    }
    if (whole || (i0 >= 0 && i0 + V <= a.vocab)) {
      store_values<O, V, FAR>(out + i0, o);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i0 + e >= 0 && i0 + e < a.vocab) out[i0 + e] = from_f32<O>(o[e]);
    }
  }
}

// ---------------------------------------------------------------- the LM head's rows
// Statistics of 128-column groups [group][ldp] from the LM head's product joined: R rows a workgroup, NT / R threads a row, each a
// fixed set of groups.  16 rows side by side read whole lines (4096 rows of 1187 groups: 58 MB in 25 us); up to 256 rows take a
// workgroup each, which reads a part of each line but spreads over the CUs (8 rows 6 us and 10, 256 8 and
// 10, 400 14 and 10).
struct Head {
  const float *m, *rest, *u, *pick;
  int64_t ldp;
  int groups;
};
template <int R, int NT> __global__ __launch_bounds__(NT) void head_finish_kernel(Head h, Fwd a) {
  constexpr int G = NT / R, W = NT / 64;
  __shared__ Part part[W][R];
  const int lr = threadIdx.x % R, sl = threadIdx.x / R, lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * R + lr, rc = min(r, a.rows - 1);
  const float c2 = a.c * kLog2e;
  Part p{-INFINITY, 0.f, 0.f};
  for (int i = sl; i < h.groups; i += 4 * G) {
    Part q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t at = (int64_t)min(i + k * G, h.groups - 1) * h.ldp + rc;
      q[k] = Part{h.m[at], h.rest[at], h.u[at]};
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k * G < h.groups) p = join(p, q[k], c2);
  }
#pragma unroll
  for (int o = R; o < 64; o <<= 1)
    p = join(p, Part{__shfl_xor(p.m, o, 64), __shfl_xor(p.rest, o, 64), __shfl_xor(p.u, o, 64)}, c2);
  if (lane < R) part[threadIdx.x >> 6][lr] = p;
  __syncthreads();
  if (sl != 0 || r >= a.rows) return;
  for (int k = 1; k < W; ++k) p = join(p, part[k][lr], c2);
  const int64_t t = a.tok[r];
  if (t == a.ignore) {
    left_out(a, r, 0);
    return;
  }
  const bool valid = t >= 0 && t < a.vocab;
  finish_row(a, r, p, valid ? h.pick[r] : 0.f, valid);
}

// dz from what the product left of the logits (their distances to their group's maximum), in its place or elsewhere: as grad_kernel, with
// log2 p = (c2 (m_group - M) - ls log2(e)) - distance; the given token's log p is the result itself.  Bound by z, read and written
// (4096 x 151936: 2.5 GB in 446 us, 5.6 TB/s).
template <typename O> __global__ __launch_bounds__(kThreads) void head_grad_kernel(Head h, Bwd a, const float* logprob, int slices) {
  constexpr int C = kGradVectors, N = kThreads * 8 * C;
  const int64_t r = blockIdx.x / (unsigned)slices;
  const int base = (int)(blockIdx.x - (unsigned)(r * slices)) * N + (int)threadIdx.x * 8, vocab = (int)a.vocab;
  const int64_t t = a.tok[r];
  const u16* row = (const u16*)a.z + r * a.ld;
  u16* out = (u16*)a.dz + r * a.ldo;
  const bool live = t != a.ignore;
  i32x4 raw[C];
  float gm[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int i0 = base + i * (kThreads * 8);
    if (live && i0 < vocab) {
      raw[i] = *reinterpret_cast<const i32x4*>(row + i0);
      gm[i] = h.m[(int64_t)(i0 >> 7) * h.ldp + r];
    }
  }
  float m = 0.f, ls = 0.f, g = 0.f, gh = 0.f, ent = 0.f, tlp = 0.f;
  if (live) {
    m = a.m[r];
    ls = a.ls[r];
    ent = a.entropy[r];
    tlp = logprob[r];
    const float by = O::code == Q3_F16 ? scale_of(a) : 1.f;
    g = a.g ? (t >= 0 && t < vocab ? a.g[r] * by : NAN) : 0.f;
    gh = a.gh ? a.gh[r] * by : 0.f;
  }
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int i0 = base + i * (kThreads * 8);
    if (i0 >= vocab) continue;
    float o[8];
    if (live) {
      float at = fmaf(gm[i] - m, a.c, -ls) * kLog2e;
      at = at < kDeep ? kDeep : at;  // a group of -inf only too
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t gap = ((uint32_t)raw[i][e >> 1] >> (16 * (e & 1))) & 0xffffu;
        const float l2 = fmaf((float)gap, -kGapStep, at), p = gap == 0xffffu ? 0.f : __builtin_amdgcn_exp2f(l2);
        o[e] = -a.c * p * fmaf(gh, fmaf(l2, kLn2, ent), g);
      }
      const int64_t mine = t - i0;
      if (mine >= 0 && mine < 8) {
        const float p = __builtin_amdgcn_exp2f(tlp * kLog2e);
        const float v = a.c * (-expm1f(tlp) * g - p * gh * (fmaxf(tlp, kDeep) + ent));
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e == mine) o[e] = v;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = 0.f;
    }
    store_values<O, 8, false>(out + i0, o);
  }
}

// ---------------------------------------------------------------- host
bool dtype_ok(int dt) { return dt == Q3_F32 || dt == Q3_F16 || dt == Q3_BF16; }
int vec_of(int dtype) { return dtype == Q3_F32 ? 4 : 8; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of up to 4 slices of 4 vectors a thread take a workgroup each and no second launch, however few they are (20 of one
// row of 5000 9.0 us and 13.3 in two launches, of 32000 12.4 and 13.6, 10 of 256 rows of 32000 12.2 and 16.8; 500 rows of 5000 without
// alternatives 6.1 and 9.3, one of 32000 7.3 and 7.1).
bool one_launch(int dtype, int64_t vocab) { return vocab + vec_of(dtype) - 1 <= 4 * kThreads * vec_of(dtype) * 4; }
// Vectors of a slice per thread: 4 where that leaves 1024 workgroups (or a row has very many values), else 1, which spreads the search
// for alternatives (rows of 151936, 20 of one row 14.5 us and 17.1 with 4, 5 of 64 rows 25.8 and 22.3).  Without alternatives the
// rule is the same, for the same bits with and without (one row 8.1 us and 7.6 with 4, 64 rows 13.7 and 10.7).
int chunks_for(int dtype, int64_t rows, int64_t vocab) {
  return one_launch(dtype, vocab) || vocab > (1 << 18) || rows * cdiv(vocab, (int64_t)kThreads * vec_of(dtype) * 4) >= 1024 ? 4 : 1;
}
// A row may start up to a vector before its first element's boundary.
int64_t slices_for(int dtype, int64_t rows, int64_t vocab) {
  return cdiv(vocab + vec_of(dtype) - 1, (int64_t)kThreads * vec_of(dtype) * chunks_for(dtype, rows, vocab));
}
bool sizes_ok(int dtype, int64_t rows, int64_t vocab, int64_t top) {
  if (!dtype_ok(dtype) || rows < 1 || vocab < 1 || vocab >= (1ll << 30) || top < 0 || top > kMaxTop || top > vocab) return false;
  if (rows >= (1ll << 31)) return false;
  return rows * cdiv(vocab + 16, kThreads * vec_of(dtype)) < (1ll << 31) - 1;
}

// Slices of a workgroup, dealt out evenly.  Without alternatives as many as leave 4096 workgroups (rows of 151936 bf16: 4096 of them 206
// us, 229 with one slice each, 2048 108).  With them as many as leave 2048, at most 6, since each workgroup ends with a search (5 of
// 777 rows 59 us, leaving 4096 66; 20 of 300 41 and 54; 5 of 777 fp32 rows 89, with up to 13 slices 93).
int per_for(int dtype, int64_t rows, int64_t vocab, int64_t slices, int64_t top) {
  if (one_launch(dtype, vocab)) return (int)slices;
  const int64_t most = top > 0 ? std::min<int64_t>(std::min<int64_t>(slices, 6), rows * slices / 2048) : std::min(slices, rows * slices / 4096);
  return (int)cdiv(slices, cdiv(slices, std::max<int64_t>(1, most)));
}

// Whether each workgroup has a whole row, whose results it writes itself.
bool writes_results(int dtype, int64_t rows, int64_t vocab, int64_t slices, int64_t top) {
  return chunks_for(dtype, rows, vocab) == 4 && per_for(dtype, rows, vocab, slices, top) >= slices;
}

template <typename T, int C, bool ONE> void slices(const Fwd& a, hipStream_t s) {
  const unsigned n = (unsigned)(a.rows * a.parts);
  if (a.top) slice_kernel<T, C, true, ONE><<<n, kThreads, 0, s>>>(a);
  else slice_kernel<T, C, false, ONE><<<n, kThreads, 0, s>>>(a);
}

template <typename T> int forward(const Fwd& a, int chunks, hipStream_t s) {
  const bool one = chunks == 4 && a.parts == 1;  // as writes_results
  if (one) slices<T, 4, true>(a, s);
  else if (chunks == 4) slices<T, 4, false>(a, s);
  else slices<T, 1, false>(a, s);
  const int rc = (int)hipGetLastError();
  if (rc != 0) return rc;
  if (one) return rc;
  if (a.top) {
    finish_top_kernel<T><<<(unsigned)a.rows, kThreads, 0, s>>>(a);
  } else {
    finish_kernel<T><<<(unsigned)cdiv(a.rows, kThreads / 64), kThreads, 0, s>>>(a);
  }
  return (int)hipGetLastError();
}

template <typename T, typename O> int backward(const Bwd& a, hipStream_t s) {
  const int64_t n = cdiv(a.vocab + T::vec - 1, (int64_t)kThreads * T::vec * kGradVectors);
  // A gradient of more than 256 MiB does not pass through the caches (2048 x 151936 bf16 276 us and 288 through them, 777 fp32 157 and
  // 170); a smaller one is there for who reads it next.
  if (a.rows * a.vocab * (int64_t)sizeof(typename O::storage) > (256 << 20))
    grad_kernel<T, O, true><<<(unsigned)(a.rows * n), kThreads, 0, s>>>(a, (int)n);
  else
    grad_kernel<T, O, false><<<(unsigned)(a.rows * n), kThreads, 0, s>>>(a, (int)n);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t q3_token_logprobs_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int64_t top) {
  if (!sizes_ok(dtype, rows, vocab, top)) return 0;
  const int64_t slices = slices_for(dtype, rows, vocab);
  if (writes_results(dtype, rows, vocab, slices, top)) return 0;
  const size_t n = (size_t)rows * (size_t)slices;
  return (n * sizeof(Part) + 7) / 8 * 8 + n * (size_t)top * sizeof(uint64_t);
}

int q3_token_logprobs(int dtype, const void* z, int64_t ld, int64_t rows, int64_t vocab, const int64_t* tokens,
                      int64_t ignore_index, float inv_temperature, int64_t top, float* logprob, float* entropy, float* row_max,
                      float* row_log, float* top_logprob, int64_t* top_token, void* workspace, size_t workspace_bytes,
                      hipStream_t stream) {
  Q3_REQUIRE(sizes_ok(dtype, rows, vocab, top) && z && tokens && logprob && entropy && !row_max == !row_log && ld >= vocab);
  Q3_REQUIRE((top == 0 || (top_logprob && top_token)) && inv_temperature > 0.f && inv_temperature < INFINITY);
  const size_t need = q3_token_logprobs_workspace_bytes(dtype, rows, vocab, top);
  Q3_REQUIRE(((uintptr_t)z & (dtype == Q3_F32 ? 3 : 1)) == 0 &&
             (need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need)));
  const int n = (int)slices_for(dtype, rows, vocab), per = per_for(dtype, rows, vocab, n, top), c = chunks_for(dtype, rows, vocab), v = vec_of(dtype);
  // one vector a thread: slices of a size (a short last one would have many candidates for its alternatives: T = 1, top 20
  // 19 -> 9 us)
  const int span = c == 1 ? (int)cdiv(cdiv(vocab + v - 1, v), n) * v : kThreads * v * c;
  Fwd a{z, ld, rows, vocab, tokens, ignore_index, inv_temperature, (int)top, n, span, per, (int)cdiv(n, per),
        (Part*)workspace, nullptr, logprob, entropy, row_max, row_log, top_logprob, top_token};
  if (need > 0) a.key = (uint64_t*)((char*)workspace + ((size_t)rows * n * sizeof(Part) + 7) / 8 * 8);
  if (dtype == Q3_BF16) return forward<BF16>(a, c, stream);
  if (dtype == Q3_F16) return forward<F16>(a, c, stream);
  return forward<F32>(a, c, stream);
}

int q3_token_logprobs_bwd_scaled(int dtype, int out_dtype, const void* z, int64_t ld, int64_t rows, int64_t vocab, const int64_t* tokens,
                                 int64_t ignore_index, float inv_temperature, int64_t top, const int64_t* top_token,
                                 const float* row_max, const float* row_log, const float* entropy, const float* g, const float* gh,
                                 const float* gtop, void* dz, int64_t ldo, const float* scale,
                                 hipStream_t stream) {
  Q3_REQUIRE(sizes_ok(dtype, rows, vocab, top) && z && tokens && row_max && row_log && entropy && dz && ld >= vocab &&
             ldo >= vocab && (!gtop || (top > 0 && top_token)) && inv_temperature > 0.f && inv_temperature < INFINITY);
  Q3_REQUIRE(!scale || (dtype == Q3_F32 && out_dtype == Q3_F16 && ((uintptr_t)scale & 3) == 0));
  Q3_REQUIRE(out_dtype == dtype || (dtype == Q3_F32 && dtype_ok(out_dtype)));
  Q3_REQUIRE(((uintptr_t)z & (dtype == Q3_F32 ? 3 : 1)) == 0 && ((uintptr_t)dz & (out_dtype == Q3_F32 ? 3 : 1)) == 0 && dz != z);
  const Bwd a{z, ld, rows, vocab, tokens, ignore_index, inv_temperature, (int)top, top_token, row_max, row_log, entropy, g, gh,
              gtop, dz, ldo, scale};
  if (dtype == Q3_BF16) return backward<BF16, BF16>(a, stream);
  if (dtype == Q3_F16) return backward<F16, F16>(a, stream);
  if (out_dtype == Q3_BF16) return backward<F32, BF16>(a, stream);
  if (out_dtype == Q3_F16) return backward<F32, F16>(a, stream);
  return backward<F32, F32>(a, stream);
}

int q3_token_logprobs_bwd(int dtype, int out_dtype, const void* z, int64_t ld, int64_t rows, int64_t vocab, const int64_t* tokens,
                          int64_t ignore_index, float inv_temperature, int64_t top, const int64_t* top_token,
                          const float* row_max, const float* row_log, const float* entropy, const float* g, const float* gh,
                          const float* gtop, void* dz, int64_t ldo, hipStream_t stream) {
  return q3_token_logprobs_bwd_scaled(dtype, out_dtype, z, ld, rows, vocab, tokens, ignore_index, inv_temperature, top, top_token,
                                      row_max, row_log, entropy, g, gh, gtop, dz, ldo, nullptr, stream);
}

int q3_logprobs_grad_scale(const float* g, const float* gh, const float* gtop, int64_t rows, int64_t vocab, int64_t top,
                           const int64_t* tokens, int64_t ignore_index, float inv_temperature, float* scale, hipStream_t stream) {
  Q3_REQUIRE(rows > 0 && rows < (1ll << 31) && vocab > 0 && vocab < (1ll << 30) && top >= 0 && top <= kMaxTop && tokens && scale &&
             ((uintptr_t)scale & 3) == 0 && (!gtop || top > 0) && inv_temperature > 0.f && inv_temperature < INFINITY);
  Bwd a{};
  a.rows = rows;
  a.tok = tokens;
  a.ignore = ignore_index;
  a.c = inv_temperature;
  a.top = (int)top;
  a.g = g;
  a.gh = gh;
  a.gtop = gtop;
  scale_kernel<<<1, kScaleThreads, 0, stream>>>(a, logf((float)vocab), scale);
  return (int)hipGetLastError();
}

int q3_unscale_f16(const float* x, void* y, int64_t n, const float* scale, hipStream_t stream) {
  Q3_REQUIRE(x && y && scale && n > 0 && ((uintptr_t)x & 3) == 0 && ((uintptr_t)y & 1) == 0 && ((uintptr_t)scale & 3) == 0);
  unscale_kernel<<<(unsigned)std::min<int64_t>(cdiv(n, kThreads), 4096), kThreads, 0, stream>>>(x, (u16*)y, n, scale);
  return (int)hipGetLastError();
}

int q3_head_logprobs_finish(const float* m_part, const float* rest_part, const float* u_part, int64_t ldp, const float* pick,
                            int64_t rows, int64_t vocab, const int64_t* tokens, int64_t ignore_index, float inv_temperature,
                            float* logprob, float* entropy, float* row_max, float* row_log, hipStream_t stream) {
  Q3_REQUIRE(m_part && rest_part && u_part && pick && tokens && logprob && entropy && row_max && row_log && rows > 0 &&
             rows < (1ll << 31) && vocab > 0 && vocab < (1ll << 30) && ldp >= rows && inv_temperature > 0.f && inv_temperature < INFINITY);
  Fwd a{};
  a.rows = rows;
  a.vocab = vocab;
  a.tok = tokens;
  a.ignore = ignore_index;
  a.c = inv_temperature;
  a.logprob = logprob;
  a.entropy = entropy;
  a.m = row_max;
  a.ls = row_log;
  const Head h{m_part, rest_part, u_part, pick, ldp, (int)cdiv(vocab, 128)};
  if (rows <= 256) head_finish_kernel<1, 256><<<(unsigned)rows, 256, 0, stream>>>(h, a);
  else head_finish_kernel<16, 1024><<<(unsigned)cdiv(rows, 16), 1024, 0, stream>>>(h, a);
  return (int)hipGetLastError();
}

int q3_head_logprobs_grad(int dtype, const void* z, int64_t ldz, void* dz, int64_t ldo, int64_t rows, int64_t vocab, const int64_t* tokens,
                          int64_t ignore_index, float inv_temperature, const float* m_part, int64_t ldp, const float* row_max,
                          const float* row_log, const float* logprob, const float* entropy, const float* g, const float* gh,
                          const float* scale, hipStream_t stream) {
  Q3_REQUIRE((dtype == Q3_BF16 || dtype == Q3_F16) && z && ((uintptr_t)z & 15) == 0 && vocab > 0 && vocab < (1ll << 30) - (1 << 16) &&
             vocab % 8 == 0 && ldz >= vocab && ldz % 8 == 0 && rows > 0 && rows < (1ll << 31) && ldp >= rows && tokens && m_part &&
             row_max && row_log && logprob && entropy && inv_temperature > 0.f && inv_temperature < INFINITY);
  Q3_REQUIRE(dz && ((uintptr_t)dz & 15) == 0 && ldo >= vocab && ldo % 8 == 0 && (dz != z || ldo == ldz));
  Q3_REQUIRE(!scale || (dtype == Q3_F16 && ((uintptr_t)scale & 3) == 0));
  const int64_t n = cdiv(vocab, (int64_t)kThreads * 8 * kGradVectors);
  Q3_REQUIRE(rows * n < (1ll << 31));
  const Bwd a{z, ldz, rows, vocab, tokens, ignore_index, inv_temperature, 0, nullptr, row_max, row_log, entropy, g, gh, nullptr, dz, ldo, scale};
  const Head h{m_part, nullptr, nullptr, nullptr, ldp, 0};
  if (dtype == Q3_BF16) head_grad_kernel<BF16><<<(unsigned)(rows * n), kThreads, 0, stream>>>(h, a, logprob, (int)n);
  else head_grad_kernel<F16><<<(unsigned)(rows * n), kThreads, 0, stream>>>(h, a, logprob, (int)n);
  return (int)hipGetLastError();
}

int q3_head_logprobs_bwd(int dtype, void* z, int64_t ldz, int64_t rows, int64_t vocab, const int64_t* tokens, int64_t ignore_index,
                         float inv_temperature, const float* m_part, int64_t ldp, const float* row_max, const float* row_log,
                         const float* logprob, const float* entropy, const float* g, const float* gh, hipStream_t stream) {
  return q3_head_logprobs_grad(dtype, z, ldz, z, ldz, rows, vocab, tokens, ignore_index, inv_temperature, m_part, ldp, row_max, row_log,
                               logprob, entropy, g, gh, nullptr, stream);
}

}  // extern "C"
