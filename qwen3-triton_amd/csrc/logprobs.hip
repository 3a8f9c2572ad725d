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
// registers: the slice's maximum, then the sums, then the alternatives are taken from them.  Many rows take slices of 64 values a
// thread; few rows small ones, so that one row's latency is spread over many CUs.  A second launch joins a row's slices.
#include <type_traits>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f;

// Statistics of a part of a row.  m = -inf: nothing but -inf there (rest 0, or NaN where there is a NaN too).
struct Part {
  float m, rest, u;
};
Q3_DEV float part_total(const Part& a) { return a.m == -INFINITY ? a.rest : 1.f + a.rest; }
// c2 = c log2(e)
Q3_DEV Part join(const Part& a, const Part& b, float c2) {
  const bool first = a.m >= b.m;
  const Part &hi = first ? a : b, &lo = first ? b : a;
  if (lo.m == -INFINITY) return Part{hi.m, hi.rest + lo.rest, hi.u};
  const float d = lo.m - hi.m, w = __builtin_amdgcn_exp2f(d * c2), t = 1.f + lo.rest;
  return Part{hi.m, fmaf(t, w, hi.rest), fmaf(w, fmaf(t, fmaxf(d, -1e30f), lo.u), hi.u)};
}

// ---------------------------------------------------------------- the largest k
// Values as whole numbers in their order, NaN above all, the lower index first among equals.  A slice of 16-bit values fits
// value and place into 32 bits; otherwise 64.
Q3_DEV uint32_t order32(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as +0
  return x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
Q3_DEV float unorder32(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
template <typename T> Q3_DEV uint32_t order16(float x) {  // of a value of a 16-bit type
  const uint32_t h = from_f32<T>(x + 0.f);
  return x != x ? 0xffffu : (h & 0x8000u) ? (~h & 0xffffu) : (h | 0x8000u);
}
Q3_DEV uint64_t key64(float x, uint32_t index) { return ((uint64_t)order32(x) << 32) | (uint32_t)~index; }

template <typename K> Q3_DEV K shfl_key(K x, int mask) {
  if constexpr (sizeof(K) == 4) return (K)__shfl_xor((int)x, mask, 64);
  else return ((K)(uint32_t)__shfl_xor((int)(uint32_t)(x >> 32), mask, 64) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)x, mask, 64);
}

// The k largest of a workgroup's keys (all different; 0: none), in order, to emit(rank, key) by some thread each; ranks that no
// key takes get 0.  `each(f)` calls f with every key of the calling thread.
//  * The 64 maxima of groups of 4 threads: the k-th largest of those is a bound that at least k keys reach (k <= 64), and only
//    keys of k groups do, so what passes it fits `cand` (k x 4 threads' keys), whatever the data.
//  * What passes is ranked by counting the larger ones.
template <typename K> struct TopScratch {
  alignas(16) K group[64];
  K bound;
  int count;
};
template <typename K, typename Each, typename Emit>
Q3_DEV void block_top(TopScratch<K>& sc, K* cand, int k, Each&& each, Emit&& emit) {
  const int tid = threadIdx.x;
  K best = 0;
  each([&](K x) { best = x > best ? x : best; });
  K g = best;
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    const K y = shfl_key(g, o);
    g = y > g ? y : g;
  }
  if ((tid & 3) == 0) sc.group[tid >> 2] = g;
  if (tid == 0) sc.count = 0;
  __syncthreads();
  if (tid < 64) {
    const K mine = sc.group[tid];
    int larger = 0;
#pragma unroll 8
    for (int i = 0; i < 64; ++i) {
      const K o = sc.group[i];
      larger += (o > mine || (o == mine && i < tid)) ? 1 : 0;  // equal ones are all 0: no key
    }
    if (larger == k - 1) sc.bound = mine;
  }
  __syncthreads();
  const K bound = sc.bound;
  if (best >= bound && best != 0)
    each([&](K x) {
      if (x >= bound && x != 0) cand[atomicAdd(&sc.count, 1)] = x;
    });
  __syncthreads();
  const int n = sc.count;
  for (int i = tid; i < n; i += kThreads) {
    const K mine = cand[i];
    int larger = 0;
    for (int j = 0; j < n; ++j) larger += cand[j] > mine ? 1 : 0;
    if (larger < k) emit(larger, mine);
  }
  for (int r = n + tid; r < k; r += kThreads) emit(r, (K)0);
}

// ---------------------------------------------------------------- one slice of a row
struct Fwd {
  const void* z;
  int64_t ld, rows, vocab;
  const int64_t* tok;
  int64_t ignore;
  float c;      // 1 / temperature
  int top, slices;
  Part* part;   // [rows][slices]
  uint64_t* key;  // [rows][slices][top]
  float *logprob, *entropy, *m, *ls;  // ls: log1p(rest)
  float* top_logprob;
  int64_t* top_token;
};

// 16 bytes from element i0 of a row of n on, whatever the row's alignment: i0 counts from a 16-byte boundary at or before the
// row, so only a row's first and last vectors are not whole; elements outside the row are -inf.
template <typename T> Q3_DEV Vec<T> load_edge(const typename T::storage* row, int64_t i0, int64_t n) {
  if (i0 >= 0 && i0 + T::vec <= n) return load_vec<T>(row + i0);
  Vec<T> v;
#pragma unroll
  for (int e = 0; e < T::vec; ++e) v.v[e] = i0 + e >= 0 && i0 + e < n ? to_f32<T>(row[i0 + e]) : -INFINITY;
  return v;
}
// Elements between the 16-byte boundary before a row and its start.
template <typename T> Q3_DEV int misaligned(const typename T::storage* row) {
  return (int)(((uintptr_t)row & 15) / sizeof(typename T::storage));
}

template <typename T, int C, bool TOP>
__global__ __launch_bounds__(kThreads) void slice_kernel(Fwd a) {
  typedef typename T::storage S;
  constexpr int V = T::vec, N = kThreads * V * C;
  typedef typename std::conditional<V == 8, uint32_t, uint64_t>::type K;
  const int64_t r = blockIdx.x / a.slices;
  const int sl = (int)(blockIdx.x - r * a.slices), tid = threadIdx.x;
  if (a.tok[r] == a.ignore) return;  // the whole workgroup: nothing of the row is read
  const S* row = (const S*)a.z + r * a.ld;
  const int64_t base = (int64_t)sl * N - misaligned<T>(row);
  Vec<T> x[C];
#pragma unroll
  for (int i = 0; i < C; ++i) x[i] = load_edge<T>(row, base + (int64_t)(i * kThreads + tid) * V, a.vocab);

  Part p{-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) p.m = fmaxf(p.m, x[i].v[e]);
  const float c2 = a.c * kLog2e;
  {
    const float ref = p.m == -INFINITY ? 0.f : p.m;  // only -inf (e^d = 0) and NaN then
    int same = 0;
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = x[i].v[e] - ref;
        const bool top = d == 0.f;
        const float w = top ? 0.f : __builtin_amdgcn_exp2f(d * c2);
        same += top ? 1 : 0;
        p.rest += w;
        p.u = fmaf(w, fmaxf(d, -1e30f), p.u);
      }
    if (p.m != -INFINITY) p.rest += (float)(same - 1);
    if (p.m == INFINITY) p.rest = NAN;  // inf - inf
  }
  // over the wave: one lane that holds the maximum gives its rest, the others their totals
  const float wm = group_max<64>(p.m);
  {
    const uint64_t at = __ballot(p.m == wm);
    const bool one = (threadIdx.x & 63) == (unsigned)__builtin_ctzll(at | (1ull << 63));
    const float d = p.m - wm, w = p.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(d * c2);
    const float t = one ? p.rest : part_total(p);
    const float full = part_total(p);
    p.u = group_sum<64>(p.m == -INFINITY ? 0.f : w * fmaf(full, fmaxf(d, -1e30f), p.u));
    p.rest = group_sum<64>(t * w);
    p.m = wm;
  }
  __shared__ Part wave_part[kThreads / 64];
  if ((tid & 63) == 0) wave_part[tid >> 6] = p;
  __syncthreads();
  if (tid == 0) {
    p = wave_part[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) p = join(p, wave_part[w], c2);
    a.part[r * a.slices + sl] = p;
  }
  if constexpr (TOP) {
    __shared__ TopScratch<K> sc;
    extern __shared__ uint64_t cand_mem[];  // top x 4 threads' keys
    K* cand = (K*)cand_mem;
    uint64_t* out = a.key + (r * a.slices + sl) * a.top;
    auto each = [&](auto&& f) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int at = (i * kThreads + tid) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int64_t j = base + at + e;
          const bool in = j >= 0 && j < a.vocab;
          if constexpr (V == 8) {
            const uint32_t k = (order16<T>(x[i].v[e]) << 16) | (uint32_t)(0xffff - (at + e));
            f(in ? k : 0u);
          } else {
            f(in ? key64(x[i].v[e], (uint32_t)j) : (uint64_t)0);
          }
        }
      }
    };
    block_top<K>(sc, cand, a.top, each, [&](int rank, K k) {
      if constexpr (V == 8) {
        const int64_t j = base + (0xffff - (int)(k & 0xffffu));
        out[rank] = k == 0 ? 0 : key64(to_f32<T>(row[j]), (uint32_t)j);
      } else {
        out[rank] = k;
      }
    });
  }
}

// ---------------------------------------------------------------- a row's slices joined
Q3_DEV void finish_row(const Fwd& a, int64_t r, const Part& p, float picked, bool valid) {
  const float ls = log1pf(p.rest), d = picked - p.m;
  const bool none = p.m == -INFINITY;
  a.logprob[r] = valid ? fmaf(d, a.c, -ls) : NAN;
  a.entropy[r] = none ? NAN : fmaf(-a.c, p.u / (1.f + p.rest), ls);
  a.m[r] = p.m;
  a.ls[r] = none ? NAN : ls;
}

Q3_DEV void left_out(const Fwd& a, int64_t r) {
  a.logprob[r] = a.entropy[r] = a.m[r] = a.ls[r] = 0.f;
}

// One wave a row, no alternatives.
template <typename T> __global__ __launch_bounds__(kThreads) void finish_kernel(Fwd a) {
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (r >= a.rows) return;
  const int64_t t = a.tok[r];
  if (t == a.ignore) {
    if (lane == 0) left_out(a, r);
    return;
  }
  const bool valid = t >= 0 && t < a.vocab;
  const float picked = valid ? to_f32<T>(((const typename T::storage*)a.z)[r * a.ld + t]) : 0.f;
  const float c2 = a.c * kLog2e;
  Part p{-INFINITY, 0.f, 0.f};
  for (int i = lane; i < a.slices; i += 64) p = join(p, a.part[r * a.slices + i], c2);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
    p = join(p, Part{__shfl_xor(p.m, o, 64), __shfl_xor(p.rest, o, 64), __shfl_xor(p.u, o, 64)}, c2);
  if (lane == 0) finish_row(a, r, p, picked, valid);
}

// One workgroup a row: the alternatives are the largest of its slices' largest.
template <typename T> __global__ __launch_bounds__(kThreads) void finish_top_kernel(Fwd a) {
  __shared__ TopScratch<uint64_t> sc;
  extern __shared__ uint64_t cand_mem[];
  uint64_t* cand = cand_mem;
  __shared__ Part row_part;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t t = a.tok[r];
  if (t == a.ignore) {
    if (tid == 0) left_out(a, r);
    if (tid < a.top) {
      a.top_logprob[r * a.top + tid] = 0.f;
      a.top_token[r * a.top + tid] = 0;
    }
    return;
  }
  if (tid < 64) {
    const bool valid = t >= 0 && t < a.vocab;
    const float picked = valid ? to_f32<T>(((const typename T::storage*)a.z)[r * a.ld + t]) : 0.f;
    const float c2 = a.c * kLog2e;
    Part p{-INFINITY, 0.f, 0.f};
    for (int i = tid; i < a.slices; i += 64) p = join(p, a.part[r * a.slices + i], c2);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
      p = join(p, Part{__shfl_xor(p.m, o, 64), __shfl_xor(p.rest, o, 64), __shfl_xor(p.u, o, 64)}, c2);
    if (tid == 0) {
      finish_row(a, r, p, picked, valid);
      row_part = p;
    }
  }
  const uint64_t* key = a.key + r * a.slices * a.top;
  const int n = a.slices * a.top;
  block_top<uint64_t>(sc, cand, a.top, [&](auto&& f) {
    for (int i = tid; i < n; i += kThreads) f(key[i]);
  }, [&](int rank, uint64_t k) {  // behind barriers: row_part is there
    a.top_token[r * a.top + rank] = (int64_t)(uint32_t)~(uint32_t)k;
    const uint32_t o = (uint32_t)(k >> 32);
    const float x = o == 0xffffffffu ? NAN : unorder32(o);
    a.top_logprob[r * a.top + rank] = row_part.m == -INFINITY ? NAN : fmaf(x - row_part.m, a.c, -log1pf(row_part.rest));
  });
}

// ---------------------------------------------------------------- gradient
// N values as one store of N elements.
template <typename O, int N> Q3_DEV void store_values(typename O::storage* p, const float (&v)[N]) {
  if constexpr (N == O::vec) {
    Vec<O> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = v[e];
    store_vec<O>(p, o);
  } else {
    static_assert(N == 4 && O::vec == 8, "fp32 logits, 16-bit gradient");
    *reinterpret_cast<i32x2*>(p) = i32x2{(int)pack2<O>(v[0], v[1]), (int)pack2<O>(v[2], v[3])};
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
};

// 16 values a thread, in vectors of 16 bytes of logits.  Rows left out are zeros, and nothing of them is read.
template <typename T, typename O> __global__ __launch_bounds__(kThreads) void grad_kernel(Bwd a, int slices) {
  typedef typename T::storage S;
  typedef typename O::storage SO;
  constexpr int V = T::vec, C = 16 / V;
  const int64_t r = blockIdx.x / slices;
  const int sl = (int)(blockIdx.x - r * slices), tid = threadIdx.x;
  const int64_t t = a.tok[r];
  const bool live = t != a.ignore;
  const S* row = (const S*)a.z + r * a.ld;
  SO* out = (SO*)a.dz + r * a.ldo;
  const int mis = (int)(((uintptr_t)out & (V * sizeof(SO) - 1)) / sizeof(SO));
  const bool same = misaligned<T>(row) == mis;
  const int64_t base = (int64_t)sl * (kThreads * V * C) - mis;
  Vec<T> x[C];
  if (live) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int64_t i0 = base + (int64_t)(i * kThreads + tid) * V;
      if (same) {
        x[i] = load_edge<T>(row, i0, a.vocab);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[i].v[e] = i0 + e >= 0 && i0 + e < a.vocab ? to_f32<T>(row[i0 + e]) : -INFINITY;
      }
    }
  }
  float m = 0.f, ls = 0.f, g = 0.f, gh = 0.f, ent = 0.f, all = 0.f;
  if (live) {
    m = a.m[r];
    ls = a.ls[r];
    ent = a.entropy[r];
    g = a.g ? (t >= 0 && t < a.vocab ? a.g[r] : NAN) : 0.f;
    gh = a.gh ? a.gh[r] : 0.f;
    all = g;
    if (a.gtop)
      for (int j = 0; j < a.top; ++j) all += a.gtop[r * a.top + j];
  }
  const float c2 = a.c * kLog2e, l2 = ls * kLog2e;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int64_t i0 = base + (int64_t)(i * kThreads + tid) * V;
    if (i0 + V <= 0 || i0 >= a.vocab) continue;
    struct { float v[V]; } o;
    if (live) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = x[i].v[e] - m;
        const float p = __builtin_amdgcn_exp2f(fmaf(d, c2, -l2));
        const float lp = fmaxf(fmaf(d, a.c, -ls), -1e30f);
        o.v[e] = -a.c * p * fmaf(gh, lp + ent, all);
      }
      // the given token, and the alternatives
      for (int j = -1; j < (a.gtop ? a.top : 0); ++j) {
        const int64_t at = (j < 0 ? t : a.top_token[r * a.top + j]) - i0;
        if (at < 0 || at >= V) continue;
        float mine = i0 + at == t ? g : 0.f;
        if (a.gtop)
          for (int k = 0; k < a.top; ++k) mine += a.top_token[r * a.top + k] == i0 + at ? a.gtop[r * a.top + k] : 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (e != at) continue;
          const float lp = fmaf(x[i].v[e] - m, a.c, -ls), p = __builtin_amdgcn_exp2f(fmaf(x[i].v[e] - m, c2, -l2));
          o.v[e] = a.c * (-expm1f(lp) * mine - p * fmaf(gh, fmaxf(lp, -1e30f) + ent, all - mine));
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) o.v[e] = 0.f;
    }
    if (i0 >= 0 && i0 + V <= a.vocab) {
      store_values<O, V>(out + i0, o.v);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i0 + e >= 0 && i0 + e < a.vocab) out[i0 + e] = from_f32<O>(o.v[e]);
    }
  }
}

// ---------------------------------------------------------------- host
bool dtype_ok(int dt) { return dt == Q3_F32 || dt == Q3_F16 || dt == Q3_BF16; }
int vec_of(int dtype) { return dtype == Q3_F32 ? 4 : 8; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Vectors of a slice per thread: 8 where that leaves enough workgroups for the chip (or a row has very many values), else 1.
int chunks_for(int dtype, int64_t rows, int64_t vocab) {
  return vocab > (1 << 18) || rows * cdiv(vocab, (int64_t)kThreads * vec_of(dtype) * 8) >= 1024 ? 8 : 1;
}
// A row may start up to a vector before its first element's boundary.
int64_t slices_for(int dtype, int64_t rows, int64_t vocab) {
  return cdiv(vocab + vec_of(dtype) - 1, (int64_t)kThreads * vec_of(dtype) * chunks_for(dtype, rows, vocab));
}
bool sizes_ok(int dtype, int64_t rows, int64_t vocab, int64_t top) {
  if (!dtype_ok(dtype) || rows < 1 || vocab < 1 || vocab >= (1ll << 30) || top < 0 || top > kMaxTop || top > vocab) return false;
  if (rows >= (1ll << 31) || (top > 0 && vocab > (1 << 21))) return false;
  return rows * cdiv(vocab + 16, kThreads * vec_of(dtype)) < (1ll << 31) - 1;
}

template <typename T, int C> void slices(const Fwd& a, hipStream_t s) {
  const unsigned n = (unsigned)(a.rows * a.slices);
  const size_t lds = (size_t)a.top * 4 * C * T::vec * (T::vec == 8 ? 4 : 8);
  if (a.top) slice_kernel<T, C, true><<<n, kThreads, lds, s>>>(a);
  else slice_kernel<T, C, false><<<n, kThreads, 0, s>>>(a);
}

template <typename T> int forward(const Fwd& a, int chunks, hipStream_t s) {
  if (chunks == 8) slices<T, 8>(a, s);
  else slices<T, 1>(a, s);
  const int rc = (int)hipGetLastError();
  if (rc != 0) return rc;
  if (a.top) {
    // a thread of the joining workgroup takes its share of the slices' keys: at most 64 of them (2^21 values of 8192 a slice)
    const size_t lds = (size_t)a.top * 4 * (size_t)cdiv((int64_t)a.slices * a.top, kThreads) * sizeof(uint64_t);
    finish_top_kernel<T><<<(unsigned)a.rows, kThreads, lds, s>>>(a);
  } else {
    finish_kernel<T><<<(unsigned)cdiv(a.rows, kThreads / 64), kThreads, 0, s>>>(a);
  }
  return (int)hipGetLastError();
}

template <typename T, typename O> int backward(const Bwd& a, hipStream_t s) {
  const int64_t n = cdiv(a.vocab + T::vec - 1, kThreads * 16);
  grad_kernel<T, O><<<(unsigned)(a.rows * n), kThreads, 0, s>>>(a, (int)n);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t q3_token_logprobs_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int64_t top) {
  if (!sizes_ok(dtype, rows, vocab, top)) return 0;
  const size_t n = (size_t)rows * (size_t)slices_for(dtype, rows, vocab);
  return (n * sizeof(Part) + 7) / 8 * 8 + n * (size_t)top * sizeof(uint64_t);
}

int q3_token_logprobs(int dtype, const void* z, int64_t ld, int64_t rows, int64_t vocab, const int64_t* tokens,
                      int64_t ignore_index, float inv_temperature, int64_t top, float* logprob, float* entropy, float* row_max,
                      float* row_log, float* top_logprob, int64_t* top_token, void* workspace, size_t workspace_bytes,
                      hipStream_t stream) {
  Q3_REQUIRE(sizes_ok(dtype, rows, vocab, top) && z && tokens && logprob && entropy && row_max && row_log && ld >= vocab);
  Q3_REQUIRE((top == 0 || (top_logprob && top_token)) && inv_temperature > 0.f && inv_temperature < INFINITY);
  Q3_REQUIRE(((uintptr_t)z & (dtype == Q3_F32 ? 3 : 1)) == 0 && workspace && ((uintptr_t)workspace & 15) == 0 &&
             workspace_bytes >= q3_token_logprobs_workspace_bytes(dtype, rows, vocab, top));
  Fwd a{z, ld, rows, vocab, tokens, ignore_index, inv_temperature, (int)top, (int)slices_for(dtype, rows, vocab),
        (Part*)workspace, nullptr, logprob, entropy, row_max, row_log, top_logprob, top_token};
  a.key = (uint64_t*)((char*)workspace + ((size_t)rows * a.slices * sizeof(Part) + 7) / 8 * 8);
  const int c = chunks_for(dtype, rows, vocab);
  if (dtype == Q3_BF16) return forward<BF16>(a, c, stream);
  if (dtype == Q3_F16) return forward<F16>(a, c, stream);
  return forward<F32>(a, c, stream);
}

int q3_token_logprobs_bwd(int dtype, int out_dtype, const void* z, int64_t ld, int64_t rows, int64_t vocab, const int64_t* tokens,
                          int64_t ignore_index, float inv_temperature, int64_t top, const int64_t* top_token,
                          const float* row_max, const float* row_log, const float* entropy, const float* g, const float* gh,
                          const float* gtop, void* dz, int64_t ldo, hipStream_t stream) {
  Q3_REQUIRE(sizes_ok(dtype, rows, vocab, top) && z && tokens && row_max && row_log && entropy && dz && ld >= vocab &&
             ldo >= vocab && (!gtop || (top > 0 && top_token)) && inv_temperature > 0.f && inv_temperature < INFINITY);
  Q3_REQUIRE(out_dtype == dtype || (dtype == Q3_F32 && dtype_ok(out_dtype)));
  Q3_REQUIRE(((uintptr_t)z & (dtype == Q3_F32 ? 3 : 1)) == 0 && ((uintptr_t)dz & (out_dtype == Q3_F32 ? 3 : 1)) == 0 && dz != z);
  const Bwd a{z, ld, rows, vocab, tokens, ignore_index, inv_temperature, (int)top, top_token, row_max, row_log, entropy, g, gh,
              gtop, dz, ldo};
  if (dtype == Q3_BF16) return backward<BF16, BF16>(a, stream);
  if (dtype == Q3_F16) return backward<F16, F16>(a, stream);
  if (out_dtype == Q3_BF16) return backward<F32, BF16>(a, stream);
  if (out_dtype == Q3_F16) return backward<F32, F16>(a, stream);
  return backward<F32, F32>(a, stream);
}

}  // extern "C"
