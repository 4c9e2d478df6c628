// Log probabilities of rows of logits [M, V]: log p of a given token, the entropy, the token's rank and the best `top` tokens.
//
// With a reference m near the maximum, d_v = l_v - m, S = sum e^d_v and T = sum d_v e^d_v:  log p(t) = d_t - ln S,  H = ln S - T / S,
// rank(t) = 1 + #{l_v > l_t} + #{v < t : l_v = l_t}; the sums computed with 2^ and log2. An entry that is -infinity (int64: at most -2^62) is masked: it has no
// probability and is no alternative. int64 logits are fixed point: l_v - m is taken exactly, then as a float.
//
// ONE pass over the rows: every thread keeps a reference at or above its own entries so far with S and T relative to it (32 bits; they
// are rescaled when it grows), a count, and offers entries for the best list; the next tile's loads are under way meanwhile. A row is cut over a cluster of CTAs, whose first
// one joins the parts through shared memory: one launch, no workspace, sums in a fixed order.
//
// The best list. Every few tiles a warp finds the k-th largest of 32 running maxima of disjoint parts of the row so far: at least
// k entries reach that threshold, so a later entry must exceed it. Some 31 entries per doubling of the entries seen do; they
// go to a buffer in shared memory, in any order, and are ranked at the end by (value, lower index). Rows in an order that defeats
// this (ascending, constant) overflow the buffer and are read again, with the buffer cut to the best k before it can overflow.
//
// What bounds it (rows of 128256, one B200): bf16 the exponentials, one per entry at 16 a cycle and SM, and the issue slots around them (2000 rows in
// 114 us, 4.5 TB/s; 118 when the rows are others in every call; 130 where their logits are around 1e5); int64 the ALU and issue (256 rows with the best 20 in 61 us, 4.3 TB/s); fp32 the ends of short parts (700 rows, half
// masked, with the best 5 in 100 us, 3.6 TB/s); few rows the latency of reading and joining (one row in 12 us).
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "bx_ptx.cuh"

namespace bx {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_MAX_TOP = 32, LP_MAX_CLUSTER = 16, LP_FEW = 256;
constexpr float LP_LOG2E = 1.4426950408889634f;
using i64_t = long long;

struct LogProbs {
  const void* logits;
  long long ld;
  const long long* tok;                                    // NULL: no tokens are given
  int V, top, shift;                                       // shift: bits of an int64 difference below 2^-24
  int near;                                                // int64: 256 units are at most 1, and none of them below 2^-24
  float scale;                                             // of a difference after the shift
  float *logp, *entropy;
  long long *rank, *ids;
  float* top_logp;
};

template <class T>
struct LpOf;                                               // how the entries of a row are read

template <>
struct LpOf<float> {
  using Val = float;
  static constexpr int VEC = 4, VECS = 8;                  // entries of a 16-byte load, loads of a thread per tile
  static __device__ __forceinline__ Val none() { return -INFINITY; }
  static __device__ __forceinline__ Val one(const float* p) { return *p; }
  static __device__ __forceinline__ Val get(const uint4& v, int e) { return __uint_as_float(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w); }
};

template <>
struct LpOf<__nv_bfloat16> {
  using Val = float;
  static constexpr int VEC = 8, VECS = 4;
  static __device__ __forceinline__ Val none() { return -INFINITY; }
  static __device__ __forceinline__ Val one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
  static __device__ __forceinline__ Val get(const uint4& v, int e) {
    const uint32_t w = word(v, e / 2);
    return __uint_as_float(e % 2 ? w & 0xffff0000u : w << 16);
  }
};

template <>
struct LpOf<long long> {
  using Val = long long;
  static constexpr int VEC = 2, VECS = 8;
  static __device__ __forceinline__ Val none() { return -(1ll << 62); }
  static __device__ __forceinline__ Val one(const long long* p) { return max(*p, none()); }
  static __device__ __forceinline__ Val get(const uint4& v, int e) {
    return (long long)((unsigned long long)(e ? v.w : v.y) << 32 | (e ? v.z : v.x));
  }
};

__device__ __forceinline__ float lp_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// x - m for x <= m as a float: at any distance, and (lp_delta) as the argument of e^, -infinity where that is 0 anyway.
__device__ __forceinline__ float lp_distance(float x, float m, const LogProbs&) { return x - m; }
__device__ __forceinline__ float lp_distance(long long x, long long m, const LogProbs& a) {
  return -(float)(((unsigned long long)m - (unsigned long long)x) >> a.shift) * a.scale;
}
__device__ __forceinline__ float lp_delta(float x, float m, const LogProbs&) { return x - m; }
__device__ __forceinline__ float lp_delta(long long x, long long m, const LogProbs& a) {
  const unsigned long long u = ((unsigned long long)m - (unsigned long long)x) >> a.shift;
  return u >> 32 ? -INFINITY : -(float)(uint32_t)u * a.scale;
}

// The largest value below x (above masked ones).
__device__ __forceinline__ float lp_below(float x) { return nextafterf(x, -INFINITY); }
__device__ __forceinline__ long long lp_below(long long x) { return x - 1; }

// Sums of some entries relative to a reference m at or above all of them: S = sum 2^y, T = sum y 2^y with y = log2(e) (l - m).
template <class Val>
struct LpSums {
  Val m;
  float s, t;

  __device__ __forceinline__ static float y_of(Val x, Val m, const LogProbs& a) { return lp_delta(x, m, a) * LP_LOG2E; }
  __device__ __forceinline__ void shift_to(Val m2, Val none, const LogProbs& a) {
    if (!(m2 > m)) return;
    if (m > none) {                                        // nothing but masked entries (and NaN) before: s is 0 or NaN
      const float d = fmaxf(y_of(m, m2, a), -1e4f), f = lp_exp2(d);
      t = f * fmaf(s, d, t);
      s *= f;
    }
    m = m2;
  }
};

__device__ __forceinline__ float lp_shfl(float v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ long long lp_shfl(long long v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// The sums of a warp's lanes, to all of them.
template <class Val>
__device__ __forceinline__ void lp_warp_join(LpSums<Val>& sum, int& count, Val none, const LogProbs& a) {
  Val m = sum.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, lp_shfl(m, o));
  sum.shift_to(m, none, a);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum.s += lp_shfl(sum.s, o);
    sum.t += lp_shfl(sum.t, o);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
}

template <class Val>
struct LpPart {
  Val m;
  float s, t;
  int count;
};

template <class Val>
__host__ __device__ constexpr int lp_capacity() { return sizeof(Val) == 8 ? 1024 : 2304; }

template <class Val>
struct LpShared {
  LpPart<Val> warp[LP_WARPS], part[LP_MAX_CLUSTER];
  Val group[2][32], threshold;
  int count, few;
  // candidates, those that reach the last threshold, the CTA's best k, and in the first CTA everybody's
  Val val[lp_capacity<Val>()], best_val[LP_MAX_TOP], all_val[LP_MAX_CLUSTER * LP_MAX_TOP];
  Val few_val[LP_FEW];
  int few_idx[LP_FEW], idx[lp_capacity<Val>()], best_idx[LP_MAX_TOP], all_idx[LP_MAX_CLUSTER * LP_MAX_TOP];
};

template <class Val>
__device__ __forceinline__ bool lp_better(Val a, int ia, Val b, int ib) { return a > b || (a == b && ia < ib); }

// The best k of n candidates, in order, to out_*; the places behind the last one get (none, -1). The whole block, which has to be
// in step before and after.
template <class Val>
__device__ __forceinline__ void lp_rank(const Val* val, const int* idx, int n, int k, Val* out_val, int* out_idx, Val none) {
  for (int i = threadIdx.x; i < k; i += LP_THREADS)
    if (i >= n) out_val[i] = none, out_idx[i] = -1;
  for (int i = threadIdx.x; i < n; i += LP_THREADS) {
    const Val v = val[i];
    const int at = idx[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += lp_better(val[j], idx[j], v, at);
    if (r < k) out_val[r] = v, out_idx[r] = at;
  }
}

// Stores into the shared memory of the cluster's first CTA.
__device__ __forceinline__ void lp_put(uint32_t at, int v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void lp_put(uint32_t at, float v) { lp_put(at, __float_as_int(v)); }
__device__ __forceinline__ void lp_put(uint32_t at, long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }

template <class T>
struct LpRow {                                             // the part of a row that belongs to one CTA
  using O = LpOf<T>;
  using Val = typename O::Val;
  const T* p;                                              // the row, back to a 16-byte boundary
  int lead, end;                                           // entries of p before the row, and up to its end
  int v0, v1;                                              // vectors, those that reach over the row's ends among them

  __device__ __forceinline__ bool whole(int v) const { return v * O::VEC >= lead && v * O::VEC + O::VEC <= end; }
  __device__ __forceinline__ uint4 load(int v) const { return *reinterpret_cast<const uint4*>(p + (i64_t)v * O::VEC); }
  // Any vector: its entries, those outside the row as masked ones. Entry e is token v VEC + e - lead.
  __device__ __forceinline__ void load(int v, Val* x) const {
#pragma unroll
    for (int e = 0; e < O::VEC; ++e) {
      const int i = v * O::VEC + e;
      x[e] = i >= lead && i < end ? O::one(p + i) : O::none();
    }
  }
};

// The second reading: candidates by single vectors a thread, the buffer cut to the best k whenever another step could overflow it.
template <class T>
__device__ __noinline__ void lp_again(const LpRow<T>& row, int k, LpShared<typename LpOf<T>::Val>* sh) {
  using O = LpOf<T>;
  using Val = typename O::Val;
  constexpr int CAP = lp_capacity<Val>(), STEP = LP_THREADS * O::VEC;
  static_assert(CAP >= STEP + LP_MAX_TOP, "a step fits behind the best k");
  Val threshold = O::none();
  if (threadIdx.x == 0) sh->count = 0;
  for (int v = row.v0; v < row.v1; v += LP_THREADS) {
    __syncthreads();
    const bool full = sh->count > CAP - STEP;
    __syncthreads();                                       // everybody has seen the same count
    if (full) {
      lp_rank(sh->val, sh->idx, sh->count, k, sh->best_val, sh->best_idx, O::none());
      __syncthreads();
      if (threadIdx.x < k) sh->val[threadIdx.x] = sh->best_val[threadIdx.x], sh->idx[threadIdx.x] = sh->best_idx[threadIdx.x];
      if (threadIdx.x == 0) sh->count = k;
      threshold = sh->best_val[k - 1];                     // later entries have higher indices: they must exceed it
      __syncthreads();
    }
    if (v + (int)threadIdx.x < row.v1) {
      Val x[O::VEC];
      row.load(v + threadIdx.x, x);
#pragma unroll
      for (int e = 0; e < O::VEC; ++e)
        if (x[e] > threshold) {
          const int n = atomicAdd(&sh->count, 1);
          sh->val[n] = x[e];
          sh->idx[n] = (v + threadIdx.x) * O::VEC + e - row.lead;
        }
    }
  }
  __syncthreads();
}

// An entry above the threshold goes to the buffer.
template <class Val>
__device__ __forceinline__ void lp_offer(LpShared<Val>* sh, Val x, int idx) {
  const int n = atomicAdd(&sh->count, 1);
  if (n < lp_capacity<Val>()) sh->val[n] = x, sh->idx[n] = idx;
}

// What a thread keeps of its entries, and how it takes in those of N vectors.
template <class T>
struct LpState {
  using O = LpOf<T>;
  using Val = typename O::Val;
  using Sums = LpSums<Val>;
  static constexpr int VEC = O::VEC;
  Sums sum;
  Val peak;                                                // the largest entry, or (int64) a value that one of them reaches
  Val best;                                                // none of the last vectors' entries is above this
  int count;                                               // entries that rank before the given token
  bool special;                                            // a tile was not of the usual kind

  // Any entries, x(e).
  template <int E, class X>
  __device__ __forceinline__ void add(X&& x, const LogProbs& a) {
    const Val none = O::none();
    best = none;
#pragma unroll
    for (int e = 0; e < E; ++e) best = max(best, x(e));
    peak = max(peak, best);
    sum.shift_to(best, none, a);
    const Val m = sum.m > none ? sum.m : Val(0);
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float y = sizeof(Val) == 4 || x(e) > none ? Sums::y_of(x(e), m, a) : -INFINITY, w = lp_exp2(y);
      s += w;
      t = fmaf(w, fmaxf(y, -2e4f), t);                     // a masked entry: 0 and not 0 times -infinity
    }
    sum.s += s;
    sum.t += t;
  }

  // Vectors of a row. Where no special case is met, that is floats below some 2800 without masked entries (a sum that is no number shows them) and int64
  // within 2^38 of zero and 2^32 of the reference, which then is a value at most 255 units above the largest entry, found from upper bits:
  // with fewer operations.
  template <int N>
  __device__ __forceinline__ void add_vectors(const uint4 (&v)[N], const LogProbs& a) {
    constexpr int E = N * VEC;
    auto x = [&](int e) { return O::get(v[e / VEC], e % VEC); };
    if (special) return add<E>(x, a);
    if constexpr (sizeof(Val) == 4) {
      if constexpr (VEC == 8) {                            // bf16: pairs
        __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&v[0].x);
#pragma unroll
        for (int i = 1; i < 4 * N; ++i) {
          const uint32_t w = O::word(v[i / 4], i % 4);
          b = __hmax2(b, *reinterpret_cast<const __nv_bfloat162*>(&w));
        }
        best = fmaxf(__low2float(b), __high2float(b));
      } else {
        best = x(0);
#pragma unroll
        for (int e = 1; e < E; ++e) best = fmaxf(best, x(e));
      }
      if (best > peak) {
        peak = best;
        sum.shift_to(best, O::none(), a);
      }
      // y by one fused multiply-add against the rounded product c = log2(e) m; what the rounding (off) makes of the sums is taken back by
      // the first two terms of 2^-off. |c| < 2^12 keeps off within half a unit of that, 2^-13, and the third term below 2^-28; larger
      // references (and infinities) take exact differences.
      const float c = sum.m * LP_LOG2E, off = fmaf(sum.m, LP_LOG2E, -c), back = fmaf(off, -0.6931471805599453f, 1.0f);
      float s = 0.0f, t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float y = fmaf(x(e), LP_LOG2E, -c), w = lp_exp2(y);
        s += w;
        t = fmaf(w, y, t);
      }
      if (fabsf(c) < 4096.0f && fabsf(t) < INFINITY) {
        sum.s = fmaf(s, back, sum.s);
        sum.t = fmaf(fmaf(-off, s, t), back, sum.t);
      } else {
        special = true;                                    // tiles like this one will follow
        add<E>(x, a);
      }
    } else {
      uint32_t far = 0;
      int hi = -0x7fffffff - 1, lo = 0x7fffffff;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t up = (uint32_t)(x(e) >> 32);
        const int t8 = __funnelshift_r((uint32_t)x(e), up, 8);
        far |= up + 64;
        hi = max(hi, t8);
        lo = min(lo, t8);
      }
      const Val ref = max(sum.m, ((Val)hi << 8) + 255);
      if (far >= 128 || (unsigned long long)(ref - ((Val)lo << 8)) >> 32 || !a.near) {
        special = true;
        return add<E>(x, a);
      }
      best = ((Val)hi << 8) + 255;
      peak = max(peak, (Val)hi << 8);
      sum.shift_to(ref, O::none(), a);
      float s = 0.0f, t = 0.0f;
      const float rate = -a.scale * LP_LOG2E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float y = (float)((uint32_t)ref - (uint32_t)x(e)) * rate, w = lp_exp2(y);
        s += w;
        t = fmaf(w, y, t);
      }
      sum.s += s;
      sum.t += t;
    }
  }

  // Entries that rank before the token: those above it, and equal ones at lower indices. N vectors that lie on one side of it ...
  template <int N>
  __device__ __forceinline__ void rank(const uint4 (&v)[N], bool before, Val mine) {
    if (before && !(mine > O::none())) {
      count += N * VEC;                                    // a masked token ranks behind everything before it
      return;
    }
    if constexpr (VEC == 8) {                              // pairs: 1 for each that does, at most 4 N in a sum
      const __nv_bfloat162 m = __float2bfloat162_rn(mine);
      __nv_bfloat162 n = __float2bfloat162_rn(0.0f);
#pragma unroll
      for (int i = 0; i < 4 * N; ++i) {
        const uint32_t w = O::word(v[i / 4], i % 4);
        const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w);
        n = __hadd2(n, before ? __hge2(x, m) : __hgt2(x, m));
      }
      count += (int)(__low2float(n) + __high2float(n));
    } else if (before) {
#pragma unroll
      for (int e = 0; e < N * VEC; ++e) count += O::get(v[e / VEC], e % VEC) >= mine;
    } else {
#pragma unroll
      for (int e = 0; e < N * VEC; ++e) count += O::get(v[e / VEC], e % VEC) > mine;
    }
  }
  // ... and any vector; i: index of its first entry, those outside 0 .. V - 1 do not count.
  template <class X>
  __device__ __forceinline__ void rank_any(X&& x, int i, int V, int tok, Val mine) {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (i + e >= 0 && i + e < V) count += i + e < tok ? mine > O::none() ? x(e) >= mine : 1 : i + e > tok && x(e) > mine;
  }
};

template <class T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 4) log_probs_kernel(const LogProbs a) {
  using O = LpOf<T>;
  using Val = typename O::Val;
  constexpr int VEC = O::VEC, CAP = lp_capacity<Val>(), VECS = O::VECS, STEP = LP_THREADS * VECS;
  extern __shared__ __align__(16) uint8_t lp_smem[];
  auto* sh = reinterpret_cast<LpShared<Val>*>(lp_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank, ctas;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  const long long m_row = blockIdx.x >> (__ffs(ctas) - 1);
  const Val none = O::none();
  if (ctas > 1) cluster_arrive();
  if (TOP && tid == 0) sh->count = 0, sh->few = 0, sh->threshold = none;
  if (TOP) __syncthreads();
  wait_previous();
  launch_next();

  const T* p = static_cast<const T*>(a.logits) + m_row * a.ld;
  LpRow<T> row;
  row.lead = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  row.p = p - row.lead;
  row.end = row.lead + a.V;
  // whole vectors of the row, dealt to the cluster in tiles; its first and last vector may be partly outside
  const int vecs = (row.end + VEC - 1) / VEC, wa = row.whole(0) ? 0 : 1, wb = max(wa, row.whole(vecs - 1) ? vecs : vecs - 1);
  const int tiles = (wb - wa + STEP - 1) / STEP;
  const int parts = __ffs(ctas) - 1;                       // ctas is a power of two
  const int w0 = min(wb, wa + (int)((long long)tiles * rank >> parts) * STEP), w1 = min(wb, wa + (int)((long long)tiles * (rank + 1) >> parts) * STEP);
  row.v0 = rank == 0 ? 0 : w0;
  row.v1 = rank == ctas - 1 ? vecs : w1;
  const long long tok64 = a.tok ? a.tok[m_row] : -1;
  const bool given = tok64 >= 0 && tok64 < a.V;
  const int tok = given ? (int)tok64 : -1;
  const Val mine = given ? O::one(p + tok) : none;

  LpState<T> st{{none, 0.0f, 0.0f}, none, none, 0, false};
  // the vectors at the row's ends, by one thread; their entries are all offered
  auto edge = [&](int v) {
    Val x[VEC];
    row.load(v, x);
    st.template add<VEC>([&](int e) { return x[e]; }, a);
    if (given) st.rank_any([&](int e) { return x[e]; }, v * VEC - row.lead, a.V, tok, mine);
    if (TOP)
      for (int e = 0; e < VEC; ++e)
        if (x[e] > none) lp_offer(sh, x[e], v * VEC + e - row.lead);
  };
  // N vectors of a thread, 256 apart from vector v on (negative: none)
  auto take = [&](auto n, int v) {
    constexpr int N = decltype(n)::value;
    uint4 raw[N];
#pragma unroll
    for (int u = 0; u < N; ++u) raw[u] = v >= 0 ? row.load(v + u * LP_THREADS) : uint4{};
    if (v >= 0) st.add_vectors(raw, a);
    if (given && v >= 0) {
      const int first = v * VEC - row.lead, end = first + ((N - 1) * LP_THREADS + 1) * VEC;      // of the thread
      if (first > tok || end <= tok) {
        st.rank(raw, end <= tok, mine);
      } else {
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const int i = first + u * LP_THREADS * VEC;
          const uint4 one[1] = {raw[u]};
          if (i > tok || i + VEC <= tok) st.rank(one, i <= tok, mine);
          else st.rank_any([&](int e) { return O::get(raw[u], e); }, i, a.V, tok, mine);
        }
      }
    }
    return [=, &sh](Val threshold) {                       // offers those above it
      if (!(st.best > threshold)) return;
#pragma unroll
      for (int e = 0; e < N * VEC; ++e) {
        const Val x = O::get(raw[e / VEC], e % VEC);
        if (x > threshold) lp_offer(sh, x, (v + e / VEC * LP_THREADS) * VEC + e % VEC - row.lead);
      }
    };
  };
  auto threshold = [&] { return *reinterpret_cast<volatile Val*>(&sh->threshold); };
  int updates = 0;
  auto update = [&] {
    Val* group = sh->group[updates++ & 1];                 // the other one may still be read
    Val g = st.peak;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) g = max(g, lp_shfl(g, o));
    if ((lane & 7) == 0) group[tid >> 3] = g;
    __syncthreads();
    if (warp == 0) {
      const Val own = group[lane];
      int r = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) r += lp_better(group[j], j, own, lane);
      if (r == a.top - 1) *reinterpret_cast<volatile Val*>(&sh->threshold) = own;
    }
  };
  // What a step offers is held against what came before it; only the first step is against itself, entries that equal the threshold
  // among them. The threshold is found anew when the entries behind it have doubled.
  int steps = 0;
  auto settle = [&](auto&& offer) {
    if (steps > 0) offer(threshold());
    if ((steps & (steps + 1)) == 0) update();
    if (steps == 0) {
      __syncthreads();
      offer(threshold() > none ? lp_below(threshold()) : none);
    }
    ++steps;
  };
  if (tid == 0 && rank == 0 && wa > 0) edge(0);
  int v = w0;
  for (; v + STEP <= w1; v += STEP) {
    auto offer = take(std::integral_constant<int, VECS>{}, v + tid);
    if (TOP) settle(offer);
  }
  for (; v < w1; v += LP_THREADS) {                        // less than a tile is left
    const bool in = v + tid < w1;
    auto offer = take(std::integral_constant<int, 1>{}, in ? v + tid : -1);
    if (TOP) settle([&](Val t) { if (in) offer(t); });
  }
  if (tid == 0 && rank == ctas - 1 && wb < vecs && vecs - 1 >= wa) edge(vecs - 1);
  LpSums<Val> sum = st.sum;
  int count = st.count;

  // ---- the CTA's part ----
  lp_warp_join(sum, count, none, a);
  if (lane == 0) sh->warp[warp] = {sum.m, sum.s, sum.t, count};
  if (TOP) update();
  __syncthreads();
  if (ctas > 1) cluster_wait();                            // the first CTA of the cluster runs: its shared memory may be written
  if (TOP) {
    const int n = sh->count;
    if (n > CAP) {
      __syncthreads();                                     // everybody has seen it
      lp_again<T>(row, a.top, sh);
      lp_rank(sh->val, sh->idx, sh->count, a.top, sh->best_val, sh->best_idx, none);
    } else {
      // few candidates reach the last threshold
      const Val t = sh->threshold;
      for (int i = tid; i < n; i += LP_THREADS)
        if (sh->val[i] >= t) {
          const int to = atomicAdd(&sh->few, 1);
          if (to < LP_FEW) sh->few_val[to] = sh->val[i], sh->few_idx[to] = sh->idx[i];
        }
      __syncthreads();
      const bool some = sh->few <= LP_FEW;
      lp_rank(some ? sh->few_val : sh->val, some ? sh->few_idx : sh->idx, some ? sh->few : n, a.top, sh->best_val, sh->best_idx, none);
    }
    __syncthreads();
    if (tid < a.top) {
      lp_put(mapa_shared(smem_u32(&sh->all_val[rank * a.top + tid]), 0), sh->best_val[tid]);
      lp_put(mapa_shared(smem_u32(&sh->all_idx[rank * a.top + tid]), 0), sh->best_idx[tid]);
    }
  }
  if (warp == 0) {
    LpSums<Val> all{none, 0.0f, 0.0f};
    int n = 0;
    if (lane < LP_WARPS) all = {sh->warp[lane].m, sh->warp[lane].s, sh->warp[lane].t}, n = sh->warp[lane].count;
    lp_warp_join(all, n, none, a);
    if (lane == 0) {
      LpPart<Val>* to = &sh->part[rank];
      lp_put(mapa_shared(smem_u32(&to->m), 0), all.m);
      lp_put(mapa_shared(smem_u32(&to->s), 0), all.s);
      lp_put(mapa_shared(smem_u32(&to->t), 0), all.t);
      lp_put(mapa_shared(smem_u32(&to->count), 0), n);
    }
  }
  if (ctas > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (rank != 0) return;

  // ---- the row ----
  LpSums<Val> all{none, 0.0f, 0.0f};
  int n = 0;
  if (lane < ctas) all = {sh->part[lane].m, sh->part[lane].s, sh->part[lane].t}, n = sh->part[lane].count;
  lp_warp_join(all, n, none, a);
  // a row without any entry, or with NaN or +infinity among them, has no probabilities
  const bool live = all.m > none && all.s > 0.0f && all.s < INFINITY;
  const float log_s = log2f(all.s);
  // (the distance is a logarithm already: by way of log2 it would be rounded twice more; a sum rounded to below 1 makes no p above 1)
  auto log_p = [&](Val v) { return fminf(fmaf(-0.6931471805599453f, log_s, lp_distance(v, all.m, a)), 0.0f); };
  if (tid == 0) {
    if (a.tok) {
      a.logp[m_row] = !live || !given ? NAN : mine > none ? log_p(mine) : -INFINITY;
      a.rank[m_row] = live && given ? n + 1 : 0;
    }
    a.entropy[m_row] = live ? 0.6931471805599453f * (log_s - all.t / all.s) : NAN;
  }
  if (TOP) {
    // every list is in order, its empty places at the end: those of all lists rank behind every entry
    const int total = ctas * a.top;
    for (int i = tid; i < total; i += LP_THREADS) {
      const Val v = sh->all_val[i];
      const int at = sh->all_idx[i];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < total; ++j) {
        const Val w = sh->all_val[j];
        const int aj = sh->all_idx[j];
        r += aj < 0 ? at < 0 && j < i : at < 0 || lp_better(w, aj, v, at);
      }
      if (r < a.top) {
        a.ids[m_row * a.top + r] = live ? at : -1;
        a.top_logp[m_row * a.top + r] = !live ? NAN : at >= 0 ? log_p(v) : -INFINITY;
      }
    }
  }
}

}  // namespace bx
