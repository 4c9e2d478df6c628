// Log probabilities of rows of logits [M, V]: log p of a given token, the entropy, the token's rank and the best `top` tokens.
//
// With m the maximum, d_v = l_v - m, S = sum e^d_v and T = sum d_v e^d_v:  log p(t) = d_t - ln S,  H = ln S - T / S,
// rank(t) = 1 + #{l_v > l_t} + #{v < t : l_v = l_t}. An entry that is -infinity (int64: at most -2^62) is masked: it has no
// probability and is no alternative. int64 logits are fixed point: l_v - m is taken exactly, then as a float.
//
// ONE pass over the rows: every thread keeps the running maximum of its own entries with S and T relative to it (32 bits; they are
// rescaled when the maximum grows), a count, and offers entries for the best list. A row is cut over a cluster of CTAs, whose first
// one joins the parts through shared memory: one launch, no workspace, sums in a fixed order.
//
// The best list. Every few tiles a warp finds the k-th largest of 32 running maxima of disjoint parts of the row so far: at least
// k entries reach that threshold, so a later entry must exceed it. Some 31 entries per doubling of the entries seen do; they
// go to a buffer in shared memory, in any order, and are ranked at the end by (value, lower index). Rows in an order that defeats
// this (ascending, constant) overflow the buffer and are read again, with the buffer cut to the best k before it can overflow.
#pragma once

#include <cuda_bf16.h>

#include "bx_ptx.cuh"

namespace bx {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_MAX_TOP = 32, LP_MAX_CLUSTER = 16;
constexpr int LP_VECS = 4;                                 // 16-byte loads of a thread per tile
constexpr float LP_LOG2E = 1.4426950408889634f;

struct LogProbs {
  const void* logits;
  long long ld;
  const long long* tok;                                    // NULL: no tokens are given
  int V, top, shift;                                       // shift: bits of an int64 difference below 2^-24
  float scale;                                             // of a difference after the shift
  float *logp, *entropy;
  long long *rank, *ids;
  float* top_logp;
};

template <class T>
struct LpOf;                                               // how the entries of a row are read and compared

template <>
struct LpOf<float> {
  using Val = float;
  static constexpr int VEC = 4;
  static __device__ __forceinline__ Val none() { return -INFINITY; }
  static __device__ __forceinline__ Val one(const float* p) { return *p; }
  static __device__ __forceinline__ void vec(const float* p, Val* x) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
};

template <>
struct LpOf<__nv_bfloat16> {
  using Val = float;
  static constexpr int VEC = 8;
  static __device__ __forceinline__ Val none() { return -INFINITY; }
  static __device__ __forceinline__ Val one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void vec(const __nv_bfloat16* p, Val* x) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

template <>
struct LpOf<long long> {
  using Val = long long;
  static constexpr int VEC = 2;
  static __device__ __forceinline__ Val none() { return -(1ll << 62); }
  static __device__ __forceinline__ Val one(const long long* p) { return max(*p, none()); }
  static __device__ __forceinline__ void vec(const long long* p, Val* x) {
    const longlong2 v = *reinterpret_cast<const longlong2*>(p);
    x[0] = max(v.x, none()), x[1] = max(v.y, none());
  }
};

__device__ __forceinline__ float lp_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// x - m for x <= m as a float; -infinity where e^ of it is 0 anyway.
__device__ __forceinline__ float lp_delta(float x, float m, const LogProbs&) { return x - m; }
__device__ __forceinline__ float lp_delta(long long x, long long m, const LogProbs& a) {
  const unsigned long long u = (unsigned long long)(m - x) >> a.shift;
  return u >> 32 ? -INFINITY : -(float)(uint32_t)u * a.scale;
}

// Entries that rank before one of value x: those above it, and equal ones at lower indices. Told by one comparison with a bound
// (floats with "at least", since there is none below a masked one; integers with "above", since there is none above the largest).
__device__ __forceinline__ float lp_bound(float x, bool lower) { return lower ? x : nextafterf(x, INFINITY); }
__device__ __forceinline__ long long lp_bound(long long x, bool lower) { return lower ? x - 1 : x; }
__device__ __forceinline__ bool lp_counts(float x, float bound) { return x >= bound; }
__device__ __forceinline__ bool lp_counts(long long x, long long bound) { return x > bound; }

// The largest value below x (above masked ones).
__device__ __forceinline__ float lp_below(float x) { return nextafterf(x, -INFINITY); }
__device__ __forceinline__ long long lp_below(long long x) { return x - 1; }

template <class Val>
struct LpSums {                                            // of some entries: their maximum, and S and T relative to it
  Val m;
  float s, t;

  __device__ __forceinline__ void shift_to(Val m2, Val none, const LogProbs& a) {
    if (!(m2 > m)) return;
    if (m > none) {                                        // nothing but masked entries (and NaN) before: s is 0 or NaN
      const float d = fmaxf(lp_delta(m, m2, a), -1e4f), f = lp_exp2(d * LP_LOG2E);
      t = f * fmaf(s, d, t);
      s *= f;
    }
    m = m2;
  }
  __device__ __forceinline__ void join(LpSums o, Val none, const LogProbs& a) {
    shift_to(o.m, none, a);
    o.shift_to(m, none, a);
    s += o.s;
    t += o.t;
  }
};

__device__ __forceinline__ float lp_shfl(float v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ long long lp_shfl(long long v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

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
  int count;
  // candidates, the CTA's best k, and in the first CTA everybody's
  Val val[lp_capacity<Val>()], best_val[LP_MAX_TOP], all_val[LP_MAX_CLUSTER * LP_MAX_TOP];
  int idx[lp_capacity<Val>()], best_idx[LP_MAX_TOP], all_idx[LP_MAX_CLUSTER * LP_MAX_TOP];
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
    for (int j = 0; j < n && r < k; ++j) r += lp_better(val[j], idx[j], v, at);
    if (r < k) out_val[r] = v, out_idx[r] = at;
  }
}

// Stores into the shared memory of the cluster's first CTA.
__device__ __forceinline__ void lp_put(uint32_t at, int v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void lp_put(uint32_t at, float v) { lp_put(at, __float_as_int(v)); }
__device__ __forceinline__ void lp_put(uint32_t at, long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }

template <class T>
struct LpRow {                                             // the vectors of a row that belong to one CTA
  using O = LpOf<T>;
  using Val = typename O::Val;
  const T* p;                                              // the row, back to a 16-byte boundary
  int lead, end;                                           // entries of p before the row, and up to its end
  int v0, v1;

  // Vector v: its entries, those outside the row as masked ones (their number is returned). Entry e is token v VEC + e - lead.
  __device__ __forceinline__ int load(int v, Val* x) const {
    const int i = v * O::VEC;
    if (i >= lead && i + O::VEC <= end) {
      O::vec(p + i, x);
      return 0;
    }
    int out = 0;
#pragma unroll
    for (int e = 0; e < O::VEC; ++e) {
      const bool in = i + e >= lead && i + e < end;
      x[e] = in ? O::one(p + i + e) : O::none();
      out += !in;
    }
    return out;
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

// The entries of a tile above the threshold go to the buffer.
template <class T>
__device__ __forceinline__ void lp_offer(const LpRow<T>& row, const typename LpOf<T>::Val* x, typename LpOf<T>::Val best,
                                         typename LpOf<T>::Val threshold, int v, LpShared<typename LpOf<T>::Val>* sh) {
  using O = LpOf<T>;
  if (!(best > threshold)) return;
#pragma unroll
  for (int e = 0; e < O::VEC * LP_VECS; ++e)
    if (x[e] > threshold) {
      const int n = atomicAdd(&sh->count, 1);
      if (n < lp_capacity<typename O::Val>()) {
        sh->val[n] = x[e];
        sh->idx[n] = (v + e / O::VEC * LP_THREADS + (int)threadIdx.x) * O::VEC + e % O::VEC - row.lead;
      }
    }
}

template <class T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 4) log_probs_kernel(const LogProbs a) {
  using O = LpOf<T>;
  using Val = typename O::Val;
  constexpr int E = O::VEC * LP_VECS, CAP = lp_capacity<Val>();
  extern __shared__ __align__(16) uint8_t lp_smem[];
  auto* sh = reinterpret_cast<LpShared<Val>*>(lp_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank, ctas;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  const long long m_row = blockIdx.x / ctas;
  const Val none = O::none();
  cluster_arrive();
  if (TOP && tid == 0) sh->count = 0, sh->threshold = none;
  if (TOP) __syncthreads();
  launch_next();
  wait_previous();

  const T* p = static_cast<const T*>(a.logits) + m_row * a.ld;
  LpRow<T> row;
  row.lead = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  row.p = p - row.lead;
  row.end = row.lead + a.V;
  const int vecs = (row.end + O::VEC - 1) / O::VEC;
  row.v0 = (int)((long long)vecs * rank / ctas);
  row.v1 = (int)((long long)vecs * (rank + 1) / ctas);
  const long long tok = a.tok ? a.tok[m_row] : -1;
  const bool given = tok >= 0 && tok < a.V;
  const Val mine = given ? O::one(p + tok) : none, lower = lp_bound(mine, true), higher = lp_bound(mine, false);

  LpSums<Val> sum{none, 0.0f, 0.0f};
  int count = 0, updates = 0;
  for (int v = row.v0, tile = 0; v < row.v1; v += LP_THREADS * LP_VECS, ++tile) {
    Val x[E];
    int outside = 0;
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u) {
      const int at = v + u * LP_THREADS + tid;
      if (at < row.v1) outside += row.load(at, x + u * O::VEC);
      else {
#pragma unroll
        for (int e = 0; e < O::VEC; ++e) x[u * O::VEC + e] = none;
        outside += O::VEC;
      }
    }
    Val best = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) best = max(best, x[e]);
    sum.shift_to(best, none, a);
    const Val m = sum.m > none ? sum.m : Val(0);
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = lp_delta(x[e], m, a), w = lp_exp2(d * LP_LOG2E);
      s += w;
      t = fmaf(w, fmaxf(d, -1e4f), t);
    }
    sum.s += s;
    sum.t += t;
    // entries that come before the token: at lower indices the equal ones too
    if (given) {
      const long long first = (long long)v * O::VEC - row.lead, end = first + (long long)LP_THREADS * E;
      if (tok >= first && tok < end) {
#pragma unroll
        for (int u = 0; u < LP_VECS; ++u)
#pragma unroll
          for (int e = 0; e < O::VEC; ++e)
            count += lp_counts(x[u * O::VEC + e], (long long)(v + u * LP_THREADS + tid) * O::VEC + e - row.lead < tok ? lower : higher);
        if (!(mine > none)) {                              // places outside the row read as masked entries
#pragma unroll 1
          for (int u = 0; u < LP_VECS; ++u)
#pragma unroll 1
            for (int e = 0; e < O::VEC; ++e) {
              const long long i = (long long)(v + u * LP_THREADS + tid) * O::VEC + e - row.lead;
              count -= i < tok && (i < 0 || v + u * LP_THREADS + tid >= row.v1);
            }
        }
      } else {
        const Val bound = tok >= end ? lower : higher;
#pragma unroll
        for (int e = 0; e < E; ++e) count += lp_counts(x[e], bound);
        if (lp_counts(none, bound)) count -= outside;
      }
    }
    if (TOP) {
      // a tile's entries are held against what came before them; only the first tile is against itself
      if (tile > 0) lp_offer<T>(row, x, best, *reinterpret_cast<volatile Val*>(&sh->threshold), v, sh);
      if ((tile & (tile + 1)) == 0 || (tile & 3) == 3) {
        Val* group = sh->group[updates++ & 1];             // the other one may still be read
        Val g = sum.m;
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
        if (tile == 0) {
          __syncthreads();
          // entries that equal the threshold count too
          const Val threshold = *reinterpret_cast<volatile Val*>(&sh->threshold);
          lp_offer<T>(row, x, best, threshold > none ? lp_below(threshold) : none, v, sh);
        }
      }
    }
  }

  // ---- the CTA's part ----
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const LpSums<Val> other{lp_shfl(sum.m, o), lp_shfl(sum.s, o), lp_shfl(sum.t, o)};
    sum.join(other, none, a);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  if (lane == 0) sh->warp[warp] = {sum.m, sum.s, sum.t, count};
  __syncthreads();
  cluster_wait();                                          // the first CTA of the cluster runs: its shared memory may be written
  if (TOP) {
    if (sh->count > CAP) {
      __syncthreads();                                     // everybody has seen it
      lp_again<T>(row, a.top, sh);
    }
    lp_rank(sh->val, sh->idx, sh->count, a.top, sh->best_val, sh->best_idx, none);
    __syncthreads();
    if (tid < a.top) {
      lp_put(mapa_shared(smem_u32(&sh->all_val[rank * a.top + tid]), 0), sh->best_val[tid]);
      lp_put(mapa_shared(smem_u32(&sh->all_idx[rank * a.top + tid]), 0), sh->best_idx[tid]);
    }
  }
  if (tid == 0) {
    LpSums<Val> all{sh->warp[0].m, sh->warp[0].s, sh->warp[0].t};
    int n = sh->warp[0].count;
#pragma unroll 1
    for (int w = 1; w < LP_WARPS; ++w) {
      all.join({sh->warp[w].m, sh->warp[w].s, sh->warp[w].t}, none, a);
      n += sh->warp[w].count;
    }
    LpPart<Val>* to = &sh->part[rank];
    lp_put(mapa_shared(smem_u32(&to->m), 0), all.m);
    lp_put(mapa_shared(smem_u32(&to->s), 0), all.s);
    lp_put(mapa_shared(smem_u32(&to->t), 0), all.t);
    lp_put(mapa_shared(smem_u32(&to->count), 0), n);
  }
  cluster_arrive();
  cluster_wait();
  if (rank != 0) return;

  // ---- the row ----
  LpSums<Val> all{sh->part[0].m, sh->part[0].s, sh->part[0].t};
  int n = sh->part[0].count;
  for (uint32_t c = 1; c < ctas; ++c) {
    all.join({sh->part[c].m, sh->part[c].s, sh->part[c].t}, none, a);
    n += sh->part[c].count;
  }
  // a row without any entry, or with NaN or +infinity among them, has no probabilities
  const bool live = all.m > none && all.s > 0.0f && all.s < INFINITY;
  const float log_s = logf(all.s);
  if (tid == 0) {
    if (a.tok) {
      a.logp[m_row] = !live || !given ? NAN : mine > none ? lp_delta(mine, all.m, a) - log_s : -INFINITY;
      a.rank[m_row] = live && given ? n + 1 : 0;
    }
    a.entropy[m_row] = live ? log_s - all.t / all.s : NAN;
  }
  if (TOP) {
    // every list is in order and without gaps: the empty places of all of them rank behind every entry
    const int total = ctas * a.top;
    for (int i = tid; i < total; i += LP_THREADS) {
      const Val v = sh->all_val[i];
      const int at = sh->all_idx[i];
      int r = 0;
      for (int j = 0; j < total && r < a.top; ++j) {
        const int aj = sh->all_idx[j];
        r += aj < 0 ? at < 0 && j < i : at < 0 || lp_better(sh->all_val[j], aj, v, at);
      }
      if (r < a.top) {
        a.ids[m_row * a.top + r] = live ? at : -1;
        a.top_logp[m_row * a.top + r] = !live ? NAN : at >= 0 ? lp_delta(v, all.m, a) - log_s : -INFINITY;
      }
    }
  }
}

}  // namespace bx
