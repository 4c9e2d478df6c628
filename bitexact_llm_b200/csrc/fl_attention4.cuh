// Grouped-query attention over the 4-bit paged cache (fl_cache4.cuh).
#pragma once

#include "fl_attention.cuh"
#include "fl_cache4.cuh"
#include "fl_gemm.cuh"

namespace bxf {

// Sums of weighted values are held times this until they are divided by the sum of the weights: 2^16 keys of the largest magnitude
// (2^127) stay finite, and the smallest (2^-90) are off by 2^-18 of themselves at most.
constexpr float A4_HEADROOM = 1.0f / 65536;

// ---- any sizes, both element types: one CTA per (query row, head), products in 32 bits ----
// A block of 64 keys at a time: two threads share a key (its scores from codes, scaled block by block of 16), then a thread owns two
// entries of the value and half of the tokens. PagedAttn's W and R are the entries of key and value, bs the tokens of a page.
// Codes become fp16 by the hardware's conversions, exactly; 20 tokens over 100 .. 800 keys of 128 + 128 entries, 16 heads: 36 us (123 with codes
// taken apart by integer operations). It does not split a context: one token over 10000 keys takes 290.
constexpr int A4_THREADS = 128;

template <class T>
__global__ void __launch_bounds__(A4_THREADS) fl_attention4_plain_kernel(const PagedAttn a, const Cache4 c) {
  extern __shared__ __align__(16) float a4_smem[];                       // query [K], then the value's accumulators [2][V]
  __shared__ __align__(16) float p[C4_TOKENS];
  __shared__ float red[2][4];
  const int m = blockIdx.x, h = blockIdx.y, g = h / a.H, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float *q = a4_smem, *acc = a4_smem + c.K;
  launch_next();
  wait_previous();
  if (a.tiles) {                                           // rows in no tile are left as they are
    bool mine = false;
    for (int t = tid; t < a.ntiles; t += A4_THREADS) mine |= m >= a.tiles[3 * t + 1] && m < a.tiles[3 * t + 1] + a.tiles[3 * t + 2];
    if (!__syncthreads_or(mine)) return;
  }
  const T* from = static_cast<const T*>(a.q) + (((i64)g * a.M + m) * a.H + h % a.H) * a.ldq;
  for (int d = tid; d < c.K; d += A4_THREADS) q[d] = d < a.W ? ld(from + d) : 0.0f;
  for (int d = tid; d < 2 * c.V; d += A4_THREADS) acc[d] = 0.0f;
  const i64 pos = min(a.pos[m], (i64)a.nblk * a.bs - 1), s = a.seq[m];
  const int first = a.first_key(pos);
  float mx = a.sink ? a.sink[h] : -INFINITY, den = a.sink ? 1.0f : 0.0f;
  __syncthreads();
  for (int k0 = first / C4_TOKENS * C4_TOKENS; k0 <= pos; k0 += C4_TOKENS) {
    const uint8_t* b = c.block(a.page_of(s, k0 / a.bs) * a.bs + k0 % a.bs, g);
    {
      const int tok = tid >> 1, half = tid & 1;
      float v = 0.0f;
      for (int j = half; j < c.K / 16; j += 2) {           // (every other one: the two threads' queries lie in different banks)
        const uint2 w = *reinterpret_cast<const uint2*>(b + tok * (c.K / 2) + j * 8);
        uint32_t codes[2][4];
        e2m1_pairs(w.x, codes[0]);
        e2m1_pairs(w.y, codes[1]);
        float even = 0.0f, odd = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 x = *reinterpret_cast<const float4*>(q + j * 16 + 4 * i);
          const float2 c0 = __half22float2(*reinterpret_cast<const __half2*>(&codes[i / 2][i % 2 * 2]));
          const float2 c1 = __half22float2(*reinterpret_cast<const __half2*>(&codes[i / 2][i % 2 * 2 + 1]));
          even = fmaf(x.x, c0.x, even), odd = fmaf(x.y, c0.y, odd);
          even = fmaf(x.z, c1.x, even), odd = fmaf(x.w, c1.y, odd);
        }
        v = fmaf(even + odd, c4_scale(b[c.key_scale(tok, j)] & 127), v);
      }
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v *= __int_as_float(b[c.key_exp(tok)] << 23) * a.scale;
      const int key = k0 + tok;
      if (key < first || key > pos) v = -INFINITY;
      if (half == 0) p[tok] = v;
      float best = warp_max(v);
      if (isnan(v)) best = v;
      best = __any_sync(0xffffffffu, isnan(v)) ? NAN : best;
      if (lane == 0) red[0][warp] = best;
    }
    __syncthreads();
    float m2 = mx;
#pragma unroll
    for (int w = 0; w < 4; ++w) m2 = isnan(red[0][w]) || isnan(m2) ? NAN : fmaxf(m2, red[0][w]);
    const float corr = mx == -INFINITY ? 0.0f : expf(mx - m2);
    float e = 0.0f;
    if (tid < C4_TOKENS) {
      const int key = k0 + tid;
      e = key < first || key > pos ? 0.0f : expf(p[tid] - m2);
    }
    const float part = warp_sum(e);
    if (lane == 0) red[1][warp] = part;
    if (tid < C4_TOKENS) p[tid] = e == 0.0f ? 0.0f : e * (__int_as_float(b[c.value_exp(tid)] << 23) * A4_HEADROOM);
    __syncthreads();
    den = den * corr + ((red[1][0] + red[1][1]) + (red[1][2] + red[1][3]));
    mx = m2;
    for (int col = tid >> 1; col < c.V / 2; col += C4_TOKENS) {
      const int j = col / 8, half = tid & 1;
      const uint8_t *codes = b + 36 * c.K + col * C4_TOKENS, *scales = b + 36 * c.K + 32 * c.V + j * C4_TOKENS;
      float* o = acc + half * c.V + j * 16 + col % 8;
      float lo = o[0] * corr, hi = o[8] * corr;
#pragma unroll
      for (int t = half * 32; t < half * 32 + 32; t += 16) {             // (what lies behind the last token is finite and has no weight)
        const uint4 vc = *reinterpret_cast<const uint4*>(codes + t), vs = *reinterpret_cast<const uint4*>(scales + t);
        const uint32_t cw[4] = {vc.x, vc.y, vc.z, vc.w}, sw[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 w = *reinterpret_cast<const float4*>(p + t + 4 * x);
          const float weight[4] = {w.x, w.y, w.z, w.w};
          uint32_t e[4];
          e2m1_pairs(cw[x], e);
          const uint32_t f[2] = {e4m3_pair(sw[x] & 0x7f7f7f7fu), e4m3_pair(sw[x] >> 16 & 0x7f7fu)};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t v = hmul2(e[y], __byte_perm(f[y / 2], 0, y % 2 ? 0x3232 : 0x1010));           // exact
            const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&v));
            lo = fmaf(weight[y], z.x, lo);
            hi = fmaf(weight[y], z.y, hi);
          }
        }
      }
      o[0] = lo;
      o[8] = hi;
    }
    __syncthreads();
  }
  T* o = static_cast<T*>(a.out) + m * a.out_tok + h * a.out_head;
  const float inv = den == 0.0f ? 0.0f : 1.0f / A4_HEADROOM / den;
  for (int d = tid; d < a.R; d += A4_THREADS) st(o + d, (acc[d] + acc[c.V + d]) * inv);
}

// ---- bf16 queries, keys and values of 64 or 128 entries: matrix instructions on operands that are made in registers ----
//
// The cache rows are the M side: scores S^T = K Q^T and outputs O^T = V^T P^T by m16n8k16 with fp32 accumulators, the query rows (tokens
// x heads of a group) being the N side in groups of 8: a decoding tile of 4 or 8 rows fills it where it would leave half or more of the
// M side empty. A 16-byte load from a block in shared memory holds the codes of a thread's own operand registers (the contraction
// index of a product may be dealt in any order as long as both operands agree). They become fp16 by one conversion and one
// product with the block's scale, both exact; the row's power of two goes into the score, or into the weight:
//   keys     s = 2^e_k (code scale . q) / sqrt(d); the query row is held in fp16 times a power of two that brings its largest entry to
//            2^14, so bf16 entries down to 2^-31 of that are exact
//   values   w = e^(s - max) 2^(e_v - E) 2^14 in fp16 (11 bits; the sum of the weights is of the unrounded ones), E the largest exponent of the
//            values that the row has seen: like the running maximum, the accumulators follow it when it grows. (The rows of one token see
//            the same; where a tile has several, a row has its own E, so that no later token costs an earlier one its digits.)
// A transposed 8x8 register exchange (movmatrix) turns P into the second product's operand: nothing goes through shared memory but the blocks.
//
// A tile belongs to one warp (CTAs of one: many tiles), to the W = 4 warps of a CTA, or to a cluster of those (few tiles). A warp takes every
// W-th block of its CTA's keys, in a ring of its own filled by bulk copies (one per block): warps never wait for one another until
// the end. The parts are joined through shared memory and that of the cluster in a fixed order, so there is one launch, no scratch
// memory, and the same bits in every call.
//
// What bounds it: the ALU (66 %) and issue (62 %), which conversions, scales and permutes of the codes take: 64 tokens over 8192 keys of 128 + 128 entries,
// 8 heads, in 134 us (4.6 TB/s; 144 when the cache is another one in every call); short contexts what a CTA does once, half of its time (256 tokens over 64 .. 1100 keys of 64 + 64: 40 us).
constexpr int A4_STAGES = 2, A4_MAX_CLUSTER = 16, A4_ROWS_MAX = 16;
constexpr int A4_BIAS = 14;            // weights are kept times 2^14

template <int W>
struct A4Shared {
  uint64_t full[W][A4_STAGES];
  float max_[W][A4_ROWS_MAX], den[W][A4_ROWS_MAX];                       // per warp and row
  float row_max[A4_ROWS_MAX], row_den[A4_ROWS_MAX];                      // of the CTA
  uint32_t abort_flag;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float a4_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
template <int N>
__device__ __forceinline__ void lds(uint32_t (&w)[N], const uint8_t* p) {
  static_assert(N == 2 || N == 4, "8 or 16 bytes");
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  }
}
// 2^14 over the power of two of a row's largest magnitude, and back.
__device__ __forceinline__ int a4_query_exponent(float most) {
  return most > 0.0f && most < INFINITY ? min(max((__float_as_int(most) >> 23) - 127, -100), 127) : 0;
}

template <int K, int V>
__host__ __device__ constexpr int a4_block_bytes() { return 36 * (K + V) + 2 * C4_TOKENS; }
// The warps' rings; at the end the same memory holds the warps' outputs, rows of V floats (and 4: the rows that a warp writes at a time lie in
// different banks).
template <int K, int V, int NT, int W>
__host__ __device__ constexpr int a4_ring_bytes() {
  const int ring = W * A4_STAGES * a4_block_bytes<K, V>(), out = (W > 1 ? W + 1 : 1) * 8 * NT * (V + 4) * 4;
  return ring > out ? ring : out;
}

// TILES: of one token or several; else single tokens.
template <int K, int V, int NT, int W, bool TILES>
__global__ void __launch_bounds__(32 * W, (NT == 1 ? 12 : 8) / W) fl_attention4_kernel(const PagedAttn a, const Cache4 c, int max_rows) {
  constexpr int BYTES = a4_block_bytes<K, V>(), KS = K / 16, KW = K / 32, ROWS = 8 * NT, PITCH = V + 4;
  extern __shared__ __align__(128) uint8_t a4_raw[];
  uint8_t* ring_all = a4_raw;
  auto* sh = reinterpret_cast<A4Shared<W>*>(a4_raw + a4_ring_bytes<K, V, NT, W>());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  uint32_t rank, ctas;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  if (threadIdx.x == 0) {
    for (int w = 0; w < W; ++w)
      for (int s = 0; s < A4_STAGES; ++s) mbar_init(&sh->full[w][s], 1);
    sh->abort_flag = *reinterpret_cast<volatile int*>(&g_wait_timeouts) != 0;
    fence_barrier_init();
  }
  if constexpr (W > 1) __syncthreads();
  else __syncwarp();
  launch_next();
  wait_previous();

  // ---- the tile ----
  const int tile = blockIdx.x >> (__ffs(ctas) - 1), group = blockIdx.y;
  int tok0, ntok;
  i64 seq;
  if constexpr (TILES) {
    const int* t = a.tiles + (i64)tile * 3;
    seq = t[0], tok0 = t[1], ntok = t[2];
  } else {
    tok0 = tile, ntok = 1;
    seq = a.seq[tok0];
  }
  const int row0 = blockIdx.z * ROWS, rows = min(ROWS, ntok * a.H - row0);
  if (rows <= 0 || TILES && ntok * a.H > max_rows) return;             // all CTAs of the cluster alike; taller tiles are another kernel's
  const i64 limit = (i64)a.nblk * a.bs - 1;
  // what depends on nothing but the tile is asked for ahead of the chain position, page, block
  uint32_t q[NT][KS][2];
  i64 row_pos[NT][2];                                      // of rows 2 tig, 2 tig + 1
  const bool wide = a.ldq % 4 == 0 && (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int flat = row0 + min(8 * t + gid, rows - 1);
    const bf16* from = static_cast<const bf16*>(a.q) + (((i64)group * a.M + tok0 + flat / a.H) * a.H + flat % a.H) * a.ldq + tig * (K / 4);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = tig * (K / 4) + 4 * s;
      if (wide && d + 4 <= a.W) {
        const uint2 v = *reinterpret_cast<const uint2*>(from + 4 * s);
        q[t][s][0] = v.x, q[t][s][1] = v.y;
      } else {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = d + e < a.W ? ld(from + 4 * s + e) : 0.0f;
        q[t][s][0] = pack_bf16(v[0], v[1]);
        q[t][s][1] = pack_bf16(v[2], v[3]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) row_pos[t][h] = a.pos[tok0 + (row0 + min(8 * t + 2 * tig + h, rows - 1)) / a.H];
  }
  const int t_first = row0 / a.H, t_last = (row0 + rows - 1) / a.H;
  const i64 p_first = min(a.pos[tok0 + t_first], limit), p_last = min(a.pos[tok0 + t_last], limit);
  const int lo_all = a.first_key(p_first), b_lo = lo_all / C4_TOKENS, b_hi = p_last < 0 ? b_lo : (int)(p_last / C4_TOKENS) + 1;
  const int b0 = b_lo + (int)((i64)(b_hi - b_lo) * rank / ctas), b1 = b_lo + (int)((i64)(b_hi - b_lo) * (rank + 1) / ctas);
  const int n = b1 - b0 > warp ? (b1 - b0 - warp + W - 1) / W : 0;          // the warp's blocks: b0 + warp + 4 i
  uint8_t* ring = ring_all + warp * A4_STAGES * BYTES;
  bool ok = sh->abort_flag == 0;

  int held = 0;
  auto fetch = [&](int i) {                                // block i of the warp; the warp reads the block table for 32 blocks at a time
    if ((i & 31) == 0) {
      const int b = min(b0 + warp + (i + lane) * W, b_hi - 1);
      held = (int)a.page_of(seq, min(b * C4_TOKENS / a.bs, a.nblk - 1));
    }
    const i64 page = __shfl_sync(0xffffffffu, held, i & 31);
    if (lane == 0) {
      const int in_page = (b0 + warp + i * W) % (a.bs / C4_TOKENS);
      uint64_t* bar = &sh->full[warp][i % A4_STAGES];
      mbar_arrive_expect_tx(bar, BYTES);
      bulk_load(ring + i % A4_STAGES * BYTES, c.p + ((page * a.G + group) * (a.bs / C4_TOKENS) + in_page) * BYTES, bar, BYTES);
    }
  };
  if (ok)
    for (int i = 0; i < A4_STAGES && i < n; ++i) fetch(i);

  // ---- queries: thread (gid, tig) holds, of row gid of every group of 8, entries tig K / 4 .. ----
  float row_scale[NT][2];                                  // of rows 2 tig, 2 tig + 1: what a score is worth in powers of two
  int row_lo[NT][2], row_hi[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float most = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        most = fmaxf(most, fmaxf(fabsf(__uint_as_float(q[t][s][h] << 16)), fabsf(__uint_as_float(q[t][s][h] & 0xffff0000u))));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = a4_query_exponent(most);
    // times 2^(14 - e), in two steps that cannot overflow on their own
    const float up = c4_power((A4_BIAS - e) / 2), up2 = c4_power(A4_BIAS - e - (A4_BIAS - e) / 2);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        q[t][s][h] = pack_half(__uint_as_float(q[t][s][h] << 16) * up * up2, __uint_as_float(q[t][s][h] & 0xffff0000u) * up * up2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int back = __shfl_sync(0xffffffffu, e, (2 * tig + h) * 4) - A4_BIAS;
      row_scale[t][h] = a.scale * 1.4426950408889634f * c4_power(back / 2) * c4_power(back - back / 2);
      const i64 p = min(row_pos[t][h], limit);
      row_lo[t][h] = a.first_key(p);
      row_hi[t][h] = (int)p;
    }
  }
  const int whole_lo = a.first_key(p_last), whole_hi = (int)p_first;       // keys that every row sees

  float out[V / 16][NT][4] = {};                           // entries 16 j + gid (+ 8) of rows 2 tig (+ 1)
  float top[NT][2], den[NT][2];
  int E[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) top[t][h] = -INFINITY, den[t][h] = 0.0f, E[t][h] = 0;

  for (int i = 0; ok && i < n; ++i) {
    if (!mbar_wait(&sh->full[warp][i % A4_STAGES], (i / A4_STAGES) & 1)) ok = false;
    if (!__all_sync(0xffffffffu, ok)) {
      // give up: what is in flight has to land before the memory is used for anything else
      ok = false;
      if (lane == 0) {
        atomicAdd(&g_wait_timeouts, 1);
        for (int k = i; k < min(n, i + A4_STAGES); ++k) mbar_wait(&sh->full[warp][k % A4_STAGES], (k / A4_STAGES) & 1);
      }
      __syncwarp();
      break;
    }
    const uint8_t* blk = ring + i % A4_STAGES * BYTES;
    const int k0 = (b0 + warp + i * W) * C4_TOKENS;

    // ---- scores: m-tile u holds tokens 16 (gid / 2) + 4 u + gid % 2 in its rows gid, and those + 2 in rows gid + 8 ----
    float s[4][NT][4] = {};
    const int tok = (gid >> 1) * 16 + (gid & 1);
    uint32_t ks[K / 32];
    lds<K / 32>(ks, blk + 32 * K + (((gid >> 1) * 2 + (gid & 1)) * (K / 16) + tig * (K / 64)) * 8);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t k_lo[KW], k_hi[KW];
      lds<KW>(k_lo, blk + (tok + 4 * u) * (K / 2) + tig * (K / 8));
      lds<KW>(k_hi, blk + (tok + 4 * u + 2) * (K / 2) + tig * (K / 8));
#pragma unroll
      for (int w = 0; w < KW; ++w) {                       // 8 codes: two steps of the contraction, within a block of 16
        const int j = w / 2;
        uint32_t lo[4], hi[4];
        const uint32_t pair = e4m3_pair(ks[j * 2 + u / 2] >> (u % 2 * 16));
        const uint32_t s_lo = __byte_perm(pair, 0, 0x1010), s_hi = __byte_perm(pair, 0, 0x3232);
        e2m1_pairs(k_lo[w], lo);
        e2m1_pairs(k_hi[w], hi);
#pragma unroll
        for (int x = 0; x < 4; ++x) lo[x] = hmul2(lo[x], s_lo), hi[x] = hmul2(hi[x], s_hi);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_f16(s[u][t], lo[0], hi[0], lo[1], hi[1], q[t][2 * w][0], q[t][2 * w][1]);
          mma_f16(s[u][t], lo[2], hi[2], lo[3], hi[3], q[t][2 * w + 1][0], q[t][2 * w + 1][1]);
        }
      }
    }

    // ---- exponents of the thread's tokens tok + 2 x, x = 0 .. 7: bytes 0 and 2 of four words ----
    uint32_t ke[4], ve[4];
    lds<4>(ke, blk + 36 * (K + V) + (gid >> 1) * 16);
    lds<4>(ve, blk + 36 * (K + V) + C4_TOKENS + (gid >> 1) * 16);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      ke[w] = ke[w] >> ((gid & 1) * 8) & 0x00ff00ffu;
      ve[w] = ve[w] >> ((gid & 1) * 8) & 0x00ff00ffu;
    }
    const bool edge = k0 < whole_lo || k0 + C4_TOKENS - 1 > whole_hi;
    if (edge) {                                            // exponents of tokens that no row of the tile sees
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int key = k0 + tok + 2 * x;
        if (key < lo_all || key > p_last) ve[x / 2] &= x % 2 ? 0x000000ffu : 0x00ff0000u;
      }
    }
    uint32_t big = __vmaxu2(__vmaxu2(ve[0], ve[1]), __vmaxu2(ve[2], ve[3]));
    int e_new = (int)max(big & 0xffffu, big >> 16);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) e_new = max(e_new, __shfl_xor_sync(0xffffffffu, e_new, o));

    // ---- the running maximum ----
    bool grows = false;
    float f[NT][2];
    if constexpr (TILES) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int e = e_new;
          if (edge) {
            e = 0;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const int key = k0 + tok + 2 * x;
              if (key >= row_lo[t][h] && key <= row_hi[t][h]) e = max(e, (int)(x % 2 ? ve[x / 2] >> 16 : ve[x / 2] & 0xffffu));
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) e = max(e, __shfl_xor_sync(0xffffffffu, e, o));
          }
          e = max(e, E[t][h]);
          grows |= e > E[t][h];
          f[t][h] = E[t][h] == 0 ? 0.0f : c4_power(max(E[t][h] - e, -126));
          E[t][h] = e;
        }
    } else {
      e_new = max(e_new, E[0][0]);
      grows = e_new > E[0][0];
      const float f_e = E[0][0] == 0 ? 0.0f : c4_power(max(E[0][0] - e_new, -126));
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) f[t][h] = f_e, E[t][h] = e_new;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int x = 0; x < 2; ++x) {                    // key rows gid and gid + 8 of m-tile u: token tok + 2 (2 u + x)
            float& v = s[u][t][2 * x + h];
            v *= __uint_as_float(x ? ke[u] << 7 & 0x7f800000u : ke[u] << 23) * row_scale[t][h];
            if (edge) {
              const int key = k0 + tok + 4 * u + 2 * x;
              if (key < row_lo[t][h] || key > row_hi[t][h]) v = -INFINITY;
            }
            m = fmaxf(m, v);
          }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (m > top[t][h]) {
          const float g = a4_exp2(top[t][h] - m);          // 0 for the first keys
          f[t][h] *= g;
          den[t][h] *= g;
          top[t][h] = m;
          grows = true;
        }
      }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int j = 0; j < V / 16; ++j)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) out[j][t][x] *= f[t][x & 1];
    }

    // ---- weights: their sum as they are, then times the values' powers of two, transposed ----
    uint32_t p[4][NT][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float g[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int e = (int)(x ? ve[u] >> 16 : ve[u] & 0xffffu) - E[0][0] + 127 + A4_BIAS;
        g[x] = __int_as_float(max(e, 0) << 23);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float w[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float m = top[t][h] == -INFINITY ? 0.0f : top[t][h];
            w[h] = a4_exp2(s[u][t][2 * x + h] - m);
            den[t][h] += w[h];
            if constexpr (TILES) {                         // (a key that the row does not see may have a larger exponent)
              const int e = min((int)(x ? ve[u] >> 16 : ve[u] & 0xffffu) - E[t][h], 0) + 127 + A4_BIAS;
              g[x] = __int_as_float(max(e, 0) << 23);
            }
            w[h] *= g[x];
          }
          p[u][t][x] = transposed(pack_half(w[0], w[1]));
        }
    }

    // ---- values: entries 16 j + gid and + 8 of tokens 16 tig .. + 15 ----
#pragma unroll
    for (int j = 0; j < V / 16; ++j) {
      uint32_t vc[4], vs[4];
      lds<4>(vc, blk + 36 * K + (j * 8 + gid) * C4_TOKENS + tig * 16);
      lds<4>(vs, blk + 36 * K + 32 * V + j * C4_TOKENS + tig * 16);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t x[4];
        e2m1_pairs(vc[u], x);
        const uint32_t s01 = e4m3_pair(vs[u]), s23 = e4m3_pair(vs[u] >> 16);
        const uint32_t a0 = hmul2(__byte_perm(x[0], x[1], 0x5410), s01), a1 = hmul2(__byte_perm(x[0], x[1], 0x7632), s01);
        const uint32_t a2 = hmul2(__byte_perm(x[2], x[3], 0x5410), s23), a3 = hmul2(__byte_perm(x[2], x[3], 0x7632), s23);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16(out[j][t], a0, a1, a2, a3, p[u][t][0], p[u][t][1]);
      }
    }
    __syncwarp();                                          // the block is read: its place may be filled again
    if (i + A4_STAGES < n) fetch(i + A4_STAGES);
  }

  // ---- the CTA's part: rows of V outputs per warp, times A4_HEADROOM ----
  auto together = [] {
    if constexpr (W > 1) __syncthreads();
    else __syncwarp();
  };
  if (!ok) sh->abort_flag = 1;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) den[t][h] += __shfl_xor_sync(0xffffffffu, den[t][h], o);
      if (gid == 0) sh->max_[warp][8 * t + 2 * tig + h] = top[t][h], sh->den[warp][8 * t + 2 * tig + h] = den[t][h];
    }
  together();                                              // all rings are done with
  const bool dead = sh->abort_flag != 0;
  float* slab = reinterpret_cast<float*>(ring_all);        // [row][V] of the CTA, then (W > 1) of every warp
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * t + 2 * tig + h;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) m = fmaxf(m, sh->max_[w][r]);
      const float unit = E[t][h] == 0 ? 0.0f : c4_power(max(E[t][h] - 127 - A4_BIAS, -126));
      const float g = unit * A4_HEADROOM * (top[t][h] == -INFINITY ? 0.0f : a4_exp2(top[t][h] - m));
      float* to = slab + ((W > 1 ? warp + 1 : 0) * ROWS + r) * PITCH + gid;
#pragma unroll
      for (int j = 0; j < V / 16; ++j) {
        to[16 * j] = out[j][t][h] * g;
        to[16 * j + 8] = out[j][t][h + 2] * g;
      }
      if (warp == 0 && gid == 0) {
        float d = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) d += sh->max_[w][r] == -INFINITY ? sh->den[w][r] : sh->den[w][r] * a4_exp2(sh->max_[w][r] - m);
        sh->row_max[r] = m;
        sh->row_den[r] = d;
      }
    }
  together();
  if constexpr (W > 1) {
    for (int i = 4 * threadIdx.x; i < ROWS * PITCH; i += 128 * W) {
      float4 v = *reinterpret_cast<const float4*>(slab + ROWS * PITCH + i);
#pragma unroll
      for (int w = 2; w <= W; ++w) {
        const float4 u = *reinterpret_cast<const float4*>(slab + w * ROWS * PITCH + i);
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
      }
      *reinterpret_cast<float4*>(slab + i) = v;
    }
    __syncthreads();
  }
  // ---- the rows: every CTA of the cluster finishes a part of the outputs, a thread four entries ----
  const bool quads = a.R % 4 == 0 && a.out_tok % 4 == 0 && a.out_head % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0;
  if (ctas > 1) {
    cluster_arrive();
    cluster_wait();
  } else if (dead) {
    return;
  }
  const uint32_t slab_at = smem_u32(slab), max_at = smem_u32(sh->row_max), den_at = smem_u32(sh->row_den);
  for (int i = (rank * 32 * W + threadIdx.x) * 4; i < rows * V && !dead; i += ctas * 32 * W * 4) {
    const int r = i / V, d = i % V, at = r * PITCH + d, flat = row0 + r, head = group * a.H + flat % a.H;
    if (d >= a.R) continue;
    const float sink = a.sink ? a.sink[head] * 1.4426950408889634f : -INFINITY;
    float m = sink, sum = 0.0f, v[4] = {};
    if (ctas == 1) {
      const float mk = sh->row_max[r], dk = sh->row_den[r];
      m = fmaxf(m, mk);
      const float g = mk == -INFINITY ? (dk == 0.0f ? 0.0f : 1.0f) : a4_exp2(mk - m);      // a part with no key has no weight
      sum = g * dk;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = g * slab[at + e];
    } else {
      for (uint32_t k = 0; k < ctas; ++k) m = fmaxf(m, ld_cluster(mapa_shared(max_at + 4 * r, k)));
      for (uint32_t k = 0; k < ctas; ++k) {
        const float mk = ld_cluster(mapa_shared(max_at + 4 * r, k)), dk = ld_cluster(mapa_shared(den_at + 4 * r, k));
        const float g = mk == -INFINITY ? (dk == 0.0f ? 0.0f : 1.0f) : a4_exp2(mk - m);
        const uint32_t from = mapa_shared(slab_at + 4 * at, k);
        sum += g * dk;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += g * ld_cluster(from + 4 * e);
      }
    }
    if (sink != -INFINITY) sum += a4_exp2(sink - m);       // (m is -infinity too where the row sees nothing)
    const float inv = sum == 0.0f ? 0.0f : 1.0f / A4_HEADROOM / sum;
    bf16* to = static_cast<bf16*>(a.out) + (tok0 + flat / a.H) * a.out_tok + head * a.out_head + d;
    if (quads) {
      st4(to, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < a.R) st(to + e, v[e] * inv);
    }
  }
  if (ctas == 1) return;
  cluster_arrive();                                        // nobody leaves while its memory may be read
  cluster_wait();
}

}  // namespace bxf
