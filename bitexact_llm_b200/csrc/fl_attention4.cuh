// Grouped-query attention over the 4-bit paged cache (fl_cache4.cuh).
#pragma once

#include "fl_attention.cuh"
#include "fl_cache4.cuh"

namespace bxf {

// ---- any sizes, both element types: one CTA per (query row, head), products in 32 bits ----
// A block of 64 keys at a time: two threads share a key (its scores from codes, scaled block by block of 16), then a thread owns two
// entries of the value and half of the tokens. PagedAttn's W and R are the entries of key and value, bs the tokens of a page.
constexpr int A4_THREADS = 128;

template <class T>
__global__ void __launch_bounds__(A4_THREADS) fl_attention4_plain_kernel(const PagedAttn a, const Cache4 c) {
  extern __shared__ float a4_smem[];                       // query [K], then the value's accumulators [2][V]
  __shared__ float p[C4_TOKENS], red[2][4];
  const int m = blockIdx.x, h = blockIdx.y, g = h / a.H, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float *q = a4_smem, *acc = a4_smem + c.K;
  launch_next();
  wait_previous();
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
      const int tok = tid >> 1, half = tid & 1, j0 = half * (c.K / 32);
      float v = 0.0f;
      for (int j = j0; j < j0 + c.K / 32; ++j) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(b + tok * (c.K / 2) + j * 8);
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) part = fmaf(q[j * 16 + i], c4_code(w[i / 8] >> (i % 8 * 4) & 15), part);
        v = fmaf(part, c4_scale(b[c.key_scale(tok, j)] & 127), v);
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
    if (tid < C4_TOKENS) p[tid] = e == 0.0f ? 0.0f : e * __int_as_float(b[c.value_exp(tid)] << 23);
    __syncthreads();
    den = den * corr + ((red[1][0] + red[1][1]) + (red[1][2] + red[1][3]));
    mx = m2;
    for (int col = tid >> 1; col < c.V / 2; col += C4_TOKENS) {
      const int j = col / 8, half = tid & 1;
      const uint8_t *codes = b + 36 * c.K + col * C4_TOKENS, *scales = b + 36 * c.K + 32 * c.V + j * C4_TOKENS;
      float* o = acc + half * c.V + j * 16 + col % 8;
      float lo = o[0] * corr, hi = o[8] * corr;
      for (int t = half * 32; t < half * 32 + 32; ++t) {
        const float w = p[t];
        if (w == 0.0f) continue;                           // behind the last token lies whatever was there before
        const float f = w * c4_scale(scales[t] & 127);
        lo = fmaf(f, c4_code(codes[t] & 15), lo);
        hi = fmaf(f, c4_code(codes[t] >> 4), hi);
      }
      o[0] = lo;
      o[8] = hi;
    }
    __syncthreads();
  }
  T* o = static_cast<T*>(a.out) + m * a.out_tok + h * a.out_head;
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  for (int d = tid; d < a.R; d += A4_THREADS) st(o + d, (acc[d] + acc[c.V + d]) * inv);
}

}  // namespace bxf
