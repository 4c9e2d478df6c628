// A paged cache of keys and values in 4 bits, and the kernels that write rows to it and read them back.
//
// An entry is code * scale * 2^e: a code of 4 bits (e2m1: a sign and 0, 0.5, 1, 1.5, 2, 3, 4 or 6), a scale of 8 (e4m3) for every 16
// entries, an exponent e of 8 for the row (a token's key or value of one head). e is the exponent of the row's largest magnitude
// less 10, the scale the smallest that keeps its 16 entries within 6 steps, the code the nearest (ties to the even one). Codes and
// scales together have 6 significant bits, so an entry is exact in bf16, code * scale alone in fp16, and every decision above is
// a comparison of exact products: the stored bits do not depend on rounding anywhere. 4.5 bits an entry and a byte a row, 146 bytes
// for 128 + 128 entries where bf16 takes 512.
//
// A row with NaN or an infinity in its key or its value has the scales of its key set to NaN and a value of zeros: a query that sees
// it becomes NaN, one that does not never multiplies it. Magnitudes above 2^127 are kept as 2^127.
//
// Layout: blocks of 64 tokens of one head, K and V = entries of a key and a value rounded up to multiples of 64.
//   key codes     [64 tokens][K / 2]      entry 2 i in the low half of byte i
//   key scales    [4][2][K / 16][8]       of token 16 a + 2 t + b, entries 16 j .. 16 j + 15 at [a][b][j][t]
//   value codes   [V / 16][8][64 tokens]  [j][i][token]: entry 16 j + i in the low half, 16 j + i + 8 in the high half
//   value scales  [V / 16][64 tokens]
//   key exponents [64], value exponents [64] (e + 127)
// Keys are read along a row, values along the tokens, the way the matrix instructions of the attention kernel contract them: a
// thread's 16-byte load holds just the codes of its own operand registers. No byte belongs to two tokens, so rows are written
// independently of each other.
#pragma once

#include <cuda_fp16.h>

#include "fl_common.cuh"

namespace bxf {

constexpr int C4_TOKENS = 64, C4_MAX = 512, C4_MIN_E = -100, C4_MAX_E = 117, C4_NAN = 127;

struct Cache4 {
  uint8_t* p;                          // [nb][G][page / 64] blocks
  int nb, G, page, dim, vdim, K, V;

  __host__ __device__ int bytes() const { return 36 * (K + V) + 2 * C4_TOKENS; }
  __device__ __forceinline__ bool has(i64 slot) const { return slot >= 0 && slot < (i64)nb * page; }
  __device__ __forceinline__ uint8_t* block(i64 slot, int g) const {
    // the division in 32 bits where the slots of the cache have no more (a 64-bit one is some hundred instructions)
    const i64 n = (i64)nb * page <= 0x7fffffffll ? (i64)((uint32_t)slot / (uint32_t)page) : slot / page;
    return p + ((n * G + g) * (page / C4_TOKENS) + (int)(slot - n * page) / C4_TOKENS) * bytes();
  }
  __device__ __forceinline__ int key_scale(int tok, int j) const {
    return 32 * K + ((tok / 16 * 2 + tok % 2) * (K / 16) + j) * 8 + tok % 16 / 2;
  }
  __device__ __forceinline__ int value_code(int tok, int j, int i) const { return 36 * K + (j * 8 + i) * C4_TOKENS + tok; }
  __device__ __forceinline__ int value_scale(int tok, int j) const { return 36 * K + 32 * V + j * C4_TOKENS + tok; }
  __device__ __forceinline__ int key_exp(int tok) const { return 36 * (K + V) + tok; }
  __device__ __forceinline__ int value_exp(int tok) const { return 36 * (K + V) + C4_TOKENS + tok; }
};

// Four bytes of two e2m1 codes each -> four pairs of fp16. (The compiler of CUDA 12.9 gives zeros for a word that it knows to be a zero-extended
// 16-bit load: such a one is handed over twice, in both halves.)
__device__ __forceinline__ void e2m1_pairs(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 x, y, z, w;\n\t"
      "mov.b32 {x, y, z, w}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, x;\n\tcvt.rn.f16x2.e2m1x2 %1, y;\n\tcvt.rn.f16x2.e2m1x2 %2, z;\n\tcvt.rn.f16x2.e2m1x2 %3, w;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// The two e4m3 scales in the low half of w -> a pair of fp16.
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ float c4_power(int e) { return __int_as_float((e + 127) << 23); }

// e4m3 byte (0 .. 127) -> its value; code 0 .. 15 -> its value.
__device__ __forceinline__ float c4_scale(int c) {
  return c >= 8 ? c == C4_NAN ? NAN : __int_as_float((c << 20) + (120 << 23)) : c * 0.001953125f;
}
__device__ __forceinline__ float c4_code(int c) {
  const int m = c & 7;
  const float v = m < 4 ? 0.5f * m : m == 7 ? 6.0f : (float)(m - 2);
  return c & 8 ? -v : v;
}

// The smallest scale of which 6 steps reach `most` (below 2048): an estimate from below, which is one less unless it is exact (two where a
// 32-bit `most` is the next number above a multiple).
template <class T>
__device__ __forceinline__ int c4_scale_for(float most) {
  const float f = __fmul_rd(most, 0.16666666f);
  int c = f < 0.015625f ? (int)(f * 512.0f) : (__float_as_int(f) - (120 << 23)) >> 20;
  c += 6.0f * c4_scale(c) < most;
  if constexpr (sizeof(T) == 4) c += 6.0f * c4_scale(c) < most;
  return c;
}
// Codes of four entries in steps of `step` (inv = about 1 / step; both 0 where the block is): the quotient, corrected by its exact
// remainder, is the correctly rounded one, and exact where it is a tie. The entries of bf16 rows come no nearer to a tie without being
// one than 2^-12 of it; those of 32-bit rows may round to one, and are set beside it by the sign of what remains.
template <class T>
__device__ __forceinline__ int c4_codes(const float (&y)[4], float step, float inv) {
  float q[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float t = y[k] * inv;
    q[k] = fmaf(fmaf(-t, step, y[k]), inv, t);
    if constexpr (sizeof(T) == 4) {
      const float rest = fmaf(-q[k], step, y[k]);
      const int bits = __float_as_int(q[k]), outward = (rest > 0.0f) == (q[k] > 0.0f) ? 1 : -1;
      if (rest != 0.0f && q[k] != 0.0f) q[k] = __int_as_float(bits + outward);
    }
  }
  uint32_t c;
  asm("{\n\t.reg .b8 x, y, z;\n\tmov.b32 {x, y, z, _}, 0;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 x, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 y, %4, %3;\n\tmov.b32 %0, {x, y, z, z};\n\t}"
      : "=r"(c)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]));
  return (int)c;
}

// A warp's row: lane l holds entries 128 i + 4 l .. + 3, i < N.
template <class T, int N>
struct C4Row {
  float x[N][4];

  __device__ __forceinline__ void load(const T* p, int n, int lane) {
    const bool wide = (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = 128 * i + 4 * lane;
      if (wide && d + 4 <= n) {
        if constexpr (sizeof(T) == 4) {
          const float4 v = *reinterpret_cast<const float4*>(p + d);
          x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(p + d);
          x[i][0] = __uint_as_float(v.x << 16), x[i][1] = __uint_as_float(v.x & 0xffff0000u);
          x[i][2] = __uint_as_float(v.y << 16), x[i][3] = __uint_as_float(v.y & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[i][k] = d + k < n ? ld(p + d + k) : 0.0f;
      }
    }
  }
  // -> the largest magnitude of the row as bits, which order like the numbers; NaN and infinities are above all of them.
  __device__ __forceinline__ uint32_t most() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) m = max(m, __float_as_uint(x[i][k]) & 0x7fffffffu);
    return __reduce_max_sync(0xffffffffu, m);
  }
  // Entries that are no numbers become 0, those beyond 2^127 that; -> the largest magnitude of the row then.
  __device__ __noinline__ float mend() {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (!(fabsf(x[i][k]) < INFINITY)) x[i][k] = 0.0f;
        x[i][k] = fminf(fmaxf(x[i][k], -1.7014118e38f), 1.7014118e38f);
        m = fmaxf(m, fabsf(x[i][k]));
      }
    return warp_max(m);
  }
  // Codes of the lane's four entries (4 bits each) and the scale of their block.
  __device__ __forceinline__ int codes(int i, float unit, int& scale) const {
    const float y[4] = {x[i][0] * unit, x[i][1] * unit, x[i][2] * unit, x[i][3] * unit};
    float m = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    scale = c4_scale_for<T>(m);
    const float step = c4_scale(scale);
    return c4_codes<T>(y, step, step > 0.0f ? __fdividef(1.0f, step) : 0.0f);
  }
};

__device__ __forceinline__ int c4_exponent(float most) {
  const int e = (__float_as_int(most) >> 23) - 127 - 10;                          // subnormal magnitudes end below the limit
  return most > 0.0f ? min(max(e, C4_MIN_E), C4_MAX_E) : C4_MIN_E;
}

template <class T>
struct Store4 {
  const T *k, *v;                      // [M][G] rows
  i64 k_row, k_head, v_row, v_head;
  const i64* slot;
  int M;
  Cache4 c;
};

constexpr int S4_THREADS = 128;

// ROWS rows of one head per CTA, a warp per row. Keys go out as they are made (a row is contiguous); the bytes of values lie along the
// tokens: with many rows they are put together in shared memory, and 16 (or 4) rows that lie in a run of slots go out as one store.
template <class T, int ROWS, int N>
__global__ void __launch_bounds__(S4_THREADS) fl_store4_kernel(const Store4<T> a) {
  constexpr int PITCH = ROWS + 4;      // bytes of a value column of the CTA's rows
  extern __shared__ __align__(16) uint8_t s4_smem[];
  __shared__ i64 slots[ROWS];
  __shared__ uint8_t* blocks[ROWS];                        // of the rows' tokens; NULL: a row that is left out
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = blockIdx.y, row0 = blockIdx.x * ROWS;
  const Cache4& c = a.c;
  launch_next();
  wait_previous();
  if (threadIdx.x < ROWS) {
    const i64 s = row0 + (int)threadIdx.x < a.M ? a.slot[row0 + threadIdx.x] : -1;
    slots[threadIdx.x] = c.has(s) ? s : -1;
    blocks[threadIdx.x] = c.has(s) ? c.block(s, g) : nullptr;
  }
  __syncthreads();
  const int columns = c.V / 2 + c.V / 16 + 1;              // of value bytes: codes, scales, the exponent
  C4Row<T, N> k, v, k_next, v_next;
  auto fetch = [&](int r) {
    if (r >= ROWS || slots[r] < 0) return;
    const i64 m = row0 + r;
    k_next.load(a.k + m * a.k_row + g * a.k_head, c.dim, lane);
    v_next.load(a.v + m * a.v_row + g * a.v_head, c.vdim, lane);
  };
  fetch(warp);
  for (int r = warp; r < ROWS; r += S4_THREADS / 32) {
    k = k_next, v = v_next;
    fetch(r + S4_THREADS / 32);
    if (slots[r] < 0) continue;
    const int tok = (int)(slots[r] % C4_TOKENS);
    uint8_t* block = blocks[r];
    const uint32_t bits_k = k.most(), bits_v = v.most();
    const bool bad = max(bits_k, bits_v) >= 0x7f800000u;
    float most_k = __uint_as_float(bits_k), most_v = __uint_as_float(bits_v);
    if (max(bits_k, bits_v) > 0x7f000000u) most_k = k.mend(), most_v = v.mend();
    const int ek = c4_exponent(most_k), ev = c4_exponent(most_v);
    const float uk = c4_power(-ek), uv = bad ? 0.0f : c4_power(-ev);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (128 * i >= c.K) break;
      int scale;
      const int code = k.codes(i, uk, scale), d = 128 * i + 4 * lane;
      if (d < c.K) {
        *reinterpret_cast<uint16_t*>(block + tok * (c.K / 2) + d / 2) = (uint16_t)code;
        if ((lane & 3) == 0) block[c.key_scale(tok, d / 16)] = bad ? C4_NAN : scale;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (128 * i >= c.V) break;
      int scale;
      const int code = v.codes(i, uv, scale), other = __shfl_xor_sync(0xffffffffu, code, 2), d = 128 * i + 4 * lane;
      if (d < c.V) {
        const int j = d / 16;
        if ((lane & 2) == 0) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint8_t byte = (code >> (4 * q) & 15) | (other >> (4 * q) & 15) << 4;
            const int at = (lane & 1) * 4 + q;
            if (ROWS > 4) s4_smem[(j * 8 + at) * PITCH + r] = byte;
            else block[c.value_code(tok, j, at)] = byte;
          }
        } else if ((lane & 3) == 3) {
          if (ROWS > 4) s4_smem[(c.V / 2 + j) * PITCH + r] = scale;
          else block[c.value_scale(tok, j)] = scale;
        }
      }
    }
    if (lane == 0) {
      block[c.key_exp(tok)] = ek + 127;
      if (ROWS > 4) s4_smem[(columns - 1) * PITCH + r] = ev + 127;
      else block[c.value_exp(tok)] = ev + 127;
    }
  }
  if (ROWS <= 4) return;
  __syncthreads();
  // value bytes: [column][token] in the block, columns 64 apart from its codes on, the exponents at their own place
  for (int i = threadIdx.x; i < columns * (ROWS / 16); i += S4_THREADS) {
    const int col = i % columns, r0 = i / columns * 16;
    const uint8_t* from = s4_smem + col * PITCH + r0;
    const i64 s0 = slots[r0];
    const int place = col < columns - 1 ? 36 * c.K + col * C4_TOKENS : 36 * (c.K + c.V) + C4_TOKENS;
    auto at = [&](int r) { return blocks[r] + place + (int)(slots[r] % C4_TOKENS); };
    bool run = s0 >= 0 && s0 % 16 == 0;
#pragma unroll
    for (int k = 1; k < 16; ++k) run &= slots[r0 + k] == s0 + k;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(from);
    if (run) {
      *reinterpret_cast<uint4*>(at(r0)) = make_uint4(w[0], w[1], w[2], w[3]);
      continue;
    }
    for (int k = 0; k < 16; k += 4) {
      const i64 s = slots[r0 + k];
      if (s >= 0 && s % 4 == 0 && slots[r0 + k + 1] == s + 1 && slots[r0 + k + 2] == s + 2 && slots[r0 + k + 3] == s + 3) {
        *reinterpret_cast<uint32_t*>(at(r0 + k)) = w[k / 4];
        continue;
      }
      for (int n = k; n < k + 4; ++n)
        if (slots[r0 + n] >= 0) *at(r0 + n) = from[n];
    }
  }
}

// The entries that the cache holds at `slot`: k T [M][G][dim], v T [M][G][vdim]; slots outside the cache give zeros. A warp per row and
// head, a lane for four entries (the codes of a key row lie together; a lane's four of a value are four bytes 64 apart).
constexpr int R4_WARPS = 8;

template <class T>
__device__ __forceinline__ void c4_put(T* p, int d, int n, const float (&x)[4]) {
  if (d + 4 <= n && (reinterpret_cast<uintptr_t>(p + d) & (4 * sizeof(T) - 1)) == 0) st4(p + d, x[0], x[1], x[2], x[3]);
  else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (d + q < n) st(p + d + q, x[q]);
  }
}

template <class T>
__global__ void __launch_bounds__(32 * R4_WARPS) fl_read4_kernel(const Cache4 c, const i64* slot, T* k, T* v, i64 rows) {
  launch_next();
  wait_previous();
  const uint32_t at = blockIdx.x * R4_WARPS + (threadIdx.x >> 5);          // below 2^31 + 8
  const int lane = threadIdx.x & 31;
  if (at >= rows) return;
  const uint32_t m = at / (uint32_t)c.G;
  const i64 s = slot[m];
  const bool in = c.has(s);
  const int tok = in ? (int)(s % C4_TOKENS) : 0;
  const uint8_t* b = c.block(in ? s : 0, (int)(at - m * c.G));
  const float pk = in ? __int_as_float(b[c.key_exp(tok)] << 23) : 0.0f, pv = in ? __int_as_float(b[c.value_exp(tok)] << 23) : 0.0f;
  auto put = [&](T* to, int d, int n, uint32_t codes, uint32_t scale, float power) {
    uint32_t h[4];
    e2m1_pairs(codes, h);
    const uint32_t f = e4m3_pair((scale & 127) * 0x0101u);
    float x[4];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t v = hmul2(h[q], f);
      const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&v));
      x[2 * q] = in ? w.x * power : 0.0f, x[2 * q + 1] = in ? w.y * power : 0.0f;
    }
    c4_put(to, d, n, x);
  };
  for (int d = 4 * lane; d < c.dim; d += 128)
    put(k + (i64)at * c.dim, d, c.dim, *reinterpret_cast<const uint16_t*>(b + tok * (c.K / 2) + d / 2) * 0x10001u, b[c.key_scale(tok, d / 16)], pk);
  for (int d = 4 * lane; d < c.vdim; d += 128) {
    const uint8_t* from = b + c.value_code(tok, d / 16, d % 8);
    const int half = d % 16 / 8 * 4;
    const uint32_t codes = (from[0] >> half & 15) | (from[C4_TOKENS] >> half & 15) << 4 | (from[2 * C4_TOKENS] >> half & 15) << 8 |
                           (from[3 * C4_TOKENS] >> half & 15) << 12;
    put(v + (i64)at * c.vdim, d, c.vdim, codes, b[c.value_scale(tok, d / 16)], pv);
  }
}

}  // namespace bxf
