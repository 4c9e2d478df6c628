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

// Four bytes of two e2m1 codes each -> four pairs of fp16. (Not for words that are zero-extended 16-bit loads: the compiler of CUDA 12.9
// gives zeros for those.)
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

// e4m3 byte (0 .. 127) -> its value.
__device__ __forceinline__ float c4_scale(int c) {
  return c >= 8 ? c == C4_NAN ? NAN : __int_as_float((c << 20) + (120 << 23)) : c * 0.001953125f;
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
// one than 2^-12 of it. A quotient of a 32-bit row may be rounded to a tie (three significant bits: only then is the rest of it looked at, since a
// step aside may end on one), and is set beside it by the sign of what remains.
template <class T>
__device__ __forceinline__ uint32_t c4_codes(const float (&y)[4], float step, float inv) {
  float q[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float t = y[k] * inv;
    q[k] = fmaf(fmaf(-t, step, y[k]), inv, t);
    if constexpr (sizeof(T) == 4) {
      const float rest = fmaf(-q[k], step, y[k]);
      const int bits = __float_as_int(q[k]), outward = (rest > 0.0f) == (q[k] > 0.0f) ? 1 : -1;
      if (rest != 0.0f && q[k] != 0.0f && bits << 12 == 0) q[k] = __int_as_float(bits + outward);
    }
  }
  uint32_t c;
  asm("{\n\t.reg .b8 x, y, z;\n\tmov.b32 {x, y, z, _}, 0;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 x, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 y, %4, %3;\n\tmov.b32 %0, {x, y, z, z};\n\t}"
      : "=r"(c)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]));
  return c;
}

// A row of half a warp: lane l of 16 holds entries 128 i + 8 l .. + 7, i < N, so that two lanes share a block of 16 and its scale.
template <class T, int N>
struct C4Row {
  float x[N][8];

  __device__ __forceinline__ void load(const T* p, int n, int l) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = 128 * i + 8 * l;
      if ((at & 15) == 0 && d + 8 <= n) {
        if constexpr (sizeof(T) == 4) {
          const float4 v = *reinterpret_cast<const float4*>(p + d), w = *reinterpret_cast<const float4*>(p + d + 4);
          x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w, x[i][4] = w.x, x[i][5] = w.y, x[i][6] = w.z, x[i][7] = w.w;
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(p + d);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) x[i][2 * k] = __uint_as_float(w[k] << 16), x[i][2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k] = d + k < n ? ld(p + d + k) : 0.0f;
      }
    }
  }
  // -> the largest magnitude of the row as bits, which order like the numbers; NaN and infinities are above all of them.
  __device__ __forceinline__ uint32_t most(int lane) const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(x[i][k]) & 0x7fffffffu);
    return __reduce_max_sync(0xffffu << (lane & 16), m);
  }
  // Entries that are no numbers become 0, those beyond 2^127 that; -> the largest magnitude of the row then.
  __device__ __noinline__ float mend() {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (!(fabsf(x[i][k]) < INFINITY)) x[i][k] = 0.0f;
        x[i][k] = fminf(fmaxf(x[i][k], -1.7014118e38f), 1.7014118e38f);
        m = fmaxf(m, fabsf(x[i][k]));
      }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
  // Codes of the lane's eight entries (4 bits each) and the scale of their block.
  __device__ __forceinline__ uint32_t codes(int i, float unit, int& scale) const {
    float y[8], m = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      y[k] = x[i][k] * unit;
      m = fmaxf(m, fabsf(y[k]));
    }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    scale = c4_scale_for<T>(m);
    const float step = c4_scale(scale), inv = step > 0.0f ? __fdividef(1.0f, step) : 0.0f;
    return c4_codes<T>({y[0], y[1], y[2], y[3]}, step, inv) | c4_codes<T>({y[4], y[5], y[6], y[7]}, step, inv) << 16;
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

__host__ __device__ constexpr int s4_threads(int rows) { return rows < 8 ? 16 * rows : 128; }

// ROWS rows of one head per CTA, half a warp per row. Keys go out as they are made (a row is contiguous); the bytes of values lie along the
// tokens: with many rows they are put together in shared memory, and 16 (or 4) rows that lie in a run of slots go out as one store.
// What bounds it is issue, at some 240 instructions for 256 entries of bf16: 8192 rows of 8 heads in 29 us with cold caches (1.5 TB/s; 22 on the same rows
// again; a warp per row, in which four lanes made the scale of a block, took 42). 32-bit rows: 29 on the same rows again.
template <class T, int ROWS, int N>
__global__ void __launch_bounds__(s4_threads(ROWS)) fl_store4_kernel(const Store4<T> a) {
  constexpr int PITCH = ROWS + 4, THREADS = s4_threads(ROWS), STEP = THREADS / 16;  // bytes of a value column of the CTA's rows; rows at a time
  constexpr bool GATHER = ROWS > STEP;
  extern __shared__ __align__(16) uint8_t s4_smem[];
  __shared__ i64 slots[ROWS];
  __shared__ uint8_t* blocks[ROWS];                        // of the rows' tokens; NULL: a row that is left out
  __shared__ uint32_t in16, in4;                           // rows whose slot follows on from a multiple of 16 (4) of the first of their 16 (4)
  const int lane = threadIdx.x & 31, l = lane & 15, g = blockIdx.y, row0 = blockIdx.x * ROWS;
  const Cache4& c = a.c;
  launch_next();
  wait_previous();
  if (threadIdx.x < ROWS) {
    const i64 s = row0 + (int)threadIdx.x < a.M ? a.slot[row0 + threadIdx.x] : -1;
    slots[threadIdx.x] = c.has(s) ? s : -1;
    blocks[threadIdx.x] = c.has(s) ? c.block(s, g) : nullptr;
    if constexpr (GATHER) {
      static_assert(ROWS == 32, "a warp");
      const i64 mine = c.has(s) ? s : -1, f16 = __shfl_sync(0xffffffffu, mine, lane & 16), f4 = __shfl_sync(0xffffffffu, mine, lane & 28);
      const uint32_t b16 = __ballot_sync(0xffffffffu, f16 >= 0 && f16 % 16 == 0 && mine == f16 + (lane & 15));
      const uint32_t b4 = __ballot_sync(0xffffffffu, f4 >= 0 && f4 % 4 == 0 && mine == f4 + (lane & 3));
      if (lane == 0) in16 = b16, in4 = b4;
    }
  }
  __syncthreads();
  const int columns = c.V / 2 + c.V / 16 + 1;              // of value bytes: codes, scales, the exponent
  C4Row<T, N> k, v, k_next, v_next;
  const i64 m0 = row0 + (int)threadIdx.x / 16;
  const T *from_k = a.k + m0 * a.k_row + g * a.k_head, *from_v = a.v + m0 * a.v_row + g * a.v_head;
  auto fetch = [&](int r) {
    if (r >= ROWS) return;
    const bool live = slots[r] >= 0;                       // (nothing is read of others)
    k_next.load(from_k, live ? c.dim : 0, l);
    v_next.load(from_v, live ? c.vdim : 0, l);
    from_k += STEP * a.k_row, from_v += STEP * a.v_row;
  };
  fetch(threadIdx.x / 16);
  for (int r = threadIdx.x / 16; r < ROWS; r += STEP) {    // (STEP divides ROWS: the halves of a warp go together)
    k = k_next, v = v_next;
    fetch(r + STEP);
    const bool live = slots[r] >= 0;
    if (!__any_sync(0xffffffffu, live)) continue;
    const int tok = (int)(slots[r] & (C4_TOKENS - 1));
    uint8_t* block = blocks[r];
    const uint32_t bits_k = k.most(lane), bits_v = v.most(lane);
    const bool bad = max(bits_k, bits_v) >= 0x7f800000u;
    float most_k = __uint_as_float(bits_k), most_v = __uint_as_float(bits_v);
    if (__any_sync(0xffffffffu, max(bits_k, bits_v) > 0x7f000000u)) most_k = k.mend(), most_v = v.mend();
    const int ek = c4_exponent(most_k), ev = c4_exponent(most_v);
    const float uk = c4_power(-ek), uv = bad ? 0.0f : c4_power(-ev);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (128 * i >= c.K) break;
      int scale;
      const uint32_t code = k.codes(i, uk, scale);
      const int d = 128 * i + 8 * l;
      if (live && d < c.K) {
        *reinterpret_cast<uint32_t*>(block + tok * (c.K / 2) + d / 2) = code;
        if ((l & 1) == 0) block[c.key_scale(tok, d / 16)] = bad ? C4_NAN : scale;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (128 * i >= c.V) break;
      int scale;
      const uint32_t code = v.codes(i, uv, scale), other = __shfl_xor_sync(0xffffffffu, code, 1);
      const int d = 128 * i + 8 * l, j = d / 16, odd = l & 1;
      if (live && d < c.V) {
        // the pair's 16 entries in 8 bytes, entry q low and q + 8 high: four to each lane, from halves of its and its neighbour's codes
        uint32_t lo = odd ? other >> 16 : code & 0xffffu, hi = odd ? code >> 16 : other & 0xffffu;
        lo = (lo | lo << 8) & 0x00ff00ffu, hi = (hi | hi << 8) & 0x00ff00ffu;
        lo = (lo | lo << 4) & 0x0f0f0f0fu, hi = (hi | hi << 4) & 0x0f0f0f0fu;
        const uint32_t bytes = lo | hi << 4;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint8_t byte = bytes >> (8 * q);
          if (GATHER) s4_smem[(j * 8 + odd * 4 + q) * PITCH + r] = byte;
          else block[c.value_code(tok, j, odd * 4 + q)] = byte;
        }
        if (odd) {
          if (GATHER) s4_smem[(c.V / 2 + j) * PITCH + r] = scale;
          else block[c.value_scale(tok, j)] = scale;
        }
      }
    }
    if (live && l == 0) {
      block[c.key_exp(tok)] = ek + 127;
      if (GATHER) s4_smem[(columns - 1) * PITCH + r] = ev + 127;
      else block[c.value_exp(tok)] = ev + 127;
    }
  }
  if (!GATHER) return;
  __syncthreads();
  // value bytes: [column][token] in the block, columns 64 apart from its codes on, the exponents at their own place
  for (int i = threadIdx.x; i < columns * (ROWS / 16); i += THREADS) {
    const int col = i % columns, r0 = i / columns * 16;
    const uint8_t* from = s4_smem + col * PITCH + r0;
    const int place = col < columns - 1 ? 36 * c.K + col * C4_TOKENS : 36 * (c.K + c.V) + C4_TOKENS;
    auto at = [&](int r) { return blocks[r] + place + ((int)slots[r] & (C4_TOKENS - 1)); };
    const uint32_t* w = reinterpret_cast<const uint32_t*>(from);
    if ((in16 >> r0 & 0xffffu) == 0xffffu) {
      *reinterpret_cast<uint4*>(at(r0)) = make_uint4(w[0], w[1], w[2], w[3]);
      continue;
    }
    for (int k = 0; k < 16; k += 4) {
      if ((in4 >> (r0 + k) & 15u) == 15u) {
        *reinterpret_cast<uint32_t*>(at(r0 + k)) = w[k / 4];
        continue;
      }
      for (int n = k; n < k + 4; ++n)
        if (slots[r0 + n] >= 0) *at(r0 + n) = from[n];
    }
  }
}

// The entries that the cache holds at `slot`: k T [M][G][dim], v T [M][G][vdim]; slots outside the cache give zeros. Half a warp per row and
// head, a lane for eight entries (of a value: four bytes 64 apart, entries 8 apart in their halves). A CTA has rows of one head: they share the sectors of the
// values' bytes where their slots are neighbours: 8192 rows of 8 heads in 15 us, 24 with the heads of a row together.
constexpr int R4_ROWS = 8;                                 // of a CTA

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
__global__ void __launch_bounds__(16 * R4_ROWS) fl_read4_kernel(const Cache4 c, const i64* slot, T* k, T* v, int M) {
  launch_next();
  wait_previous();
  const i64 m = (i64)blockIdx.x * R4_ROWS + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15, g = blockIdx.y;
  if (m >= M) return;
  const i64 s = slot[m], at = m * c.G + g;
  const bool in = c.has(s);
  const int tok = in ? (int)(s & (C4_TOKENS - 1)) : 0;
  const uint8_t* b = c.block(in ? s : 0, g);
  const float pk = in ? __int_as_float(b[c.key_exp(tok)] << 23) : 0.0f, pv = in ? __int_as_float(b[c.value_exp(tok)] << 23) : 0.0f;
  // bytes of two codes each -> their entries, x of the low codes and y of the high ones
  auto entries = [&](uint32_t codes, uint32_t scale, float power, float (&x)[4], float (&y)[4]) {
    uint32_t h[4];
    e2m1_pairs(codes, h);
    const uint32_t f = e4m3_pair((scale & 127) * 0x0101u);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t w = hmul2(h[q], f);
      const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&w));
      x[q] = in ? z.x * power : 0.0f, y[q] = in ? z.y * power : 0.0f;
    }
  };
  float x[4], y[4];
  for (int d = 8 * l; d < c.dim; d += 128) {
    entries(*reinterpret_cast<const uint32_t*>(b + tok * (c.K / 2) + d / 2), b[c.key_scale(tok, d / 16)], pk, x, y);
    c4_put(k + at * c.dim, d, c.dim, {x[0], y[0], x[1], y[1]});
    c4_put(k + at * c.dim, d + 4, c.dim, {x[2], y[2], x[3], y[3]});
  }
  for (int d = 16 * (l / 2) + 4 * (l & 1); d < c.vdim; d += 128) {
    const uint8_t* from = b + c.value_code(tok, d / 16, d % 8);
    const uint32_t lo = __byte_perm(from[0], from[C4_TOKENS], 0x0040), hi = __byte_perm(from[2 * C4_TOKENS], from[3 * C4_TOKENS], 0x0040);
    entries(__byte_perm(lo, hi, 0x5410), b[c.value_scale(tok, d / 16)], pv, x, y);
    c4_put(v + at * c.vdim, d, c.vdim, x);
    c4_put(v + at * c.vdim, d + 8, c.vdim, y);
  }
}

}  // namespace bxf
