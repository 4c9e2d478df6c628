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
  __device__ __forceinline__ uint8_t* block(i64 slot, int g) const {
    return p + ((slot / page * G + g) * (page / C4_TOKENS) + slot % page / C4_TOKENS) * bytes();
  }
  __device__ __forceinline__ int key_scale(int tok, int j) const {
    return 32 * K + ((tok / 16 * 2 + tok % 2) * (K / 16) + j) * 8 + tok % 16 / 2;
  }
  __device__ __forceinline__ int value_code(int tok, int j, int i) const { return 36 * K + (j * 8 + i) * C4_TOKENS + tok; }
  __device__ __forceinline__ int value_scale(int tok, int j) const { return 36 * K + 32 * V + j * C4_TOKENS + tok; }
  __device__ __forceinline__ int key_exp(int tok) const { return 36 * (K + V) + tok; }
  __device__ __forceinline__ int value_exp(int tok) const { return 36 * (K + V) + C4_TOKENS + tok; }
};

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

// The smallest scale of which 6 steps reach `most` (below 2048): an estimate from below, and at most two steps up.
__device__ __forceinline__ int c4_scale_for(float most) {
  const float f = __fmul_rd(most, 0.16666666f);
  int c = f < 0.015625f ? (int)(f * 512.0f) : (__float_as_int(f) - (120 << 23)) >> 20;
  c += 6.0f * c4_scale(c) < most;
  c += 6.0f * c4_scale(c) < most;
  return c;
}
// The nearest code of x in steps of `step`: x is held against exact multiples of it.
__device__ __forceinline__ int c4_nearest(float x, float step) {
  const float m = fabsf(x);
  int c = (m > 0.25f * step) + (m >= 0.75f * step) + (m > 1.25f * step) + (m >= 1.75f * step) + (m > 2.5f * step) + (m >= 3.5f * step) +
          (m > 5.0f * step);
  if (step == 0.0f) c = 0;
  return x < 0.0f ? c | 8 : c;
}

// A warp's row: lane l holds entries 128 i + 4 l .. + 3.
struct C4Row {
  float x[C4_MAX / 128][4];
  bool bad;                            // of the lane's entries

  template <class T>
  __device__ __forceinline__ float load(const T* p, int n, int lane) {           // -> the largest finite magnitude of the row
    float most = 0.0f;
    bad = false;
#pragma unroll
    for (int i = 0; i < C4_MAX / 128; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int d = 128 * i + 4 * lane + k;
        float v = d < n ? ld(p + d) : 0.0f;
        if (!(fabsf(v) < INFINITY)) bad = true, v = 0.0f;
        x[i][k] = fminf(fmaxf(v, -1.7014118e38f), 1.7014118e38f);
        most = fmaxf(most, fabsf(x[i][k]));
      }
    return warp_max(most);
  }
  // Codes of the lane's four entries (4 bits each) and the scale of their block.
  __device__ __forceinline__ int codes(int i, float unit, int& scale) const {
    const float y[4] = {x[i][0] * unit, x[i][1] * unit, x[i][2] * unit, x[i][3] * unit};
    float most = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    scale = c4_scale_for(most);
    const float step = c4_scale(scale);
    int c = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) c |= c4_nearest(y[k], step) << (4 * k);
    return c;
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
template <class T, int ROWS>
__global__ void __launch_bounds__(S4_THREADS) fl_store4_kernel(const Store4<T> a) {
  constexpr int PITCH = ROWS + 4;      // bytes of a value column of the CTA's rows
  extern __shared__ __align__(16) uint8_t s4_smem[];
  __shared__ i64 slots[ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = blockIdx.y, row0 = blockIdx.x * ROWS;
  const Cache4& c = a.c;
  const i64 most_slots = (i64)c.nb * c.page;
  launch_next();
  wait_previous();
  if (threadIdx.x < ROWS) {
    const i64 s = row0 + (int)threadIdx.x < a.M ? a.slot[row0 + threadIdx.x] : -1;
    slots[threadIdx.x] = s >= 0 && s < most_slots ? s : -1;
  }
  __syncthreads();
  const int columns = c.V / 2 + c.V / 16 + 1;              // of value bytes: codes, scales, the exponent
  for (int r = warp; r < ROWS; r += S4_THREADS / 32) {
    if (slots[r] < 0) continue;
    const int m = row0 + r, tok = (int)(slots[r] % C4_TOKENS);
    uint8_t* block = c.block(slots[r], g);
    C4Row k, v;
    const float most_k = k.load(a.k + m * a.k_row + g * a.k_head, c.dim, lane);
    const float most_v = v.load(a.v + m * a.v_row + g * a.v_head, c.vdim, lane);
    const bool bad = __any_sync(0xffffffffu, k.bad || v.bad);
    const int ek = c4_exponent(most_k), ev = c4_exponent(most_v);
    const float uk = c4_power(-ek), uv = bad ? 0.0f : c4_power(-ev);
#pragma unroll
    for (int i = 0; i < C4_MAX / 128; ++i) {
      if (128 * i >= c.K) break;
      int scale;
      const int code = k.codes(i, uk, scale), d = 128 * i + 4 * lane;
      if (d < c.K) {
        *reinterpret_cast<uint16_t*>(block + tok * (c.K / 2) + d / 2) = (uint16_t)code;
        if ((lane & 3) == 0) block[c.key_scale(tok, d / 16)] = bad ? C4_NAN : scale;
      }
    }
#pragma unroll
    for (int i = 0; i < C4_MAX / 128; ++i) {
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
    auto at = [&](i64 s) { return c.block(s, g) + (col < columns - 1 ? 36 * c.K + col * C4_TOKENS : 36 * (c.K + c.V) + C4_TOKENS) + s % C4_TOKENS; };
    bool run = s0 >= 0 && s0 % 16 == 0;
#pragma unroll
    for (int k = 1; k < 16; ++k) run &= slots[r0 + k] == s0 + k;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(from);
    if (run) {
      *reinterpret_cast<uint4*>(at(s0)) = make_uint4(w[0], w[1], w[2], w[3]);
      continue;
    }
    for (int k = 0; k < 16; k += 4) {
      const i64 s = slots[r0 + k];
      if (s >= 0 && s % 4 == 0 && slots[r0 + k + 1] == s + 1 && slots[r0 + k + 2] == s + 2 && slots[r0 + k + 3] == s + 3) {
        *reinterpret_cast<uint32_t*>(at(s)) = w[k / 4];
        continue;
      }
      for (int n = k; n < k + 4; ++n)
        if (slots[r0 + n] >= 0) *at(slots[r0 + n]) = from[n];
    }
  }
}

// The entries that the cache holds at `slot`: k T [M][G][dim], v T [M][G][vdim]; slots outside the cache give zeros. A CTA per row and head.
template <class T>
__global__ void __launch_bounds__(128) fl_read4_kernel(const Cache4 c, const i64* slot, T* k, T* v, int M) {
  launch_next();
  wait_previous();
  const int m = blockIdx.x, g = blockIdx.y;
  const i64 s = slot[m], at = (i64)m * c.G + g;
  const bool in = s >= 0 && s < (i64)c.nb * c.page;
  const int tok = in ? (int)(s % C4_TOKENS) : 0;
  const uint8_t* b = c.block(in ? s : 0, g);
  const float pk = __int_as_float(b[c.key_exp(tok)] << 23), pv = __int_as_float(b[c.value_exp(tok)] << 23);
  for (int d = threadIdx.x; d < c.dim; d += 128) {
    const float x = c4_code(b[tok * (c.K / 2) + d / 2] >> (d % 2 * 4) & 15) * c4_scale(b[c.key_scale(tok, d / 16)] & 127) * pk;
    st(k + at * c.dim + d, in ? x : 0.0f);
  }
  for (int d = threadIdx.x; d < c.vdim; d += 128) {
    const float x = c4_code(b[c.value_code(tok, d / 16, d % 8)] >> (d % 16 / 8 * 4) & 15) * c4_scale(b[c.value_scale(tok, d / 16)] & 127) * pv;
    st(v + at * c.vdim + d, in ? x : 0.0f);
  }
}

}  // namespace bxf
