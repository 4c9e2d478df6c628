// Attention over a paged cache on the tensor cores (bf16 cache, fp32 scores and softmax), one kernel for prompts and decoding.
//
// A tile is up to 128 query rows = (consecutive tokens of one sequence) x (heads of one group): all of them read the same
// cache rows, so a block of 64 rows is staged once for 128 queries. Scores Q K^T: A = Q tile [128 x W], B = the rows' keys,
// both K-major. P V: the values are staged row by row like the keys and read as an MN-major B operand (their rows are the
// contraction index), so nothing is transposed; in latent attention they are the first R entries of the staged keys
// themselves and nothing is loaded twice. A = P comes from TMEM, where
// the softmax warps leave it as bf16 in place of the scores. TMEM: two score buffers of 64 columns, then the output
// accumulator (256 columns; a wider latent is cut into value slices over blockIdx.z).
//
// Warp 0 = TMA, warp 1 = MMA, the others = softmax: a query row is shared by PARTS threads (one per warp of its TMEM lane
// quarter), 64 / PARTS of the 64 keys each; a decoding tile fills one quarter only, and a single warp per row would be bound
// by its own latency. PARTS = 4: one CTA per SM. PARTS = 2 for values of up to 128 entries: half the TMEM and half the threads,
// so that two CTAs share an SM and the scores -> softmax -> values chain of one tile runs beside the other's. The running maximum starts at the sink (denominator 1); the accumulator is rescaled only when the maximum
// grows by more than 2^8 since the last time. Few tiles (decoding): the keys of a tile are split over blockIdx.y, and a
// second kernel joins the parts.
//
// A 4-bit cache (FOUR; fl_cache4.cuh): the softmax warps also make the fp16 operands of the next block in shared memory from its codes,
// in front of a block's softmax, so that its scores are computed meanwhile. A raw block arrives by one bulk copy; keys become
// K-major rows as a TMA copy would leave them, values, whose codes lie along the tokens, a K-major V^T. An entry is its code times its
// scale times 2^(e - E), with E the largest exponent of the block's keys (it goes into the scores) or values (it goes into the weights,
// relative to the largest exponent of the values that the row has seen; the accumulator is rescaled when that grows): exact for
// tokens within 2^14 of the largest one. Values beyond are off by less than 2^-32 of that one's largest entry (a scale by 2^-25, times a
// code of up to 6, and the product by 2^-25; the entry is at least 2^10). A token that only some rows see must not cost
// the others their digits, nor a large key the scores of small ones: blocks where that could be have operands without the powers of two,
// which then go into every score and weight on its own, in 32 bits. Weights are held times 2^6 in fp16: off by 2^-12 of themselves or
// 2^-31, the larger of the two, so a token whose power of two went into its weight is off by less than 2^-30 of the largest one's largest entry.
// The queries are turned to fp16 in place, each row times a power of two. It is for tiles of
// many query rows, which share that work; short tiles have the kernel of fl_attention4.cuh, and each of the two leaves the
// other's tiles alone. (Two or four warps of their own for the operands were slower: they were a chain of latencies of 4200 cycles a
// block, where eight warps with other work beside it take turns.)
#pragma once

#include "fl_attention4.cuh"
#include "fl_gemm.cuh"

#include <type_traits>

namespace bxf {

constexpr int LT_KEYS = 64, LT_MAX_STAGES = 4, LT_MAX_SPLIT = 8, LT_VCOLS = 256;
constexpr int LT_O = 2 * LT_KEYS;                        // first TMEM column of the output accumulator
constexpr float LT_LOG2E = 1.4426950408889634f;
constexpr float LT_GROWTH = 8.0f;

struct LatentTc {
  int cols, kcols, vbox;                                 // 64-entry column blocks of a staged row, of its key; first one of its value
  int stages, qrows;                                     // key stages of the ring, rows of the Q box
  int row_blocks, vsplit;                                // blockIdx.z = (group * vsplit + value slice) * row_blocks + row block
  int splits;
  float* part;                                           // splits > 1: [splits][M G H][R] accumulators, then [splits][M G H][2]
  int min_rows;                                          // FOUR: tiles of fewer query rows are another kernel's
};

template <bool FOUR = false>
struct LatentShared {
  static constexpr int SHARE = FOUR ? 2 : 4;             // threads of a query row

  uint64_t q_full, o_done;
  uint64_t full[LT_MAX_STAGES], empty[LT_MAX_STAGES], raw_full;
  uint64_t s_full[2], p_full[2], pv_done[2];
  float row_max[2][SHARE][128], row_den[SHARE][128];
  uint64_t q_ready, raw_empty;                           // FOUR: the queries are fp16; the raw block is used
  uint32_t tmem_base, abort_flag;
};

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// The PARTS warps of a lane quarter.
template <int PARTS>
__device__ __forceinline__ void quarter_barrier(int quarter) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + quarter), "n"(32 * PARTS) : "memory");
}
__host__ __device__ constexpr int lt_threads(int parts) { return 64 + 128 * parts; }

// A pair of fp16 scales times 2^-u, u in the halves of a word; deep: some u is beyond 14, where 2^-u is no normal fp16 any more.
__device__ __forceinline__ uint32_t scaled_down(uint32_t scale, uint32_t u, bool deep) {
  const uint32_t near = __vminu2(u, 0x000e000eu);
  scale = hmul2(scale, (0x000f000fu - near) << 10);
  if (deep) scale = hmul2(scale, (0x000f000fu - __vminu2(u - near, 0x000f000fu)) << 10);
  return scale;
}

// One block's keys, by T threads: thread (row, 32 entries) writes four chunks of 16 bytes where a 128-byte-swizzled copy would put
// them. E = 0: without the powers of two; else no row that is seen is more than 2^14 below E. What is read comes first: a load is not
// moved in front of a store that might be to the same place.
template <int T>
__device__ __forceinline__ void operand_keys(const uint8_t* __restrict__ raw, uint8_t* __restrict__ st, const Cache4& c, int E, int tid) {
  const int r = tid % LT_KEYS;
  const uint32_t down = (E - min((int)raw[c.key_exp(r)], E)) * 0x00010001u;
  for (int part = tid / LT_KEYS; part < c.K / 32; part += T / LT_KEYS) {
    const uint4 v = *reinterpret_cast<const uint4*>(raw + r * (c.K / 2) + part * 16);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t scale[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) scale[j] = (raw[c.key_scale(r, part * 2 + j)] & 127) * 0x0101u;
#pragma unroll
    for (int j = 0; j < 2; ++j) scale[j] = scaled_down(e4m3_pair(scale[j]), down, false);
    uint8_t* row = st + part / 2 * (LT_KEYS * 128) + r * 128;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t h[4];
      e2m1_pairs(w[k], h);
      *reinterpret_cast<uint4*>(row + (((part % 2 * 4 + k) ^ (r & 7)) << 4)) =
          make_uint4(hmul2(h[0], scale[k / 2]), hmul2(h[1], scale[k / 2]), hmul2(h[2], scale[k / 2]), hmul2(h[3], scale[k / 2]));
    }
  }
}
// Its values as V^T: thread (byte column, 16 tokens) writes two runs of 16 tokens, of entries 16 j + i and 16 j + i + 8. deep: some row is
// more than 2^14 below E.
template <int T>
__device__ __forceinline__ void operand_values(const uint8_t* __restrict__ raw, uint8_t* __restrict__ st, const Cache4& c, int E, bool deep, int tid) {
  const int columns = c.V / 2;                           // 32 or 64
  const uint32_t most = (uint32_t)E * 0x00010001u;
  for (int u = tid; u < columns * 4; u += T) {
    const int col = u & (columns - 1), t0 = u / columns * 16, j = col / 8, i = col % 8;
    const uint4 vc = *reinterpret_cast<const uint4*>(raw + 36 * c.K + col * C4_TOKENS + t0);
    const uint4 vs = *reinterpret_cast<const uint4*>(raw + 36 * c.K + 32 * c.V + j * C4_TOKENS + t0);
    const uint4 ve = *reinterpret_cast<const uint4*>(raw + 36 * (c.K + c.V) + C4_TOKENS + t0);
    const uint32_t cw[4] = {vc.x, vc.y, vc.z, vc.w}, sw[4] = {vs.x, vs.y, vs.z, vs.w}, ew[4] = {ve.x, ve.y, ve.z, ve.w};
    uint8_t* row = st + (16 * j + i) * 128;
#pragma unroll
    for (int k = 0; k < 2; ++k) {                        // 8 tokens: a chunk of 16 bytes for each of the two entries
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t h[4];
        e2m1_pairs(cw[2 * k + q], h);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t e = __vminu2(__byte_perm(ew[2 * k + q], 0, x ? 0x4342 : 0x4140), most);
          const uint32_t scale = scaled_down(e4m3_pair(sw[2 * k + q] >> (16 * x)), most - e, deep);
          lo[2 * q + x] = hmul2(__byte_perm(h[2 * x], h[2 * x + 1], 0x5410), scale);
          hi[2 * q + x] = hmul2(__byte_perm(h[2 * x], h[2 * x + 1], 0x7632), scale);
        }
      }
      const int at = (t0 / 8 + k ^ i) << 4;              // 16 j + i and + 8 are alike modulo 8
      *reinterpret_cast<uint4*>(row + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      *reinterpret_cast<uint4*>(row + 8 * 128 + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    }
  }
}
// The 64 entries of a query row in one column box: their largest magnitude, and then bf16 -> fp16 times up * up2. Chunks are taken in an order
// that spreads the rows of a warp over the banks.
__device__ __forceinline__ float query_most(const uint8_t* row, int r) {
  float most = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + (((k + r) & 7) << 4));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int x = 0; x < 4; ++x)
      most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w[x] << 16)), fabsf(__uint_as_float(w[x] & 0xffff0000u))));
  }
  return most;
}
__device__ __forceinline__ void query_to_half(uint8_t* row, int r, float up, float up2) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint4* at = reinterpret_cast<uint4*>(row + (((k + r) & 7) << 4));
    uint32_t w[4] = {at->x, at->y, at->z, at->w};
#pragma unroll
    for (int x = 0; x < 4; ++x)
      w[x] = pack_half(__uint_as_float(w[x] << 16) * up * up2, __uint_as_float(w[x] & 0xffff0000u) * up * up2);
    *at = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// D (+)= A[tmem] * B[smem]; A: bf16 pairs, one row per lane.
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// MN-major operand in 128-byte-swizzled boxes of 64 entries x LT_KEYS rows: 8 contraction rows are 1024 bytes apart, the
// next 64 entries one box further on.
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t addr) {
  uint64_t d = umma_desc_sw128(addr);
  d &= ~(static_cast<uint64_t>(0x3FFF) << 16);
  return d | static_cast<uint64_t>((LT_KEYS * 128) >> 4) << 16;
}

template <int PARTS, bool FOUR = false>
__global__ void __launch_bounds__(lt_threads(PARTS), PARTS == 2 ? 2 : 1)
fl_paged_attention_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mc,
                             const PagedAttn a, const LatentTc c, const Cache4 c4) {
  constexpr int TCOLS = PARTS == 2 ? 256 : 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* qs = align_smem(smem_raw);
  const int q_box = c.qrows * 128;                       // bytes of a column block of the queries
  uint8_t* ring = qs + c.kcols * q_box;
  const int stage_bytes = c.cols * LT_KEYS * 128;
  using Shared = LatentShared<FOUR>;
  static_assert(PARTS <= Shared::SHARE, "threads of a row");
  Shared* sh = reinterpret_cast<Shared*>(ring + c.stages * stage_bytes);
  uint8_t* raw = reinterpret_cast<uint8_t*>(sh) + (sizeof(Shared) + 15) / 16 * 16;           // FOUR: a block as it is in the cache, and
  uint8_t* exps = raw + c4.bytes();                      // the exponents [parity of the block][keys, values][64] of blocks without them
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  wait_previous();

  // ---- the tile ----
  int tok0, ntok;
  i64 seq;
  if (a.tiles) {
    // (FOUR: from the end, where the long contexts of a prompt are, so that the last tiles to be done are short ones)
    const int* t = a.tiles + (i64)(FOUR ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * 3;
    seq = t[0];
    tok0 = t[1];
    ntok = t[2];
  } else {
    tok0 = blockIdx.x;
    ntok = 1;
    seq = a.seq[tok0];
  }
  const int row0 = (blockIdx.z % c.row_blocks) * 128, rows = min(128, ntok * a.H - row0);
  const int slice = blockIdx.z / c.row_blocks, group = slice / c.vsplit;
  const int v0 = slice % c.vsplit * LT_VCOLS, vn = min(LT_VCOLS, a.R - v0);
  const i64 limit = (i64)a.nblk * a.bs - 1;
  const i64 p_first = min(a.pos[tok0], limit), p_last = min(a.pos[tok0 + ntok - 1], limit);
  const int b_lo = a.first_key(p_first) / LT_KEYS, b_hi = (int)(p_last / LT_KEYS) + 1;
  const int b0 = b_lo + (b_hi - b_lo) * (int)blockIdx.y / c.splits, b1 = b_lo + (b_hi - b_lo) * ((int)blockIdx.y + 1) / c.splits;
  const int nb = b1 - b0;
  if (rows <= 0) return;
  if (FOUR && ntok * a.H < c.min_rows) return;
  const int quarters = (rows + 31) / 32;                 // TMEM lane quarters in use

  if (threadIdx.x == 0) {
    mbar_init(&sh->q_full, 1);
    mbar_init(&sh->o_done, 1);
    for (int i = 0; i < c.stages; ++i) {
      mbar_init(&sh->full[i], FOUR ? 4 * PARTS : 1);
      mbar_init(&sh->empty[i], 1);
    }
    mbar_init(&sh->raw_full, 1);
    mbar_init(&sh->raw_empty, 4 * PARTS);
    mbar_init(&sh->q_ready, PARTS * quarters);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->p_full[i], PARTS * quarters);
      mbar_init(&sh->pv_done[i], 1);
    }
    sh->abort_flag = *reinterpret_cast<volatile int*>(&g_wait_timeouts) != 0;
    fence_barrier_init();
    tma_prefetch_desc(&mq);
    tma_prefetch_desc(&mc);
  }
  __syncthreads();
  if (warp == 1) {
    tmem_alloc(&sh->tmem_base, TCOLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  launch_next();                                         // after the TMEM allocation
  const uint32_t tmem = sh->tmem_base;
  const bool dead = sh->abort_flag != 0;
  __syncthreads();

  auto fail = [&] {
    atomicAdd(&g_wait_timeouts, 1);
    *reinterpret_cast<volatile uint32_t*>(&sh->abort_flag) = 1;
  };

  if (dead) {
  } else if (warp == 0) {
    // ---- TMA: the queries once, then the key blocks in boxes that lie in one page. The warp reads the block table for 32
    //      boxes at a time; one lane issues the copies ----
    if (nb > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&sh->q_full, c.kcols * q_box);
        for (int j = 0; j < c.kcols; ++j)
          tma_load_3d(qs + j * q_box, &mq, &sh->q_full, j * 64, tok0 * a.H + row0, group);
      }
      const int box = min(a.bs, LT_KEYS), boxes = LT_KEYS / box;
      int i = 0, held = 0;
      bool ok = true;
      for (; !FOUR && i < nb; ++i) {
        const int s = i % c.stages, round = i / c.stages;
        if (round > 0) ok = mbar_wait(&sh->empty[s], (round - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* st = ring + s * stage_bytes;
        if (lane == 0) mbar_arrive_expect_tx(&sh->full[s], stage_bytes);
        for (int p = 0; p < boxes; ++p) {
          const int nth = i * boxes + p;                             // box of this CTA
          if ((nth & 31) == 0) {
            const int page = (b0 * LT_KEYS + (nth + lane) * box) / a.bs;
            held = (int)a.page_of(seq, min(page, a.nblk - 1)) * a.G + group;
          }
          const int page = __shfl_sync(0xffffffffu, held, nth & 31);
          if (lane == 0)
            for (int j = 0; j < c.cols; ++j)
              tma_load_3d(st + j * LT_KEYS * 128 + p * box * 128, &mc, &sh->full[s],
                          j < c.kcols ? j * 64 : a.voff + (j - c.kcols) * 64, (b0 * LT_KEYS + nth * box) % a.bs, page);
        }
      }
      // FOUR: the raw blocks, one at a time
      for (; FOUR && i < nb; ++i) {
        if (i > 0) ok = mbar_wait(&sh->raw_empty, (i - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int in_page = a.bs / LT_KEYS, bytes = c4.bytes();
        if ((i & 31) == 0) held = (int)a.page_of(seq, min((b0 + i + lane) / in_page, a.nblk - 1));
        const i64 page = __shfl_sync(0xffffffffu, held, i & 31);
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh->raw_full, bytes);
          bulk_load(raw, c4.p + ((page * a.G + group) * in_page + (b0 + i) % in_page) * bytes, &sh->raw_full, bytes);
        }
      }
      if (FOUR && !ok && lane == 0) {
        fail();
        mbar_wait(&sh->q_full, 0);
        if (i > 0) mbar_wait(&sh->raw_full, (i - 1) & 1);
      }
      if (!FOUR && !ok && lane == 0) {
        fail();
        mbar_wait(&sh->q_full, 0);
        for (int k = i > c.stages ? i - c.stages : 0; k < i; ++k) mbar_wait(&sh->full[k % c.stages], (k / c.stages) & 1);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && nb > 0) {
      // ---- MMA: scores of block i + 1 are issued before the values of block i. A query box of fewer than 128 rows is
      //      read on into what follows it in shared memory: those accumulator lanes belong to no query ----
      constexpr uint32_t HALF = FOUR ? (1u << 7) | (1u << 10) : 0u;        // the operands' type bits: bf16 set, fp16 clear
      constexpr uint32_t ID_S = umma_idesc_bf16(LT_KEYS) ^ HALF;
      const uint32_t id_v = umma_idesc_bf16((vn + 15) / 16 * 16, !FOUR) ^ HALF;
      auto scores = [&](int i) {
        const int s = i % c.stages, buf = i & 1;
        if (!mbar_wait(&sh->full[s], (i / c.stages) & 1)) return false;
        if (i >= 2 && !mbar_wait(&sh->pv_done[buf], ((i >> 1) - 1) & 1)) return false;   // P of block i - 2 is read
        tc_fence_after();
        const uint32_t qa = smem_u32(qs), ka = smem_u32(ring + s * stage_bytes);
        for (int j = 0; j < c.kcols; ++j)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_bf16(tmem + buf * LT_KEYS, umma_desc_sw128(qa + j * q_box + ks * 32),
                      umma_desc_sw128(ka + j * LT_KEYS * 128 + ks * 32), ID_S, (j | ks) != 0);
        umma_commit(&sh->s_full[buf]);
        return true;
      };
      bool ok = mbar_wait(FOUR ? &sh->q_ready : &sh->q_full, 0) && scores(0);
      for (int i = 0; i < nb && ok; ++i) {
        const int s = i % c.stages, buf = i & 1;
        if (c.stages > 1 && i + 1 < nb && !(ok = scores(i + 1))) break;
        if (!(ok = mbar_wait(&sh->p_full[buf], (i >> 1) & 1))) break;
        tc_fence_after();
        const uint32_t va = smem_u32(ring + s * stage_bytes) + (c.vbox + v0 / 64) * LT_KEYS * 128;
#pragma unroll
        for (int ks = 0; ks < LT_KEYS / 16; ++ks)
          umma_bf16_ts(tmem + LT_O, tmem + buf * LT_KEYS + ks * 8, FOUR ? umma_desc_sw128(va + ks * 32) : umma_desc_mn(va + ks * 2048), id_v, (i | ks) != 0);
        umma_commit(&sh->pv_done[buf]);
        umma_commit(&sh->empty[s]);
        if (c.stages == 1 && i + 1 < nb) ok = scores(i + 1);             // one stage: nothing to run ahead into
      }
      if (ok) umma_commit(&sh->o_done);
      else fail();
    }
  } else if (FOUR || (warp & 3) < quarters) {
    // ---- softmax. A wait that gives up is remembered and the loop goes on (the quarter's barriers count every warp) ----
    constexpr int KW = LT_KEYS / PARTS;
    const int quarter = warp & 3, part = (warp - 2) >> 2, r = quarter * 32 + lane;
    const bool live = r < rows;
    const int flat = row0 + (live ? r : 0), token = tok0 + flat / a.H, head = group * a.H + flat % a.H;
    const i64 pos = min(a.pos[token], limit);
    const int lo = a.first_key(pos), hi = (int)pos;
    constexpr float UNIT = FOUR ? 64.0f : 1.0f;          // what a weight of 1 is held as
    constexpr float SHIFT = FOUR ? 6.0f : 0.0f;
    float scale = a.scale * LT_LOG2E;
    float ref = a.sink ? a.sink[head] * LT_LOG2E : -INFINITY;
    float den = (FOUR ? ref != -INFINITY : a.sink != nullptr) && blockIdx.y == 0 && part == 0 ? UNIT : 0.0f;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    bool ok = true;
    // ---- FOUR: the operands of a block ----
    const bool used = (warp & 3) < quarters;             // the others have no queries and only help with the operands
    // keys that some row sees, that every row sees
    const int seen_lo = a.first_key(p_first), seen_hi = (int)p_last, whole_lo = a.first_key(p_last), whole_hi = (int)p_first;
    int E = 0;                                           // of the accumulator: the largest of the values that the row has seen
    // Of the keys and values of this block, and of the next one; keys' 0: the block's operands are without the powers of two. Those of values
    // stay as they were from block to block while that costs at most FEW bits.
    constexpr int FEW = 4;
    int k_exp = 0, v_exp = 0, k_exp_next = 0, v_exp_next = 0;
    auto operands = [&](int i) {
      if (ok) ok = mbar_wait(&sh->raw_full, i & 1) && (i < 2 || mbar_wait(&sh->s_full[i & 1], ((i >> 1) - 1) & 1));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      // exponents of the tokens that some row of the tile sees
      unsigned k_most = 0, v_most = 0, k_least = 255, v_least = 255;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = lane + 32 * h;
        const int key = (b0 + i) * LT_KEYS + t;
        if (key < seen_lo || key > seen_hi) continue;
        const unsigned ke = raw[c4.key_exp(t)], ve = raw[c4.value_exp(t)];
        k_most = max(k_most, ke), v_most = max(v_most, ve), k_least = min(k_least, ke), v_least = min(v_least, ve);
      }
      k_exp_next = (int)__reduce_max_sync(0xffffffffu, k_most), k_least = __reduce_min_sync(0xffffffffu, k_least);
      v_most = __reduce_max_sync(0xffffffffu, v_most), v_least = __reduce_min_sync(0xffffffffu, v_least);
      const int first = (b0 + i) * LT_KEYS;
      if (k_exp_next > (int)k_least + 14 || v_most > v_least + FEW && (first < whole_lo || first + LT_KEYS - 1 > whole_hi)) k_exp_next = 0;
      else if ((int)v_most > v_exp_next || v_exp_next > (int)v_least + FEW) v_exp_next = (int)v_most;
      uint8_t* st = ring + i % c.stages * stage_bytes;
      operand_keys<128 * PARTS>(raw, st, c4, k_exp_next, threadIdx.x - 64);
      if (i >= 2) ok = mbar_wait(&sh->pv_done[i & 1], ((i >> 1) - 1) & 1);             // the values of block i - 2 are used
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      operand_values<128 * PARTS>(raw, st + c.kcols * LT_KEYS * 128, c4, k_exp_next ? v_exp_next : 0, k_exp_next && v_most > v_least + 14,
                                  threadIdx.x - 64);
      if (k_exp_next == 0 && warp == 2)                          // (block i - 2 is done with: its values are used)
        *reinterpret_cast<uint32_t*>(exps + (i & 1) * 2 * C4_TOKENS + 4 * lane) = *reinterpret_cast<const uint32_t*>(raw + 36 * (c4.K + c4.V) + 4 * lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh->full[i % c.stages]);
        mbar_arrive(&sh->raw_empty);
      }
    };
    float row_scale = scale;
    if (FOUR && nb > 0) {
      if (used) {
        ok = mbar_wait(&sh->q_full, 0);
        float most = 0.0f;
        for (int box = part; ok && r < c.qrows && box < c.kcols; box += PARTS) most = fmaxf(most, query_most(qs + box * q_box + r * 128, r));
        sh->row_max[0][part][r] = most;
        quarter_barrier<PARTS>(quarter);
#pragma unroll
        for (int k = 0; k < PARTS; ++k) most = fmaxf(most, sh->row_max[0][k][r]);
        const int e = a4_query_exponent(most), back = e - A4_BIAS;
        const float up = c4_power(-back / 2), up2 = c4_power(-back - -back / 2);
        for (int box = part; ok && r < c.qrows && box < c.kcols; box += PARTS) query_to_half(qs + box * q_box + r * 128, r, up, up2);
        row_scale = scale * c4_power(back / 2) * c4_power(back - back / 2);
        ok = __all_sync(0xffffffffu, ok);
        fence_proxy_async_smem();
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&sh->q_ready);
        quarter_barrier<PARTS>(quarter);                   // row_max is used again
      }
      operands(0);
      k_exp = k_exp_next, v_exp = v_exp_next;
    }
    // own (FOUR): the block's operands are without the powers of two, or its values' is below E; the weights take them. Seldom so, and kept out
    // of the usual case, which is a chain of latencies (394 against 382 us for four prompts of 2048 tokens).
    auto softmax = [&](int i, auto own) {
      constexpr bool OWN = decltype(own)::value;
      const int buf = i & 1;
      ok = ok && mbar_wait(&sh->s_full[buf], (i >> 1) & 1);
      __syncwarp();
      tc_fence_after();
      uint32_t u[KW];
#pragma unroll
      for (int k = 0; k < KW; k += 16) tmem_ld16(tmem + lanes + buf * LT_KEYS + part * KW + k, *reinterpret_cast<uint32_t(*)[16]>(u + k));
      tmem_ld_wait();
      float f = 1.0f;
      const bool bare = OWN && k_exp == 0;
      if (FOUR) scale = row_scale * c4_power(max(k_exp, 1) - 127);
      const int k0 = (b0 + i) * LT_KEYS + part * KW;
      const uint8_t* block_exps = exps + buf * 2 * C4_TOKENS;
      float s[KW], mx = -INFINITY;
      if (bare) {
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          s[k] = k0 + k >= lo && k0 + k <= hi ? __uint_as_float(u[k]) * (row_scale * c4_power(block_exps[part * KW + k] - 127)) : -INFINITY;
          mx = fmaxf(mx, s[k]);
        }
      } else if (k0 >= lo && k0 + KW - 1 <= hi) {
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          s[k] = __uint_as_float(u[k]) * scale;
          mx = fmaxf(mx, s[k]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          s[k] = k0 + k >= lo && k0 + k <= hi ? __uint_as_float(u[k]) * scale : -INFINITY;
          mx = fmaxf(mx, s[k]);
        }
      }
      sh->row_max[buf][part][r] = mx;
      tc_fence_before();
      quarter_barrier<PARTS>(quarter);                     // the quarter's scores are in registers: P may replace them
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < PARTS; ++k) mx = fmaxf(mx, sh->row_max[buf][k][r]);
      if (FOUR && k0 - part * KW <= hi && k0 - part * KW + LT_KEYS > lo) {       // the row sees some of the block
        int e = v_exp;
        if (bare) {
          e = 0;
          for (int k = 0; k < LT_KEYS; ++k)
            if (k0 - part * KW + k >= lo && k0 - part * KW + k <= hi) e = max(e, (int)block_exps[C4_TOKENS + k]);
        }
        if (e > E) {
          if (E != 0) f = c4_power(max(E - e, -126));
          E = e;
        }
      }
      float g = 1.0f;
      if (mx > ref + LT_GROWTH || ref == -INFINITY) {
        g = ref == -INFINITY ? 0.0f : exp2_fast(ref - mx);
        ref = mx;
      }
      den *= g;
      f = FOUR ? f * g : g;
      if (__any_sync(0xffffffffu, f != 1.0f && live)) {    // the same in the four warps of the quarter
        if (i > 0) {
          // the accumulator may be touched once the values of block i - 1 are in
          ok = ok && mbar_wait(&sh->pv_done[buf ^ 1], ((i - 1) >> 1) & 1);
          __syncwarp();
          tc_fence_after();
          for (int q = part * 16; q < vn; q += 16 * PARTS) {
            uint32_t o[16];
            tmem_ld16(tmem + lanes + LT_O + q, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st16(tmem + lanes + LT_O + q, o);
          }
        }
      }
      const float base = ref == -INFINITY ? 0.0f : ref - SHIFT;            // no visible key yet: every weight is 0
      float d0 = 0.0f, d1 = 0.0f;
      uint32_t w[KW / 2];
#pragma unroll
      for (int k = 0; k < KW / 2; ++k) {
        const float e0 = exp2_fast(s[2 * k] - base), e1 = exp2_fast(s[2 * k + 1] - base);
        d0 += e0;
        d1 += e1;
        if constexpr (OWN) {                               // the values' power of two in 32 bits: rounded once, with the weight
          const uint8_t* e = block_exps + C4_TOKENS + part * KW + 2 * k;
          w[k] = pack_half(e0 * c4_power(max(min((bare ? e[0] : v_exp) - E, 0), -126)), e1 * c4_power(max(min((bare ? e[1] : v_exp) - E, 0), -126)));
        } else {
          w[k] = FOUR ? pack_half(e0, e1) : pack_bf16(e0, e1);
        }
      }
      den += d0 + d1;
#pragma unroll
      for (int k = 0; k < KW / 2; k += 8)
        tmem_st8(tmem + lanes + buf * LT_KEYS + part * (KW / 2) + k, *reinterpret_cast<const uint32_t(*)[8]>(w + k));
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->p_full[buf]);
    };
    for (int i = 0; i < nb; ++i) {
      if (FOUR && i + 1 < nb) operands(i + 1);
      if (!FOUR) {
        softmax(i, std::false_type{});
      } else if (used) {
        if (__any_sync(0xffffffffu, k_exp == 0 || v_exp < E)) softmax(i, std::true_type{});
        else softmax(i, std::false_type{});
        k_exp = k_exp_next, v_exp = v_exp_next;
      }
    }
    if (nb > 0) ok = ok && mbar_wait(&sh->o_done, 0);
    ok = __all_sync(0xffffffffu, ok);
    sh->row_den[part][r] = den;
    quarter_barrier<PARTS>(quarter);
    den = 0.0f;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) den += sh->row_den[k][r];
    if (!ok) {
      if (lane == 0) fail();
    } else {
      tc_fence_after();
      const i64 n = (i64)a.M * a.H * a.G, at = (i64)token * a.H * a.G + head;
      // outputs in units of 1; where a kernel behind joins parts, of the weights (FOUR: times A4_HEADROOM)
      const float units = FOUR && E != 0 ? c4_power(max(E - 127, -126)) : 1.0f;
      float inv = c.splits == 1 ? units / den : units * (FOUR ? A4_HEADROOM / UNIT : 1.0f);
      if (FOUR && c.splits == 1 && den == 0.0f) inv = 0.0f;                // a row that sees nothing
      float* acc = c.part + (blockIdx.y * n + at) * a.R + v0;
      bf16* out = static_cast<bf16*>(a.out) + token * a.out_tok + head * a.out_head + v0;
      for (int q = part * 16; q < vn; q += 16 * PARTS) {
        uint32_t u[16] = {};
        if (nb > 0) {
          tmem_ld16(tmem + lanes + LT_O + q, u);
          tmem_ld_wait();
        }
        if (!live) continue;
        const int cnt = min(16, vn - q);
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = __uint_as_float(u[k]) * inv;
        if (c.splits == 1) store_run(out + q, v, cnt);
        else store_run(acc + q, v, cnt);
      }
      if (c.splits > 1 && live && v0 == 0 && part == 0) {
        float* ml = c.part + c.splits * n * a.R + (blockIdx.y * n + at) * 2;
        ml[0] = ref;
        ml[1] = den / UNIT;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, TCOLS);
  }
}

// Joins the key splits: one CTA per query row (token, head). A part without a key has the sum 0 and no accumulators; one whose sum is NaN
// makes the row NaN, and a row that no part has a key for is 0. With tiles (of up to `tokens` tokens) blockIdx.x is (tile, token of it, head):
// rows in no tile, or in one of fewer than min_rows query rows, have no parts and are left as they are. unit: of the accumulators.
__global__ void __launch_bounds__(128) fl_attention_join_kernel(const PagedAttn a, const float* part, int splits, int tokens, int min_rows, float unit) {
  launch_next();
  wait_previous();
  const i64 heads = a.H * a.G, n = a.M * heads;
  i64 at = blockIdx.x;
  if (a.tiles) {
    const int *tile = a.tiles + at / (heads * tokens) * 3, nth = (int)(at / heads % tokens);
    if (nth >= tile[2] || tile[2] * a.H < min_rows) return;
    at = (tile[1] + nth) * heads + at % heads;
  }
  const float* ml = part + splits * n * a.R;
  float mx = -INFINITY, f[LT_MAX_SPLIT], den = 0.0f;
  for (int s = 0; s < splits; ++s)
    if (ml[(s * n + at) * 2 + 1] != 0.0f) mx = fmaxf(mx, ml[(s * n + at) * 2]);
#pragma unroll
  for (int s = 0; s < LT_MAX_SPLIT; ++s) {
    const float sum = s < splits ? ml[(s * n + at) * 2 + 1] : 0.0f;
    f[s] = sum != 0.0f ? exp2f(ml[(s * n + at) * 2] - mx) : 0.0f;
    if (f[s] != 0.0f || isnan(sum)) den += f[s] * sum;
  }
  const float inv = den == 0.0f ? 0.0f : unit / den;
  bf16* out = static_cast<bf16*>(a.out) + at / heads * a.out_tok + at % heads * a.out_head;
  for (int d = threadIdx.x; d < a.R; d += 128) {
    float o = 0.0f;
#pragma unroll
    for (int s = 0; s < LT_MAX_SPLIT; ++s)
      if (f[s] != 0.0f) o += f[s] * part[(s * n + at) * a.R + d];
    st(out + d, o * inv);
  }
}

}  // namespace bxf
