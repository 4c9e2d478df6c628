// The tables of a step's token rows from the requests' lengths, on the device: pages of finished requests go back to the pool, new
// ones are taken from it, and every row gets its request, position and cache slot.
//
// The pool is a stack of page numbers. Request b holds ceil(len / page) pages. Dropped requests push theirs in the order of the
// requests, a request's last page first; then every request takes ceil((len + n) / page) - ceil(len / page) pages, in the order of
// requests and positions. Nothing is taken or given back when something does not fit: the status tells what.
//
// One cluster of CTAs. Each CTA scans all requests' counts for itself (rows, pages pushed, pages taken: the running sums stay in
// shared memory), then rows and pages are dealt over all threads, which find their request by bisection: even work whatever the
// lengths. Inputs are read before the cluster's barrier and outputs written behind it, so that they may be the same memory. What
// bounds it is latency: a chain of three dependent loads (length, page of the table or the stack, store). 256 requests of one token take 5.4 us,
// 1000 with 59 thousand rows 12.6.
#pragma once

#include "bx_ptx.cuh"

namespace bx {

constexpr int ST_THREADS = 1024, ST_MAX_REQUESTS = 8192, ST_MAX_CLUSTER = 16;

struct StepTables {
  const long long *lens, *counts;
  const uint8_t* drop;                                     // NULL: no request is finished
  int* bt;
  long long bt_stride;
  int *free, *top, *status;
  long long *seq, *pos, *slot, *last, *lens_out;
  int* top_out;
  int B, nblk, page, pool, rows, sticky;
};

// First index of ends[0 .. n - 1] (non-decreasing) whose value exceeds i.
__device__ __forceinline__ int st_owner(const int* ends, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int st_pages(int n, int page) { return (int)(((unsigned)n + page - 1) / (unsigned)page); }

// Inclusive sums over a warp.
__device__ __forceinline__ void st_scan(long long& r, int& p, int& t, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long r2 = __shfl_up_sync(0xffffffffu, r, o);
    const int p2 = __shfl_up_sync(0xffffffffu, p, o), t2 = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) r += r2, p += p2, t += t2;
  }
}

// N rows from i on, of which those below `live` are tokens: what has to be looked up first, then the stores (a load is not moved in front
// of a store that might be to the same place). `full`: pages on the stack before any were taken.
template <int N>
__device__ __forceinline__ void st_rows(const StepTables& a, int i, int live, const int* row_end, const int* take_end, const int* base, int full) {
  int b = i < live ? st_owner(row_end, a.B, i) : 0, owner[N], pos[N], page[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    owner[k] = pos[k] = 0, page[k] = -1;
    if (i + k >= live) continue;
    while (row_end[b] <= i + k) ++b;
    const int start = base[b], held = st_pages(start, a.page);
    owner[k] = b;
    pos[k] = start + i + k - (b ? row_end[b - 1] : 0);
    const int block = (int)((unsigned)pos[k] / (unsigned)a.page);
    page[k] = block < held ? a.bt[b * a.bt_stride + block]
                           : *const_cast<volatile int*>(a.free + full - 1 - (b ? take_end[b - 1] : 0) - (block - held));
  }
  long long slot[N];
#pragma unroll
  for (int k = 0; k < N; ++k)
    slot[k] = i + k < live ? (long long)page[k] * a.page + pos[k] - (int)((unsigned)pos[k] / (unsigned)a.page) * a.page : -1;
  if (N % 2 == 0 && i + N <= a.rows && ((reinterpret_cast<uintptr_t>(a.seq) | reinterpret_cast<uintptr_t>(a.pos) | reinterpret_cast<uintptr_t>(a.slot)) & 15) == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      *reinterpret_cast<longlong2*>(a.seq + i + k) = make_longlong2(owner[k], owner[k + 1 < N ? k + 1 : k]);
      *reinterpret_cast<longlong2*>(a.pos + i + k) = make_longlong2(pos[k], pos[k + 1 < N ? k + 1 : k]);
      *reinterpret_cast<longlong2*>(a.slot + i + k) = make_longlong2(slot[k], slot[k + 1 < N ? k + 1 : k]);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (i + k < a.rows) a.seq[i + k] = owner[k], a.pos[i + k] = pos[k], a.slot[i + k] = slot[k];
}

__global__ void __launch_bounds__(ST_THREADS) step_tables_kernel(const StepTables a) {
  extern __shared__ int st_smem[];
  int* row_end = st_smem;                                  // running sums, [B] each
  int* push_end = row_end + a.B;
  int* take_end = push_end + a.B;
  int* base = take_end + a.B;                              // a request's length before its new tokens
  __shared__ long long warp_rows[32];
  __shared__ int warp_push[32], warp_take[32], bad_bits;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank, ctas;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  if (tid == 0) bad_bits = 0;
  wait_previous();
  launch_next();
  const long long most = (long long)a.nblk * a.page;
  const int top = *a.top;
  long long rows = 0;
  int push = 0, take = 0;
  for (int b0 = 0; b0 < a.B; b0 += ST_THREADS) {
    const int b = b0 + tid;
    long long n = 0;
    int gone = 0, need = 0, start = 0, bad = 0;
    if (b < a.B) {
      const long long len = a.lens[b];
      n = a.counts[b];
      const bool out = a.drop && a.drop[b];
      if (len < 0 || n < 0 || len > most) bad = BX_STEP_INVALID;
      else if ((out ? 0 : len) > most - n) bad = BX_STEP_TOO_LONG;
      if (bad) n = 0;
      else {
        start = out ? 0 : (int)len;
        gone = out ? st_pages((int)len, a.page) : 0;
        need = st_pages(start + (int)n, a.page) - st_pages(start, a.page);
      }
    }
    long long r = n;
    int p = gone, t = need;
    st_scan(r, p, t, lane);
    __syncthreads();                                       // bad_bits is set, the sums of the requests before are read
    if (bad) atomicOr(&bad_bits, bad);
    if (lane == 31) warp_rows[warp] = r, warp_push[warp] = p, warp_take[warp] = t;
    __syncthreads();
    // every warp sums up the warps' totals for itself
    long long wr = warp_rows[lane];
    int wp = warp_push[lane], wt = warp_take[lane];
    st_scan(wr, wp, wt, lane);
    const int before = max(warp - 1, 0);
    const long long br = __shfl_sync(0xffffffffu, wr, before);
    const int bp = __shfl_sync(0xffffffffu, wp, before), bt = __shfl_sync(0xffffffffu, wt, before);
    r += rows, p += push, t += take;
    if (warp > 0) r += br, p += bp, t += bt;
    rows += __shfl_sync(0xffffffffu, wr, 31);
    push += __shfl_sync(0xffffffffu, wp, 31);
    take += __shfl_sync(0xffffffffu, wt, 31);
    if (b < a.B) {
      row_end[b] = (int)min(r, 0x7fffffffll);
      push_end[b] = p;
      take_end[b] = t;
      base[b] = start;
    }
  }
  __syncthreads();
  int bad = bad_bits;
  if (top < 0 || top > a.pool - push) bad |= BX_STEP_INVALID;
  else if (take > top + push) bad |= BX_STEP_NO_PAGES;
  if (rows > a.rows) bad |= BX_STEP_TOO_MANY_ROWS;
  const int at = rank * ST_THREADS + tid, step = ctas * ST_THREADS;
  if (!bad)
    for (int i = at; i < push; i += step) {
      const int b = st_owner(push_end, a.B, i);
      a.free[top + i] = a.bt[b * a.bt_stride + push_end[b] - 1 - i];
    }
  // what is pushed is there for every CTA, and all inputs are read, before anything else is written
  if (ctas > 1) {
    if (push > 0) __threadfence();
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  const int full = top + push;
  if (rank == 0) {
    for (int b = tid; b < a.B; b += ST_THREADS) {
      const int n = row_end[b] - (b ? row_end[b - 1] : 0);
      if (!bad) a.lens_out[b] = base[b] + n;
      else if (a.lens_out != a.lens) a.lens_out[b] = a.lens[b];
      a.last[b] = !bad && n > 0 ? row_end[b] - 1 : -1;
    }
    if (tid == 0) {
      *a.top_out = bad ? top : full - take;
      *a.status = a.sticky ? *a.status | bad : bad;
    }
  }
  const volatile int* stack = a.free;                      // another CTA of the cluster may have pushed
  if (!bad)
    for (int i = at; i < take; i += step) {
      const int b = st_owner(take_end, a.B, i);
      const int nth = i - (b ? take_end[b - 1] : 0);
      a.bt[b * a.bt_stride + st_pages(base[b], a.page) + nth] = stack[full - 1 - i];
    }
  // few rows: one a thread; else runs of four, one bisection and mostly one page each
  const int live = bad ? 0 : (int)rows;
  if (a.rows <= 2 * step) {
    for (int i = at; i < a.rows; i += step) st_rows<1>(a, i, live, row_end, take_end, base, full);
  } else {
    for (int i = 4 * at; i < a.rows; i += 4 * step) st_rows<4>(a, i, live, row_end, take_end, base, full);
  }
}

}  // namespace bx
