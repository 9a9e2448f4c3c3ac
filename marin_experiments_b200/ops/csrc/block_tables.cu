// Block tables and slot maps of a paged KV cache, built on the GPU from the requests' lengths, so a
// decode step needs no host round trip to place its tokens.
//
// extend: request r holds len[r] tokens on ceil(len / page) pages and grows by new[r]. Its further
// pages come off the top of the free stack, in the order of the requests:
//   have = ceil(len / page), want = ceil((len + new) / page), off = exclusive sum of (want - have),
//   table[r, have + i] = free[count - 1 - off - i],
// and the tokens' rows are packed by request: starts = exclusive sum of new; row i of request r is
// its position p = len + i - starts[r] and its slot table[r, p / page] * page + p % page.
//
// Latency bounds this: two dependent loads, two scans over at most kMaxRequests values and a binary
// search a row. Every CTA repeats the scan (the lengths are a few KB that L2 holds), so no CTA waits
// for another and one launch does all; pages off the stack are computed, not read back from the
// table, for the same reason.
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "pdl.cuh"

namespace mxk {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Exclusive block-wide sums of (a, b); totals in ta, tb. All threads call it.
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long& ta, long long& tb,
                                            long long (*sh)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long ia = warp_scan(a, lane), ib = warp_scan(b, lane);
  if (lane == 31) {
    sh[warp][0] = ia;
    sh[warp][1] = ib;
  }
  __syncthreads();
  long long pa = 0, pb = 0;
  ta = tb = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const long long xa = sh[w][0], xb = sh[w][1];
    if (w < warp) {
      pa += xa;
      pb += xb;
    }
    ta += xa;
    tb += xb;
  }
  a = pa + ia - a;
  b = pb + ib - b;
  __syncthreads();
}

// First r with v[r + 1] > x, for ascending v[0 .. n].
__device__ __forceinline__ int owner(const int* v, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (v[mid + 1] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads)
    extend_kernel(int* __restrict__ tables, int width, const int* __restrict__ lens, const int* __restrict__ grow,
                  int R, const int* __restrict__ free_pages, int capacity, const int* __restrict__ free_count,
                  int page, int rows, int* __restrict__ lens_out, int* __restrict__ count_out,
                  int* __restrict__ starts_out, int* __restrict__ slots, int* __restrict__ requests,
                  int* __restrict__ positions, int* __restrict__ status) {
  extern __shared__ int smem[];
  int* starts = smem;              // [R + 1]
  int* offs = smem + R + 1;        // [R + 1]
  __shared__ long long sh[kWarps][2];
  __shared__ int bad_any;
  const int tid = threadIdx.x;
  if (tid == 0) bad_any = 0;
  wait_for_previous();
  const int count = *free_count;
  int bad = count < 0 || count > capacity ? kTablesBadInput : 0;
  long long sum_new = 0, sum_more = 0;
  __syncthreads();
  for (int base = 0; base < R; base += kThreads) {  // R is the same for all threads
    const int r = base + tid;
    long long a = 0, b = 0;
    if (r < R) {
      const int len = lens[r], nw = grow[r];
      if (len < 0 || nw < 0) bad |= kTablesBadInput;
      else {
        const long long want = ((long long)len + nw + page - 1) / page;
        if (want > width || (long long)len + nw > 0x7fffffffLL) bad |= kTablesTooLong;
        a = nw;
        b = want - ((long long)len + page - 1) / page;
      }
    }
    long long ta, tb;
    block_scan2(a, b, ta, tb, sh);
    if (r < R) {  // garbage past 2^31 only where the status refuses the step
      starts[r] = (int)(sum_new + a);
      offs[r] = (int)(sum_more + b);
    }
    sum_new += ta;
    sum_more += tb;
  }
  if (sum_new > rows) bad |= kTablesTooManyRows;
  if (sum_more > count) bad |= kTablesNoPages;
  if (bad) atomicOr(&bad_any, bad);
  if (tid == 0) {
    starts[R] = (int)sum_new;
    offs[R] = (int)sum_more;
  }
  __syncthreads();
  bad = bad_any;
  const int gid = blockIdx.x * kThreads + tid, gsize = gridDim.x * kThreads;
  if (gid == 0) {
    *status = bad;
    *count_out = bad ? count : count - (int)sum_more;
  }
  for (int r = gid; r <= R; r += gsize) {
    starts_out[r] = bad ? 0 : starts[r];
    if (r < R) lens_out[r] = bad ? lens[r] : lens[r] + grow[r];
  }
  if (bad) {  // nothing is placed
    for (int i = gid; i < rows; i += gsize) {
      slots[i] = -1;
      requests[i] = -1;
      positions[i] = 0;
    }
    return;
  }
  const int total_new = (int)sum_new, total_more = (int)sum_more;
  for (int p = gid; p < total_more; p += gsize) {
    const int r = owner(offs, R, p);
    const int have = (lens[r] + page - 1) / page;
    tables[(long)r * width + have + (p - offs[r])] = free_pages[count - 1 - p];
  }
  for (int i = gid; i < rows; i += gsize) {
    int slot = -1, r = -1, pos = 0;
    if (i < total_new) {
      r = owner(starts, R, i);
      const int len = lens[r];
      pos = len + (i - starts[r]);
      const int c = pos / page, have = (len + page - 1) / page;
      // a column below `have` is never written above, so the read does not race
      const int pg = c < have ? tables[(long)r * width + c] : free_pages[count - 1 - (offs[r] + c - have)];
      const long long at = (long long)pg * page + pos % page;
      slot = pg < 0 || at > 0x7fffffffLL ? -1 : (int)at;
    }
    slots[i] = slot;
    requests[i] = r;
    positions[i] = pos;
  }
}

// One CTA: the freed pages go onto the stack in the order of the requests.
__global__ void __launch_bounds__(kThreads)
    release_kernel(int* __restrict__ tables, int width, int* __restrict__ lens, const uint8_t* __restrict__ done, int R,
                   int* __restrict__ free_pages, int capacity, int* __restrict__ free_count, int page,
                   int* __restrict__ status) {
  extern __shared__ int offs[];  // [R + 1]
  __shared__ long long sh[kWarps][2];
  __shared__ int bad_any;
  const int tid = threadIdx.x;
  if (tid == 0) bad_any = 0;
  wait_for_previous();
  const int count = *free_count;
  int bad = count < 0 || count > capacity ? kTablesBadInput : 0;
  long long total = 0;
  __syncthreads();
  for (int base = 0; base < R; base += kThreads) {
    const int r = base + tid;
    long long n = 0, unused = 0, tn, tu;
    if (r < R && done[r]) {
      const int len = lens[r];
      if (len < 0) bad |= kTablesBadInput;
      else n = ((long long)len + page - 1) / page;
      if (n > width) bad |= kTablesTooLong;
    }
    block_scan2(n, unused, tn, tu, sh);
    if (r < R) offs[r] = (int)(total + n);
    total += tn;
  }
  if (total > capacity - count) bad |= kTablesBadInput;
  if (bad) atomicOr(&bad_any, bad);
  if (tid == 0) offs[R] = (int)total;
  __syncthreads();
  bad = bad_any;
  if (tid == 0) *status = bad;
  if (bad) return;
  for (int p = tid; p < (int)total; p += kThreads) {
    const int r = owner(offs, R, p);
    int* cell = tables + (long)r * width + (p - offs[r]);
    free_pages[count + p] = *cell;
    *cell = -1;
  }
  for (int r = tid; r < R; r += kThreads)
    if (done[r]) lens[r] = 0;
  if (tid == 0) *free_count = count + (int)total;
}

}  // namespace

int launch_block_tables_extend(int* tables, int width, const int* lens, const int* grow, int R, const int* free_pages,
                               int capacity, const int* free_count, int page, int rows, int* lens_out, int* count_out,
                               int* starts, int* slots, int* requests, int* positions, int* status, cudaStream_t st) {
  if (R < 1 || R > kTablesMaxRequests || page < 1 || rows < 0 || width < 0) return kErrBadArgsHost;
  // one CTA up to 2048 rows (4 a thread); each further one repeats the scan
  int grid = (rows + 4 * kThreads - 1) / (4 * kThreads);
  if (grid < 1) grid = 1;
  if (grid > 148) grid = 148;
  count_launch();
  return launch_early(extend_kernel, dim3(grid), kThreads, 2 * (R + 1) * sizeof(int), st, 1, tables, width, lens, grow, R,
                      free_pages, capacity, free_count, page, rows, lens_out, count_out, starts, slots, requests,
                      positions, status) == cudaSuccess
             ? 0
             : kErrBadArgsHost;
}

int launch_block_tables_release(int* tables, int width, int* lens, const uint8_t* done, int R, int* free_pages,
                                int capacity, int* free_count, int page, int* status, cudaStream_t st) {
  if (R < 1 || R > kTablesMaxRequests || page < 1 || width < 0) return kErrBadArgsHost;
  count_launch();
  return launch_early(release_kernel, dim3(1), kThreads, (R + 1) * sizeof(int), st, 1, tables, width, lens, done, R,
                      free_pages, capacity, free_count, page, status) == cudaSuccess
             ? 0
             : kErrBadArgsHost;
}

}  // namespace mxk
