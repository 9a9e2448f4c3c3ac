// Attention over the paged 8-bit cache: for each request, its new rows (one in decode, several when
// drafts are verified or a turn is appended) against all of its cached tokens,
//   out = sum_j softmax_j(scale * q . k_j) v_j over the positions j <= len - rows + i of row i.
//
// What bounds it: the cache is read once, 2 * hd bytes a token and kv head, for 4 * hd * rows * H/hkv
// operations; below about 60 rows of a group that is memory. The rows of one kv head (new rows x
// query heads of the group) form tiles of 8, the N of mma.sync.m16n8k16, with keys (then dims) as
// its M: scores^T = K q^T and out^T = V^T p^T, so that a decode step of 1 to 8 query heads a group
// fills its tile. A tcgen05 tile would have 128 rows, and takes no e4m3 operand against bf16 queries.
//
// Exactness: e4m3 codes convert to f16 without rounding. A query row is multiplied by a power of two
// that brings its largest value to 2^13, so its bf16 values are exact in f16 too (what is 2^-37 of
// the row's largest rounds). Scores and sums are fp32. The weights p = 2^(s - max + 15) round to f16,
// 2^-12 of a weight at most (below 2^-29 of the largest weight: absolutely). Output sums are held in
// units of the current page's scale; a page of another scale rescales them by a power of two.
//
// Conversion: cvt.f16x2.e4m3x2 runs on the XU pipe, 16 lanes a clock, which both products together
// would keep busy for 80 % of the time that memory takes. Values are converted in the ALU instead:
// the code's bits moved to f16's place are the value times 2^-8. That would turn a NaN code into a
// number, so append marks pages that hold a NaN value in the sign of v_scale, and for those the rows
// that see one are marked first. Keys keep the cvt, which keeps NaN.
//
// Split: all (request, row tile, kv head) segments are cut into steps of 128 keys, and the steps are
// shared evenly among the CTAs, whatever the lengths. A segment that one CTA has whole is written at
// once; else its CTAs write (max, sum, sum p v) and a second kernel, launched early so that its start
// overlaps, joins them in order: results do not depend on timing, and no counter outlives a call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kernels.h"

namespace mxk {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 32;           // keys a warp takes at once: always inside one page
constexpr int kStep = kChunk * kWarps;
constexpr int kMaxRequests = 4096;
constexpr int kStages = 2;
constexpr int kJoinWarps = 8;

// CTAs an SM: what its registers hold without spilling (255 at two, 168 at three, 128 at four), and
// at most what 228 KB of shared memory hold of rings (64 KB at hd 128, 32 KB at hd 64).
__host__ __device__ constexpr int ctas_per_sm(int hd, int tile) {
  return hd == 128 ? (tile == 8 ? 3 : 2) : (tile == 8 ? 4 : 3);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  const int n = in ? 16 : 0;  // 0: the 16 bytes become zeros, and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n));
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N)); }

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}

// Two e4m3 codes (the low or the high half of w) as f16x2.
__device__ __forceinline__ uint32_t f16_lo(uint32_t w) {
  uint32_t d;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(d) : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t f16_hi(uint32_t w) {
  uint32_t d;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, h;}" : "=r"(d) : "r"(w));
  return d;
}

// Bytes 0 and 2 (lo) or 1 and 3 (hi) of w, e4m3 codes that are not NaN, as f16x2 of the value * 2^-8:
// sign and eeeemmm go to f16's sign and the bits below its top exponent bit (bias 7 against 15).
__device__ __forceinline__ uint32_t alu_lo(uint32_t w) { return ((w << 8) & 0x80008000u) | ((w << 7) & 0x3f803f80u); }
__device__ __forceinline__ uint32_t alu_hi(uint32_t w) { return (w & 0x80008000u) | ((w >> 1) & 0x3f803f80u); }

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8x8 of 16-bit elements across the warp, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float quad_max(float v) {  // over the four lanes of a group
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float group_max(float v) {  // over the eight groups
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float group_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// The weight of a partial result with maximum m and sum l under the common maximum mx. A part that
// saw no key has m = -inf and l = 0; one that met a NaN score keeps it.
__device__ __forceinline__ float part_weight(float m, float l, float mx) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return exp2f(m - mx);
}

struct Work {
  float* acc;   // [2 * grid][tile][hd]
  float* ml;    // [2 * grid][tile][2]
  int* prefix;  // [R + 1] steps before each request
};
__host__ __device__ inline Work work_of(float* w, int grid, int tile, int hd) {
  Work k;
  k.acc = w;
  k.ml = w + 2L * grid * tile * hd;
  k.prefix = reinterpret_cast<int*>(k.ml + 2L * grid * tile * 2);
  return k;
}

__device__ __forceinline__ int new_rows(const Kv8Attention& a, int r, int& first) {
  if (a.starts == nullptr) {
    first = r;
    return r < a.rows ? 1 : 0;
  }
  first = a.starts[r];
  int n = a.starts[r + 1] - first;
  if (first < 0 || n < 0 || first > a.rows - n) n = 0;  // rows outside the tensors are not touched
  return n;
}

__device__ __forceinline__ int steps_of(const Kv8Attention& a, int page, int len) {
  const long most = (long)a.width * page;
  const long n = len < 0 ? 0 : (len > most ? most : len);
  return n <= kStep ? 1 : (int)((n + kStep - 1) / kStep);
}

__device__ __forceinline__ int owner(const int* v, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (v[mid + 1] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// First step of CTA i when `total` steps are shared among `grid` CTAs, and the CTA that has step x.
__device__ __forceinline__ int share(int i, int total, int grid) { return (int)((long)i * total / grid); }
__device__ __forceinline__ int cta_of(int x, int total, int grid) {
  return (int)((((long)x + 1) * grid - 1) / total);
}

// Before the values of a page that holds NaN are used: marks the (row, dim) pairs that see a NaN of
// this chunk, and zeroes the codes, which rows that do not see them would meet as 0 * NaN.
template <int HD>
__device__ __noinline__ void take_out_nan(uint8_t* values, uint8_t* marks, int lane, int key0, int rows, int rep,
                                          int row0, int pos0) {
  for (int i = lane; i < kChunk * HD; i += 32) {
    if ((values[i] & 0x7f) != 0x7f) continue;
    values[i] = 0;
    const int key = i / HD, at = i % HD;
    const int sw = HD == 128 ? ((key >> 1) & 3) << 1 : ((key >> 1) & 1) << 1;  // load's swizzle
    const int d = ((at / 16) ^ sw) * 16 + at % 16;
    for (int y = 0; y < rows; ++y)
      if (key0 + key <= pos0 + (row0 + y) / rep) marks[y * HD + d] = 1;
  }
}

// NQ: tiles of 8 rows that a segment's rows form.
template <int HD, int NQ>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(HD, 8 * NQ))
    attention_kernel(Kv8Cache c, Kv8Attention a) {
  constexpr int kRows = 8 * NQ;
  constexpr int KB = HD / 64;              // 16-byte pieces of a key a lane reads
  constexpr int MT = HD / 16;              // tiles of 16 dims of the output
  constexpr int kStageBytes = 2 * kChunk * HD;
  constexpr int kLoads = kChunk * HD / 16 / 32;  // 16-byte copies a lane, keys or values
  constexpr int VW = HD / 32;              // words a lane reads of a value row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int warp_sums[kWarps];
  __shared__ float sh_m[kWarps][kRows], sh_l[kWarps][kRows];
  __shared__ uint8_t sh_nan[kRows * HD];  // outputs that met a NaN value
  __shared__ int sh_any_nan;
  int* prefix = reinterpret_cast<int*>(smem + kWarps * kStages * kStageBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rep = a.H / c.hkv;
  const Work w = work_of(a.work, a.grid, kRows, HD);
  // the join's CTAs may take their places; they wait for this grid's end before they read
  asm volatile("griddepcontrol.launch_dependents;");

  // Steps before each request. Ascending starts keep the sum below the host's bound; with any other
  // nothing is computed.
  if (tid == 0) sh_any_nan = 0;
  for (int x = tid; x < kRows * HD; x += kThreads) sh_nan[x] = 0;
  int carry = 0, bad = 0;
  for (int base = 0; base < a.R; base += kThreads) {
    const int r = base + tid;
    int v = 0, first;
    if (r < a.R) {
      const int n = new_rows(a, r, first);
      if (a.starts != nullptr) bad |= a.starts[r + 1] < a.starts[r];
      v = (n * rep + kRows - 1) / kRows * c.hkv * steps_of(a, c.page, a.lens[r]);
    }
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int before = carry, all = carry;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) before += warp_sums[i];
      all += warp_sums[i];
    }
    if (r < a.R) prefix[r] = before + x - v;
    carry = all;
    __syncthreads();
  }
  if (tid == 0) prefix[a.R] = carry;
  bad = __syncthreads_or(bad);
  const int total = bad ? 0 : carry;
  if (blockIdx.x == 0)
    for (int r = tid; r <= a.R; r += kThreads) w.prefix[r] = r == a.R ? total : prefix[r];
  if (a.zero_tail) {  // rows behind the last request
    const int last = max(0, min(a.rows, a.starts[a.R]));
    uint4* o = reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + (long)last * a.H * HD);
    const long n = (long)(a.rows - last) * a.H * HD / 8;
    for (long i = blockIdx.x * (long)kThreads + tid; i < n; i += (long)gridDim.x * kThreads)
      o[i] = make_uint4(0, 0, 0, 0);
  }

  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(smem), ring = ring0 + warp * kStages * kStageBytes;
  const int used = min(a.grid, total);  // so that every CTA that shares has a step
  if ((int)blockIdx.x >= used) return;
  const int end = share(blockIdx.x + 1, total, used);
  int at = share(blockIdx.x, total, used);
  const int begin = at;
  while (at < end) {
    const int r = owner(prefix, a.R, at);
    const int len_in = a.lens[r];
    int row0;
    const int n_new = new_rows(a, r, row0);
    const int steps = steps_of(a, c.page, len_in);
    const int in_r = at - prefix[r], seg = in_r / steps;  // segments of a request: row tiles x kv heads
    const int s0 = in_r - seg * steps, seg_start = at - s0;
    const int kh = seg % c.hkv, tile = seg / c.hkv;
    const int s1 = min(steps, s0 + (end - at));
    const int cap = a.width * c.page;
    const bool too_long = len_in > cap;   // the table does not hold it: its rows become NaN
    const int len = max(0, min(len_in, cap));
    const int rows_here = min(kRows, n_new * rep - tile * kRows);
    const int pos0 = len_in - n_new;      // last position that new row 0 sees

    // this warp's chunks of the segment: first + kWarps * i, i < count
    const int tile_last = pos0 + (tile * kRows + rows_here - 1) / rep;  // last position any row sees
    const int tile_first = pos0 + tile * kRows / rep;                   // last position every row sees
    const int seen = max(0, min(len, tile_last + 1));
    const int chunks = min(s1 * kWarps, (seen + kChunk - 1) / kChunk);
    const int first = s0 * kWarps + warp;
    const int count = first < chunks ? (chunks - first + kWarps - 1) / kWarps : 0;
    const int* table = a.tables + (long)r * a.width;
    int page_id = 0;
    float ks_all = 0.f, vs_all = 0.f;
    auto fetch_pages = [&](int i0) {  // lane i: the page of this warp's chunk i0 + i, and its scales
      const int i = i0 + lane;
      page_id = -1;
      ks_all = NAN;  // a page that the pool does not have: the rows that see it become NaN
      vs_all = 0.f;
      if (i < count) {
        const int pg = table[(first + i * kWarps) * kChunk / c.page];
        if (pg >= 0 && pg < c.pages) {
          page_id = pg;
          ks_all = c.k_scale[(long)pg * c.hkv + kh];
          vs_all = c.v_scale[(long)pg * c.hkv + kh];
        }
      }
    };
    // Copies of chunk i (keys or values) into its stage; its block's page ids are in page_id. The
    // 16-byte columns of a row are swizzled so that the reads below meet no bank twice at hd 128.
    auto load = [&](int i, bool values) {
      const int key0 = (first + i * kWarps) * kChunk;
      const int pg = __shfl_sync(0xffffffffu, page_id, i & 31);
      const uint32_t dst = ring + (i % kStages) * kStageBytes + (values ? kChunk * HD : 0);
      const uint8_t* src = (const uint8_t*)(values ? c.v : c.k) +
                           (((long)max(pg, 0) * c.hkv + kh) * c.page + key0 % c.page) * HD;
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        const int byte = (x * 32 + lane) * 16, key = byte / HD, col = byte % HD / 16;
        const bool in = pg >= 0 && key0 + key < seen;  // what lies behind the last key is not read
        int sw;
        if (HD == 128) sw = values ? col ^ (((key >> 1) & 3) << 1) : col ^ ((key & 1) << 2);
        else sw = values ? col ^ (((key >> 1) & 1) << 1) : col;
        cp16(dst + key * HD + sw * 16, src + byte, in);
      }
      cp_commit();
    };
    float ks_use = 0.f, vs_use = 0.f;
    if (count > 0) {
      fetch_pages(0);
      ks_use = ks_all;
      vs_use = vs_all;
    }
#pragma unroll
    for (int i = 0; i < kStages; ++i) {  // one group for keys, one for values, empty past the end
      if (i < count) {
        load(i, false);
        load(i, true);
      } else {
        cp_commit();
        cp_commit();
      }
    }

    // Queries: lane (g, t) holds dims 64 b + 16 t .. + 15 of row g of each tile, four k steps of four
    // dims, the order in which the lanes read the keys' codes (16 bytes at a time).
    uint32_t qf[NQ][4 * KB][2];
    float qs[NQ][2];  // of rows 2 t and 2 t + 1
    int pos[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int y = 8 * n + g, x = tile * kRows + y;
      uint4 raw[2 * KB];
      float big = 0.f;
#pragma unroll
      for (int b = 0; b < 2 * KB; ++b) {
        raw[b] = make_uint4(0, 0, 0, 0);
        if (y < rows_here)
          raw[b] = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + (row0 + x / rep) * a.q_tok +
                                                   (long)(kh * rep + x % rep) * HD + 64 * (b / 2) + 16 * t + 8 * (b & 1));
        const uint32_t u[4] = {raw[b].x, raw[b].y, raw[b].z, raw[b].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          big = fmaxf(big, fmaxf(fabsf(__uint_as_float(u[j] << 16)), fabsf(__uint_as_float(u[j] & 0xffff0000u))));
      }
      big = quad_max(big);
      // 2^-e brings the largest to [2^13, 2^14); infinities and zeros stay
      int e = ((__float_as_int(big) >> 23) & 0xff) - 127 - 13;
      if (!(big > 0.f) || big == INFINITY) e = 0;
      e = max(-126, e);
      const float up = __int_as_float((127 - e) << 23);
      const float back = __int_as_float((127 + e) << 23) * (a.scale * 1.4426950408889634f);
#pragma unroll
      for (int b = 0; b < 2 * KB; ++b) {
        const uint32_t u[4] = {raw[b].x, raw[b].y, raw[b].z, raw[b].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          qf[n][2 * b + j / 2][j & 1] =
              pack_f16(__uint_as_float(u[j] << 16) * up, __uint_as_float(u[j] & 0xffff0000u) * up);
      }
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int yy = 8 * n + 2 * t + z;
        qs[n][z] = __shfl_sync(0xffffffffu, back, (2 * t + z) * 4);
        pos[n][z] = yy < rows_here ? pos0 + (tile * kRows + yy) / rep : -1;
      }
    }

    float o[MT][NQ][4], m[NQ][2], l[NQ][2], unit = 0.f;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[j][n][x] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }

    for (int i = 0; i < count; ++i) {
      const int key0 = (first + i * kWarps) * kChunk;
      const uint32_t kb = ring + (i % kStages) * kStageBytes, vb = kb + kChunk * HD;
      const int nx = i + kStages;
      float ks = __shfl_sync(0xffffffffu, ks_use, i & 31);
      const float vs = __shfl_sync(0xffffffffu, vs_use, i & 31);
      if (too_long || vs != vs) ks = NAN;
      cp_wait<2 * kStages - 1>();  // the keys of chunk i are there
      __syncwarp();

      // scores of 32 keys x rows: keys g and g + 8 of two tiles of 16, rows 2 t and 2 t + 1
      float s[2][NQ][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[h][n][x] = 0.f;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const int key = 16 * h + g, col = 4 * b + t;
          const uint32_t at0 = kb + key * HD + (HD == 128 ? col ^ ((key & 1) << 2) : col) * 16;
          const uint4 u = lds128(at0), v = lds128(at0 + 8 * HD);
          const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a0 = f16_lo(uw[j]), a1 = f16_lo(vw[j]), a2 = f16_hi(uw[j]), a3 = f16_hi(vw[j]);
#pragma unroll
            for (int n = 0; n < NQ; ++n) mma(s[h][n], a0, a1, a2, a3, qf[n][4 * b + j][0], qf[n][4 * b + j][1]);
          }
        }
      }
      __syncwarp();  // all lanes have read the keys: their place takes those of the chunk after next
      if (nx < count) {
        if ((nx & 31) == 0) fetch_pages(nx);
        load(nx, false);
      } else {
        cp_commit();
      }

      const bool diag = key0 + kChunk > min(len, tile_first + 1);  // some row does not see some key
      float pscale = 1.f, ratio = 1.f;
      if (fabsf(vs) > 0.f) {  // sums in units of this page's scale (2^-60 of the last at least)
        const float now = fmaxf(fabsf(vs), unit * 0x1p-60f);
        ratio = unit / now;
        pscale = fabsf(vs) / now;
        unit = now;
      }
      uint32_t pf[NQ][2][2];
      bool moved = false;
      float factor[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float v = s[h][n][x] * (qs[n][x & 1] * ks);
            if (diag && key0 + 16 * h + g + 8 * (x >> 1) > pos[n][x & 1]) v = -INFINITY;
            s[h][n][x] = v;
            top[x & 1] = fmaxf(top[x & 1], v);
          }
        float sub[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const float mn = fmaxf(m[n][z], group_max(top[z]));
          const float ref = mn == -INFINITY ? 0.f : mn;
          const float alpha = exp2f(m[n][z] - ref);
          sub[z] = ref - 15.f;
          m[n][z] = mn;
          l[n][z] *= alpha;
          factor[n][z] = alpha * ratio;
          moved |= factor[n][z] != 1.f;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            p[x] = exp2f(s[h][n][x] - sub[x & 1]);
            l[n][x & 1] += p[x];
          }
          if (pscale != 1.f) {
#pragma unroll
            for (int x = 0; x < 4; ++x) p[x] *= pscale;
          }
          pf[n][h][0] = transpose8(pack_f16(p[0], p[1]));
          pf[n][h][1] = transpose8(pack_f16(p[2], p[3]));
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[j][n][x] *= factor[n][x & 1];
      }

      // out^T += V^T p^T: lane g has the dims g * HD / 8 .. of the values
      cp_wait<2 * kStages - 1>();  // the values of chunk i are there
      __syncwarp();
      if (vs < 0.f) {
        take_out_nan<HD>(smem + (vb - ring0), sh_nan, lane, key0, rows_here, rep, tile * kRows, pos0);
        if (lane == 0) sh_any_nan = 1;
        __syncwarp();
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t vw[4][VW];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the 16
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int key = 16 * h + 2 * t + (q & 1) + 8 * (q >> 1);
          if constexpr (HD == 128) {
            const uint4 u = lds128(vb + key * HD + ((g ^ (((key >> 1) & 3) << 1)) * 16));
            vw[q][0] = u.x; vw[q][1] = u.y; vw[q][2] = u.z; vw[q][3] = u.w;
          } else {
            const uint2 u = lds64(vb + key * HD + (((g >> 1) ^ (((key >> 1) & 1) << 1)) * 16) + (g & 1) * 8);
            vw[q][0] = u.x; vw[q][1] = u.y;
          }
        }
#pragma unroll
        for (int x = 0; x < VW; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {  // two dims at a time: (key, dim), (key, dim + 1), (key + 1, dim), ..
            const uint32_t p = __byte_perm(vw[0][x], vw[1][x], y ? 0x7632 : 0x5410);
            const uint32_t q = __byte_perm(vw[2][x], vw[3][x], y ? 0x7632 : 0x5410);
            const uint32_t a0 = alu_lo(p), a1 = alu_hi(p), a2 = alu_lo(q), a3 = alu_hi(q);
#pragma unroll
            for (int n = 0; n < NQ; ++n) mma(o[2 * x + y][n], a0, a1, a2, a3, pf[n][h][0], pf[n][h][1]);
          }
      }
      __syncwarp();
      if (nx < count) load(nx, true);
      else cp_commit();
      // A block of page ids serves 32 chunks. The scales in use change to the next block's, fetched
      // when its first chunk was loaded, once the last chunk of this block is done.
      if (((i + 1) & 31) == 0) {
        ks_use = ks_all;
        vs_use = vs_all;
      }
    }
    cp_wait<0>();

    // join the warps: through shared memory, which the ring no longer needs
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem) + warp * kRows * HD;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float sum = group_sum(l[n][z]);
        const int y = 8 * n + 2 * t + z;
        if (g == 0) {
          sh_m[warp][y] = m[n][z];
          sh_l[warp][y] = sum;
        }
        if (y < rows_here) {
#pragma unroll
          for (int j = 0; j < MT; ++j)
            *reinterpret_cast<float2*>(so + y * HD + g * (HD / 8) + 2 * j) =
                make_float2(o[j][n][z] * unit * 256.f, o[j][n][z + 2] * unit * 256.f);
        }
      }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const int slot = 2 * blockIdx.x + (seg_start >= begin ? 1 : 0);
    for (int x = tid; x < rows_here * HD; x += kThreads) {
      const int y = x / HD, d = x % HD;
      float mx = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) mx = fmaxf(mx, sh_m[i][y]);
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float f = part_weight(sh_m[i][y], sh_l[i][y], mx);
        sum += sh_l[i][y] * f;
        acc += reinterpret_cast<float*>(smem)[(i * kRows + y) * HD + d] * f;
      }
      if (sh_any_nan && sh_nan[x]) {
        acc = NAN;
        sh_nan[x] = 0;
      }
      if (whole) {
        const int xr = tile * kRows + y;
        ((__nv_bfloat16*)a.out)[((long)(row0 + xr / rep) * a.H + kh * rep + xr % rep) * HD + d] =
            __float2bfloat16(sum == 0.f ? 0.f : acc / sum);
      } else {
        w.acc[((long)slot * kRows + y) * HD + d] = acc;
        if (d == 0) {
          w.ml[(slot * kRows + y) * 2] = mx;
          w.ml[(slot * kRows + y) * 2 + 1] = sum;
        }
      }
    }
    __syncthreads();
    at += s1 - s0;
  }
}

// Joins the segments that several CTAs shared: one CTA for each output row and head, whose warps
// share the parts.
template <int HD>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(Kv8Cache c, Kv8Attention a) {
  constexpr int E = HD / 32;
  __shared__ float sh[kJoinWarps][HD], sh_m[kJoinWarps], sh_l[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const Work w = work_of(a.work, a.grid, a.tile, HD);
  const int rep = a.H / c.hkv;
  // the caller's own inputs, complete before the attention kernel began
  int r = row;
  if (a.starts != nullptr) {
    if (row >= a.starts[a.R]) return;
    r = owner(a.starts, a.R, row);
  }
  int row0;
  if (row - (a.starts ? a.starts[r] : r) >= new_rows(a, r, row0)) return;
  const int steps = steps_of(a, c.page, a.lens[r]);
  if (steps == 1) return;  // one step has one CTA
  const int x = (row - row0) * rep + h % rep, tile = x / a.tile, y = x % a.tile;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int total = w.prefix[a.R];
  if (total == 0) return;
  const int used = min(a.grid, total);
  const int s0 = w.prefix[r] + (tile * c.hkv + h / rep) * steps;
  const int c0 = cta_of(s0, total, used), c1 = cta_of(s0 + steps - 1, total, used);
  if (c0 == c1) return;  // written by its CTA
  float mx = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 2
  for (int b = c0 + warp; b <= c1; b += kJoinWarps) {
    const int slot = (2 * b + (b == c0)) * a.tile + y;
    const float m = w.ml[slot * 2], l = w.ml[slot * 2 + 1];
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = w.acc[(long)slot * HD + e * 32 + lane];
    const float mn = fmaxf(mx, m);
    const float f0 = part_weight(mx, sum, mn), f1 = part_weight(m, l, mn);
    sum = sum * f0 + l * f1;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f0 + v[e] * f1;
    mx = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sh[warp][e * 32 + lane] = acc[e];
  if (lane == 0) {
    sh_m[warp] = mx;
    sh_l[warp] = sum;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= HD) return;
  float top = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll
  for (int i = 0; i < kJoinWarps; ++i) top = fmaxf(top, sh_m[i]);
#pragma unroll
  for (int i = 0; i < kJoinWarps; ++i) {
    const float f = part_weight(sh_m[i], sh_l[i], top);
    den += sh_l[i] * f;
    num += sh[i][d] * f;
  }
  ((__nv_bfloat16*)a.out)[((long)row * a.H + h) * HD + d] = __float2bfloat16(den == 0.f ? 0.f : num / den);
}

template <int HD, int NQ>
int launch(const Kv8Cache& c, const Kv8Attention& a, cudaStream_t st) {
  constexpr int kRing = kWarps * kStages * 2 * kChunk * HD;
  static_assert(kWarps * 8 * NQ * HD * 4 <= kRing, "the join fits the ring");
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<bool> raised[64];
  if (dev < 0 || dev >= 64) return kErrBadArgsHost;
  if (!raised[dev].load()) {
    if (cudaFuncSetAttribute(attention_kernel<HD, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kRing + (kMaxRequests + 1) * 4) != cudaSuccess)
      return kErrBadArgsHost;
    raised[dev].store(true);
  }
  count_launch();
  attention_kernel<HD, NQ><<<a.grid, kThreads, kRing + (a.R + 1) * 4, st>>>(c, a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * a.H));
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  if (cudaLaunchKernelEx(&cfg, join_kernel<HD>, c, a) != cudaSuccess) return kErrBadArgsHost;
  return cudaGetLastError() == cudaSuccess ? 0 : kErrBadArgsHost;
}

}  // namespace

// Rows of a tile: what a request's rows of one kv head need on average (8 in decode up to 8 query
// heads a group), 16 at most at hd 128 and 32 at hd 64, where the registers end.
int kv8_attention_tile(int rows, int H, int hkv, int R, int hd) {
  const long n = R < 1 || hkv < 1 ? 1 : ((long)rows + R - 1) / R * (H / hkv);
  return n <= 8 ? 8 : (n <= 16 || hd == 128 ? 16 : 32);
}

int kv8_attention_grid(int rows, int H, int hkv, int R, int width, int page, int hd, int sms) {
  if (R < 1 || R > kMaxRequests || rows < 0 || hkv < 1 || H % hkv || (long)width * page > 0x7fffffffL) return -1;
  if ((long)rows * H > 0x7fffffffL) return -1;
  const int tile = kv8_attention_tile(rows, H, hkv, R, hd);
  const long tiles = ((long)rows * (H / hkv) + tile - 1) / tile + R;  // each request rounds up at most once
  const long steps = ((long)width * page + kStep - 1) / kStep;
  if ((double)tiles * hkv * (steps < 1 ? 1 : steps) > 2.0e9) return -1;
  const long most = tiles * hkv * (steps < 1 ? 1 : steps);
  const long ctas = (long)sms * ctas_per_sm(hd, tile);
  return (int)(most < ctas ? (most < 1 ? 1 : most) : ctas);
}

long kv8_attention_work(int grid, int tile, int R, int hd) { return 2L * grid * tile * (hd + 2) + R + 1; }

int launch_kv8_attention(const Kv8Cache& c, const Kv8Attention& a, cudaStream_t st) {
  if (a.rows < 1) return 0;
  if (c.page % kChunk || a.grid < 1) return kErrBadArgsHost;
  if (c.hd == 64 && a.tile == 8) return launch<64, 1>(c, a, st);
  if (c.hd == 64 && a.tile == 16) return launch<64, 2>(c, a, st);
  if (c.hd == 64 && a.tile == 32) return launch<64, 4>(c, a, st);
  if (c.hd == 128 && a.tile == 8) return launch<128, 1>(c, a, st);
  if (c.hd == 128 && a.tile == 16) return launch<128, 2>(c, a, st);
  return kErrBadArgsHost;
}

}  // namespace mxk
