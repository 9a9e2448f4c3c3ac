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
// the row's largest rounds). Scores and sums are fp32. The weights 2^15 p, p = 2^(s - max), round to f16,
// 2^-12 of a weight at most (below 2^-29 of the largest weight: absolutely). Output sums are held in
// units of the current page's scale; a page of another scale rescales them by a power of two. The unit stays
// above 2^-60 of the largest that a warp has met in the segment, so the weights of pages below 2^-89 of that lose
// bits (2^15 * 2^-29 is f16's least normal number).
//
// A NaN value must reach the rows that see it and no other, but 0 * NaN would reach all rows of a
// tile. append marks pages that hold a NaN value in the sign of v_scale; before such a page's values
// are used, the outputs that see a NaN are marked and its codes are taken out.
//
// Split, many segments (a segment: one request, row tile and kv head): segments are cut into steps of
// 128 keys, and the steps are shared evenly among as many CTAs as the GPU holds, whatever the
// lengths. A segment that one CTA has whole is written at once; else its CTAs write (max, sum,
// sum p v) and a second kernel, launched early so that its start overlaps, joins them in order.
// Few segments: a cluster of up to 8 CTAs takes one segment and joins through distributed shared
// memory, one launch. Either way results do not depend on timing, and no counter outlives a call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "kernels.h"
#include "pdl.cuh"

namespace mxk {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 32;           // keys a warp takes at once: always inside one page
constexpr int kStep = kChunk * kWarps;
constexpr int kMaxRequests = 4096;
constexpr int kJoinWarps = 8;
// Long calls make up to kRounds CTAs for each that runs at once, of kManySteps steps or more: SMs are
// not equally fast, and the hardware gives the next CTA to the one that is free (48 requests of up to
// 32768 tokens: 254 us at 1 round, 249 at 2, 242 at 4, 237 at 8; 259 with 8 steps a CTA).
constexpr long kRounds = 8;
constexpr int kManySteps = 16;
// Most steps that a CTA of a cluster takes. Where clusters leave more than half of the GPU's places free,
// sharing the steps among all places is worth the join's launch from three steps on (us, in clusters and
// shared; one request of 2000 tokens, 8 kv heads: 8.35, 7.7; of 4000: 9.5, 8.3; two of 4000: 11.7, 9.7;
// 1000 tokens, two steps: 6.5, 8.1; the rule sees the table's width and not the lengths, so a table wide enough
// for 4096 tokens costs one of 1000 this). Where they fill it, not (16 requests of 500 to 2000 tokens: 15.5,
// 17.5; 24 of 7 to 6001, 2 kv heads: 11.1, 12.3).
constexpr int kClusterSteps = 16, kFewClusterSteps = 2;

// Chunks of a warp on their way, and CTAs an SM: what its registers hold without spilling (255 at
// two, 168 at three, 128 at four), and 228 KB of shared memory hold of rings (a stage is 32 KB of a
// CTA at hd 128). A cluster's CTAs have few chunks each, whose latency counts: a stage more for a CTA
// less.
__host__ __device__ constexpr int stages_of(int hd, bool cluster) { return hd == 128 ? (cluster ? 3 : 2) : (cluster ? 4 : 3); }
__host__ __device__ constexpr int ctas_per_sm(int hd, int tile, bool cluster) {
  return hd == 128 ? (tile == 8 && !cluster ? 3 : 2) : (tile == 8 && !cluster ? 4 : 3);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src));
}
__device__ __forceinline__ void cp16_if(uint32_t dst, const void* src, bool in) {
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

// 2^x, 0 below 2^-126
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

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
  return ex2(m - mx);
}

// The least power of two >= x, and the inverse of one (2^-126 to 2^126): divisions take longer.
__device__ __forceinline__ float power_of_two(float x) {
  return __int_as_float((__float_as_int(x) + 0x7fffff) & 0x7f800000);
}
__device__ __forceinline__ float inverse_power(float x) { return __int_as_float(0x7f000000 - __float_as_int(x)); }

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

// n / d for 0 <= n < 2^31, with mul = ceil(2^(31 + l) / d), l = ceil(log2 d): the product is off by
// less than n * 2^l <= 2^(31 + l), one part in mul's scale.
struct Div {
  uint32_t mul;
  int d, shift;
  __device__ __forceinline__ int by(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
};
Div make_div(int d) {
  int l = 0;
  while ((1LL << l) < d) ++l;
  Div v;
  v.d = d;
  v.mul = d == 1 ? 0 : (uint32_t)(((1ULL << (31 + l)) + d - 1) / d);
  v.shift = l - 1;
  return v;
}

struct Args {
  Kv8Cache c;
  Kv8Attention a;
  Div rep, hkv;    // query heads of a kv head; kv heads
  int page_shift;
  float down;      // 1 / (tokens of a table's row, rounded up to a power of two)
};

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

__device__ __forceinline__ int steps_of(int cap, int len) {
  return max(1, (int)(((unsigned)max(0, min(len, cap)) + kStep - 1) / kStep));
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

// CTAs that share the steps: all that the GPU holds at once, each with one step at least, and up to
// the grid's multiple of that where each still has kManySteps.
__device__ __forceinline__ int used_ctas(const Kv8Attention& a, int total) {
  return min(total, max(a.resident, min(a.grid, total / kManySteps)));
}

// `total` steps among `used` <= total CTAs: the first total % used have one more.
struct Share {
  int per, more;
  __device__ __forceinline__ Share(int total, int used) : per(total / used), more(total - per * used) {}
  __device__ __forceinline__ int first(int cta) const { return cta * per + min(cta, more); }
  __device__ __forceinline__ int cta(int step) const {
    const int big = more * (per + 1);
    return step < big ? step / (per + 1) : more + (step - big) / per;
  }
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_rank(const void* p, int rank) {  // the same place in another CTA
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return d;
}
__device__ __forceinline__ float ld_rank(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
template <int E>
__device__ __forceinline__ void store_bf16(__nv_bfloat16* p, const float (&v)[E]) {
  uint32_t u[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[e], v[e + 1]);
    u[e / 2] = *reinterpret_cast<const uint32_t*>(&h);
  }
  if constexpr (E == 4) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
  else *reinterpret_cast<uint32_t*>(p) = u[0];
}
template <int E>
__device__ __forceinline__ void load_f32(const float* p, float (&v)[E]) {
  if constexpr (E == 4) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  } else {
    const float2 u = *reinterpret_cast<const float2*>(p);
    v[0] = u.x; v[1] = u.y;
  }
}
template <int E>
__device__ __forceinline__ void store_f32(float* p, const float (&v)[E]) {
  if constexpr (E == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
}

// Before the values of a page that holds NaN are used: marks the (row, dim) pairs that see a NaN of
// this chunk, and zeroes the codes, which rows that do not see them would meet as 0 * NaN.
template <int HD>
__device__ __noinline__ void take_out_nan(uint8_t* values, uint8_t* marks, int lane, int key0, int rows, Div rep,
                                          int row0, int pos0) {
  for (int i = lane; i < kChunk * HD; i += 32) {
    if ((values[i] & 0x7f) != 0x7f) continue;
    values[i] = 0;
    const int key = i / HD, at = i % HD;
    const int sw = HD == 128 ? ((key >> 1) & 3) << 1 : ((key >> 1) & 1) << 1;  // load's swizzle
    const int d = ((at / 16) ^ sw) * 16 + at % 16;
    for (int y = 0; y < rows; ++y)
      if (key0 + key <= pos0 + rep.by(row0 + y)) marks[y * HD + d] = 1;
  }
}

// NQ: tiles of 8 rows that a segment's rows form. CLUSTER: one segment for each cluster.
template <int HD, int NQ, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(HD, 8 * NQ, CLUSTER)) attention_kernel(const __grid_constant__ Args args) {
  constexpr int kRows = 8 * NQ, kStages = stages_of(HD, CLUSTER);
  constexpr int KB = HD / 64;              // 16-byte pieces of a key a lane reads
  constexpr int MT = HD / 16;              // tiles of 16 dims of the output
  constexpr int E = HD / 32;               // dims of an output row a lane joins
  constexpr int kStageBytes = 2 * kChunk * HD;
  constexpr int kLoads = kChunk * HD / 16 / 32;  // 16-byte copies a lane, keys or values
  constexpr int VW = HD / 32;              // words a lane reads of a value row
  const Kv8Cache& c = args.c;
  const Kv8Attention& a = args.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int warp_sums[kWarps];
  __shared__ float sh_m[kWarps][kRows], sh_l[kWarps][kRows];
  __shared__ uint8_t sh_nan[kRows * HD];  // outputs that met a NaN value
  __shared__ int sh_any_nan;
  int* prefix = reinterpret_cast<int*>(smem + kWarps * kStages * kStageBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rep = args.rep.d, cap = a.width << args.page_shift;
  const Work w = work_of(a.work, a.grid, kRows, HD);

  if (tid == 0) sh_any_nan = 0;
  for (int x = tid; x < kRows * HD / 4; x += kThreads) reinterpret_cast<int*>(sh_nan)[x] = 0;
  wait_for_previous();
  if (!CLUSTER) let_next_start();

  int total = 0, bad = 0;
  // Segments of a request where all have one row: a cluster then knows its request without a sum over the
  // others' (one request of 1000 tokens: 6.8 -> 6.6 us; 24 of 7 to 6001, 2 kv heads: 11.2 -> 10.4).
  const int same = CLUSTER && a.starts == nullptr ? (rep + kRows - 1) / kRows * c.hkv : 0;
  if (same) {
    total = a.R * same;
    __syncthreads();
  } else {
    // Steps (with CLUSTER segments) before each request, each thread's requests in a row. Starts that
    // ascend within the rows keep the sum below the host's bound; with any other nothing is computed.
    const int per = (a.R + kThreads - 1) / kThreads;
    auto weight = [&](int r, int& bad) {
      int first;
      const int n = new_rows(a, r, first);
      if (a.starts != nullptr) bad |= first < 0 || a.starts[r + 1] < first || a.starts[r + 1] > a.rows;
      return (n * rep + kRows - 1) / kRows * c.hkv * (CLUSTER ? 1 : steps_of(cap, a.lens[r]));
    };
    int mine = 0;
    for (int i = 0; i < per; ++i)
      if (tid * per + i < a.R) mine += weight(tid * per + i, bad);
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    if (lane == 31) warp_sums[warp] = x;
    bad = __syncthreads_or(bad);
    int before = x - mine;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) before += warp_sums[i];
      total += warp_sums[i];
    }
    for (int i = 0; i < per; ++i) {
      const int r = tid * per + i;
      if (r < a.R) {
        prefix[r] = before;
        if (i + 1 < per) before += weight(r, bad);
      }
    }
    if (bad) total = 0;
    if (tid == 0) prefix[a.R] = total;
    __syncthreads();
  }
  if (!CLUSTER && blockIdx.x == 0)
    for (int r = tid; r <= a.R; r += kThreads) w.prefix[r] = prefix[r];
  if (a.zero_tail) {  // rows of no request: before the first, behind the last, all if starts are refused
    const int last = bad ? 0 : a.starts[a.R];
    const int lead = bad ? 0 : a.starts[0];
    constexpr int kPieces = HD / 8;
    const long per = (long)a.H * kPieces, n = (a.rows - last + lead) * per;
    uint4* o = reinterpret_cast<uint4*>(a.out);
    for (long i = blockIdx.x * (long)kThreads + tid; i < n; i += (long)gridDim.x * kThreads)
      o[i < lead * per ? i : i - lead * per + last * per] = make_uint4(0, 0, 0, 0);
  }

  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(smem), ring = ring0 + warp * kStages * kStageBytes;
  // the lane's place in a stage, of the first of its copies: 4 keys a copy at hd 128, 8 at 64
  const int col = lane % (HD / 16), row_of = lane / (HD / 16);
  const int k_place = row_of * HD + (HD == 128 ? col ^ ((row_of & 1) << 2) : col) * 16;
  const int v_place = row_of * HD + (col ^ (((row_of >> 1) & (HD == 128 ? 3 : 1)) << 1)) * 16;
  int at, end;
  const int parts = CLUSTER ? a.cluster : 1, rank = CLUSTER ? blockIdx.x % parts : 0;
  if (CLUSTER) {
    at = blockIdx.x / parts;
    end = at < total ? at + 1 : at;  // the same for the whole cluster
  } else {
    const int used = used_ctas(a, total);
    if ((int)blockIdx.x >= used) return;
    const Share sh(total, used);
    at = sh.first(blockIdx.x);
    end = sh.first(blockIdx.x + 1);
  }
  const int begin = at;
  while (at < end) {
    const int r = same ? at / same : owner(prefix, a.R, at);
    const int len_in = a.lens[r];
    int row0;
    const int n_new = new_rows(a, r, row0);
    const int steps = steps_of(cap, len_in);
    const int in_r = at - (same ? r * same : prefix[r]), seg = CLUSTER ? in_r : in_r / steps;  // segments of a request: row tiles x kv heads
    const int tile = args.hkv.by(seg), kh = seg - tile * c.hkv;
    const int s0 = CLUSTER ? steps * rank / parts : in_r - seg * steps, seg_start = at - s0;
    const int s1 = CLUSTER ? steps * (rank + 1) / parts : min(steps, s0 + (end - at));
    const bool too_long = len_in > cap;   // the table does not hold it: its rows become NaN
    const int len = max(0, min(len_in, cap));
    const int rows_here = min(kRows, n_new * rep - tile * kRows);
    const int pos0 = len_in - n_new;      // last position that new row 0 sees

    // this warp's chunks of the segment: first + kWarps * i, i < count
    const int tile_last = pos0 + args.rep.by(tile * kRows + rows_here - 1);  // last position any row sees
    const int tile_first = pos0 + args.rep.by(tile * kRows);                   // last position every row sees
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
        const int pg = table[(first + i * kWarps) * kChunk >> args.page_shift];
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
      const uint32_t stage = ring + (i % kStages) * kStageBytes;
      const uint32_t dst = values ? stage + kChunk * HD + v_place : stage + k_place;
      const uint8_t* src = (const uint8_t*)(values ? c.v : c.k) + lane * 16 +
                           (((long)max(pg, 0) * c.hkv + kh) * c.page + (key0 & (c.page - 1))) * HD;
      if (key0 + kChunk <= seen && pg >= 0) {
#pragma unroll
        for (int x = 0; x < kLoads; ++x) cp16((dst + x * 512) ^ (HD == 128 && values && x % 2 ? 64 : 0), src + x * 512);
      } else {  // what lies behind the last key is not read
#pragma unroll 1
        for (int x = 0; x < kLoads; ++x)
          cp16_if((dst + x * 512) ^ (HD == 128 && values && x % 2 ? 64 : 0), src + x * 512,
                  pg >= 0 && key0 + (x * 512 + lane * 16) / HD < seen);
      }
      cp_commit();
    };
    // Queries: lane (g, t) holds dims 64 b + 16 t .. + 15 of row g of each tile, four k steps of four
    // dims, the order in which the lanes read the keys' codes (16 bytes at a time).
    uint4 raw[NQ][2 * KB];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int y = 8 * n + g, x = tile * kRows + y, i = args.rep.by(x);
      const __nv_bfloat16* p = (const __nv_bfloat16*)a.q + (row0 + i) * a.q_tok + (long)(kh * rep + x - i * rep) * HD + 16 * t;
#pragma unroll
      for (int b = 0; b < 2 * KB; ++b) {
        raw[n][b] = make_uint4(0, 0, 0, 0);
        if (y < rows_here) raw[n][b] = *reinterpret_cast<const uint4*>(p + 64 * (b / 2) + 8 * (b & 1));
      }
    }
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

    uint32_t qf[NQ][4 * KB][2];
    float qs[NQ][2];  // of rows 2 t and 2 t + 1
    int pos[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float big = 0.f;
#pragma unroll
      for (int b = 0; b < 2 * KB; ++b) {
        const uint32_t u[4] = {raw[n][b].x, raw[n][b].y, raw[n][b].z, raw[n][b].w};
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
        const uint32_t u[4] = {raw[n][b].x, raw[n][b].y, raw[n][b].z, raw[n][b].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          qf[n][2 * b + j / 2][j & 1] =
              pack_f16(__uint_as_float(u[j] << 16) * up, __uint_as_float(u[j] & 0xffff0000u) * up);
      }
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int yy = 8 * n + 2 * t + z;
        qs[n][z] = __shfl_sync(0xffffffffu, back, (2 * t + z) * 4);
        pos[n][z] = yy < rows_here ? pos0 + args.rep.by(tile * kRows + yy) : -1;
      }
    }

    float o[MT][NQ][4], m[NQ][2], l[NQ][2], unit = 0.f, least = 0.f;
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
        float s2[NQ][4];  // every other k step: chains of dependent products half as long
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[h][n][x] = s2[n][x] = 0.f;
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
            for (int n = 0; n < NQ; ++n)
              mma(j & 1 ? s2[n] : s[h][n], a0, a1, a2, a3, qf[n][4 * b + j][0], qf[n][4 * b + j][1]);
          }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[h][n][x] += s2[n][x];
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
      const float v_unit = fabsf(vs);
      if (v_unit != unit && v_unit > 0.f) {  // sums in units of this page's scale
        // 2^-60 at least of the largest unit that the sums have had, however often it falls: a page of zeros
        // has 2^-110, and the sums (2^15 * 448 a key) times all falls stay below 2^104 for 2^20 keys.
        least = fmaxf(least, v_unit * 0x1p-60f);
        const float now = power_of_two(fmaxf(v_unit, least)), inv = inverse_power(now);
        ratio = unit * inv;
        pscale = v_unit * inv;
        unit = now;
      }
      // Weights are at most 1 and meet the values as f16 times 2^15. The 15 is no part of the exponent: it would
      // round away, or up to 32, beside scores of 2^24 and more.
      pscale *= 0x1p15f;
      uint32_t pf[NQ][2][2];
      bool moved = false;
      float factor[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float f0 = qs[n][0] * ks, f1 = qs[n][1] * ks;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[h][n][x] *= x & 1 ? f1 : f0;
        if (diag) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (key0 + 16 * h + g + 8 * (x >> 1) > pos[n][x & 1]) s[h][n][x] = -INFINITY;
        }
        float top[2];
#pragma unroll
        for (int z = 0; z < 2; ++z)
          top[z] = fmaxf(fmaxf(s[0][n][z], s[0][n][z + 2]), fmaxf(s[1][n][z], s[1][n][z + 2]));
        float ref[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const float mn = fmaxf(m[n][z], group_max(top[z]));
          ref[z] = mn == -INFINITY ? 0.f : mn;
          const float alpha = ex2(m[n][z] - ref[z]);
          m[n][z] = mn;
          l[n][z] *= alpha;
          factor[n][z] = alpha * ratio;
          moved |= factor[n][z] != 1.f;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) p[x] = ex2(s[h][n][x] - ref[x & 1]);
          l[n][0] += p[0] + p[2];
          l[n][1] += p[1] + p[3];
#pragma unroll
          for (int x = 0; x < 4; ++x) p[x] *= pscale;
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
        take_out_nan<HD>(smem + (vb - ring0), sh_nan, lane, key0, rows_here, args.rep, tile * kRows, pos0);
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
            const uint32_t p = __byte_perm(vw[0][x], vw[1][x], y ? 0x7362 : 0x5140);
            const uint32_t q = __byte_perm(vw[2][x], vw[3][x], y ? 0x7362 : 0x5140);
            const uint32_t a0 = f16_lo(p), a1 = f16_hi(p), a2 = f16_lo(q), a3 = f16_hi(q);
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
    const float o_down = args.down * 0x1p-15f;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        // The outputs' 2^15 goes, and the sum of a request's weights is kept below 1 from here on, so that no sum of
        // p v passes the largest |v|: a mean of values of 2^120 is finite where their sum is not.
        const float sum = group_sum(l[n][z]) * args.down;
        const int y = 8 * n + 2 * t + z;
        if (g == 0) {
          sh_m[warp][y] = m[n][z];
          sh_l[warp][y] = sum;
        }
        if (y < rows_here) {
#pragma unroll
          for (int j = 0; j < MT; ++j)
            *reinterpret_cast<float2*>(so + y * HD + g * (HD / 8) + 2 * j) =
                make_float2(o[j][n][z] * o_down * unit, o[j][n][z + 2] * o_down * unit);
        }
      }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const int slot = 2 * blockIdx.x + (seg_start >= begin ? 1 : 0);
    // what a cluster's CTA has of the segment, behind the warps' parts
    float* part = reinterpret_cast<float*>(smem) + kWarps * kRows * HD;
    float* part_ml = part + kRows * HD;
    auto out_row = [&](int y) {
      const int x = tile * kRows + y, i = args.rep.by(x);
      return (__nv_bfloat16*)a.out + ((long)(row0 + i) * a.H + kh * rep + x - i * rep) * HD + lane * E;
    };
    for (int y = warp; y < rows_here; y += kWarps) {
      float mx = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
      for (int i = 0; i < kWarps; ++i) mx = fmaxf(mx, sh_m[i][y]);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float f = part_weight(sh_m[i][y], sh_l[i][y], mx);
        sum += sh_l[i][y] * f;
        float v[E];
        load_f32(reinterpret_cast<float*>(smem) + (i * kRows + y) * HD + lane * E, v);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += v[e] * f;
      }
      if (sh_any_nan) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (sh_nan[y * HD + lane * E + e]) {
            acc[e] = NAN;
            sh_nan[y * HD + lane * E + e] = 0;
          }
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = sum == 0.f ? 0.f : acc[e] * inv;
        store_bf16(out_row(y), acc);
      } else {
        store_f32((CLUSTER ? part + y * HD : w.acc + ((long)slot * kRows + y) * HD) + lane * E, acc);
        if (lane == 0) {
          float* ml = CLUSTER ? part_ml + 2 * y : w.ml + (slot * kRows + y) * 2;
          ml[0] = mx;
          ml[1] = sum;
        }
      }
    }
    if constexpr (CLUSTER) {
      if (parts > 1) {  // a segment has one CTA whole only if the others have none of it
        const bool join = steps > 1;
        if (join) {
          cluster_sync();
          for (int y = rank * kWarps + warp; y < rows_here; y += parts * kWarps) {
            float mx = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = 0.f;
            for (int i = 0; i < parts; ++i) mx = fmaxf(mx, ld_rank(in_rank(part_ml + 2 * y, i)));
#pragma unroll 8
            for (int i = 0; i < parts; ++i) {
              const uint32_t ml = in_rank(part_ml + 2 * y, i), from = in_rank(part + y * HD + lane * E, i);
              const float l = ld_rank(ml + 4), f = part_weight(ld_rank(ml), l, mx);
              sum += l * f;
#pragma unroll
              for (int e = 0; e < E; ++e) acc[e] += ld_rank(from + 4 * e) * f;
            }
            const float inv = 1.f / sum;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = sum == 0.f ? 0.f : acc[e] * inv;
            store_bf16(out_row(y), acc);
          }
          cluster_sync();  // no CTA leaves while another reads its part
        }
      }
      return;
    }
    __syncthreads();
    at += s1 - s0;
  }
}

// Joins the segments that several CTAs shared: one CTA for each output row and head, whose warps
// share the parts.
template <int HD>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ Args args) {
  constexpr int E = HD / 32;
  const Kv8Cache& c = args.c;
  const Kv8Attention& a = args.a;
  __shared__ float sh[kJoinWarps][HD], sh_m[kJoinWarps], sh_l[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const Work w = work_of(a.work, a.grid, a.tile, HD);
  const int rep = args.rep.d;
  wait_for_previous();
  int r = row;
  const int total = w.prefix[a.R];
  if (total == 0) return;  // nothing was computed: starts are refused, or no request has a row
  if (a.starts != nullptr) {
    // Rows of no request. Before the first, row - starts[r] is negative: every index below would lie
    // before its array.
    if (row < a.starts[0] || row >= a.starts[a.R]) return;
    r = owner(a.starts, a.R, row);
  }
  int row0;
  const int n_new = new_rows(a, r, row0);
  if (row < row0 || row - row0 >= n_new) return;
  const int start = w.prefix[r];
  const int steps = steps_of(a.width << args.page_shift, a.lens[r]);
  if (steps == 1) return;  // one step has one CTA
  const int kh = args.rep.by(h), x = (row - row0) * rep + h - kh * rep, tile = x / a.tile, y = x % a.tile;
  const Share share(total, used_ctas(a, total));
  const int s0 = start + (tile * c.hkv + kh) * steps;
  const int c0 = share.cta(s0), c1 = share.cta(s0 + steps - 1);
  if (c0 == c1) return;  // written by its CTA
  float mx = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int b = c0 + warp; b <= c1; b += kJoinWarps) {
    const int slot = (2 * b + (b == c0)) * a.tile + y;
    const float2 ml = *reinterpret_cast<const float2*>(w.ml + slot * 2);
    float v[E];
    load_f32(w.acc + (long)slot * HD + lane * E, v);
    const float mn = fmaxf(mx, ml.x);
    const float f0 = part_weight(mx, sum, mn), f1 = part_weight(ml.x, ml.y, mn);
    sum = sum * f0 + ml.y * f1;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f0 + v[e] * f1;
    mx = mn;
  }
  store_f32(sh[warp] + lane * E, acc);
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

template <int HD, int NQ, bool CLUSTER>
int launch(const Args& args, cudaStream_t st) {
  constexpr int kRing = kWarps * stages_of(HD, CLUSTER) * 2 * kChunk * HD;
  static_assert(kWarps * 8 * NQ * HD * 4 <= kRing, "the join fits the ring");
  static_assert(!CLUSTER || (kWarps + 1) * 8 * NQ * HD * 4 + 64 * NQ <= kRing, "so does a cluster's part");
  const Kv8Attention& a = args.a;
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<bool> raised[64];
  if (dev < 0 || dev >= 64) return kErrBadArgsHost;
  if (!raised[dev].load()) {
    if (cudaFuncSetAttribute(attention_kernel<HD, NQ, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kRing + (kMaxRequests + 1) * 4) != cudaSuccess)
      return kErrBadArgsHost;
    raised[dev].store(true);
  }
  count_launch();
  if (launch_early(attention_kernel<HD, NQ, CLUSTER>, dim3((unsigned)a.grid), kThreads, kRing + (a.R + 1) * 4, st,
                   CLUSTER ? a.cluster : 1, args) != cudaSuccess)
    return kErrBadArgsHost;
  if (CLUSTER) return 0;
  count_launch();
  return launch_early(join_kernel<HD>, dim3((unsigned)(a.rows * a.H)), 32 * kJoinWarps, 0, st, 1, args) == cudaSuccess
             ? 0
             : kErrBadArgsHost;
}

}  // namespace

bool kv8_attention_plan(Kv8Attention& a, int hkv, int page, int hd, int sms) {
  if (a.R < 1 || a.R > kMaxRequests || a.rows < 0 || hkv < 1 || a.H % hkv) return false;
  if ((long)a.width * page > 1 << 30 || (long)a.rows * a.H > 1 << 30) return false;
  // Rows of a tile: what a request's rows of one kv head need on average (8 in decode up to 8 query
  // heads a group), 16 at most at hd 128 and 32 at hd 64, where the registers end.
  const long n = ((long)a.rows + a.R - 1) / a.R * (a.H / hkv);
  a.tile = n <= 8 ? 8 : (n <= 16 || hd == 128 ? 16 : 32);
  const long tiles = ((long)a.rows * (a.H / hkv) + a.tile - 1) / a.tile + a.R;  // each request rounds up at most once
  const long steps = std::max(1L, ((long)a.width * page + kStep - 1) / kStep);
  const long segs = a.starts == nullptr ? (long)a.R * hkv * ((a.H / hkv + a.tile - 1) / a.tile) : tiles * hkv;
  if ((double)tiles * hkv * steps > 2.0e9) return false;
  const long ctas = (long)sms * ctas_per_sm(hd, a.tile, false), at_once = (long)sms * ctas_per_sm(hd, a.tile, true);
  a.cluster = 0;
  int size = 8;
  while (size > 1 && segs * size > at_once) size /= 2;
  while (size > 1 && size / 2 >= steps) size /= 2;
  const long most_steps = size * (long)(2 * segs * size <= ctas ? kFewClusterSteps : kClusterSteps);
  if (a.tile <= 16 && segs * size <= at_once && steps <= most_steps) {
    a.cluster = size;
    a.grid = (int)(segs * size);
  } else {
    const long most = tiles * hkv * steps;
    a.resident = (int)std::min(most, ctas);
    a.grid = (int)std::max<long>(a.resident, std::min(kRounds * ctas, most / kManySteps));
  }
  return true;
}

long kv8_attention_work(const Kv8Attention& a, int hd) {
  return a.cluster ? 0 : 2L * a.grid * a.tile * (hd + 2) + a.R + 1;
}

int launch_kv8_attention(const Kv8Cache& c, const Kv8Attention& a, cudaStream_t st) {
  if (a.rows < 1) return 0;
  if (c.page % kChunk || (c.page & (c.page - 1)) || a.grid < 1) return kErrBadArgsHost;
  Args args{c, a, make_div(a.H / c.hkv), make_div(c.hkv), 0, 1.f};
  while ((1 << args.page_shift) < c.page) ++args.page_shift;
  for (long n = 1; n < (long)a.width * c.page; n *= 2) args.down *= 0.5f;
  if (a.cluster) {
    if (c.hd == 64 && a.tile == 8) return launch<64, 1, true>(args, st);
    if (c.hd == 64 && a.tile == 16) return launch<64, 2, true>(args, st);
    if (c.hd == 128 && a.tile == 8) return launch<128, 1, true>(args, st);
    if (c.hd == 128 && a.tile == 16) return launch<128, 2, true>(args, st);
    return kErrBadArgsHost;
  }
  if (c.hd == 64 && a.tile == 8) return launch<64, 1, false>(args, st);
  if (c.hd == 64 && a.tile == 16) return launch<64, 2, false>(args, st);
  if (c.hd == 64 && a.tile == 32) return launch<64, 4, false>(args, st);
  if (c.hd == 128 && a.tile == 8) return launch<128, 1, false>(args, st);
  if (c.hd == 128 && a.tile == 16) return launch<128, 2, false>(args, st);
  return kErrBadArgsHost;
}

}  // namespace mxk
