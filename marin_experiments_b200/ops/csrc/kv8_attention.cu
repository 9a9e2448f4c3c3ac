// Attention over the paged 8-bit cache: for each request, its new rows (one in decode, several when
// drafts are verified or a turn is appended) against all of its cached tokens,
//   out = sum_j softmax_j(scale * q . k_j) v_j over the positions j <= len - rows + i of row i.
//
// What bounds it: the cache is read once, 2 * hd bytes a token and kv head, for 4 * hd * rows * H/hkv
// operations; below about 60 rows of a group that is memory. The rows of one kv head (new rows x
// query heads of the group) form tiles of 16, the M of mma.sync.m16n8k16: a tcgen05 tile has 128
// rows, of which a decode step would fill 1 to 8, and takes no e4m3 operand against bf16 queries.
//
// Exactness: e4m3 codes convert to f16 without rounding. A query row is multiplied by a power of two
// that brings its largest value to 2^13, so its bf16 values are exact in f16 too (what is 2^-37 of
// the row's largest rounds). Scores and sums are fp32. The weights p = 2^(s - max + 15) round to f16,
// 2^-12 of a weight at most (below 2^-29 of the largest weight: absolutely); scales of pages multiply
// fp32 products, so pages of very different size do not disturb one another.
//
// Split: all (request, row tile, kv head) segments are cut into steps of 128 keys, and the steps are
// shared evenly among the CTAs, whatever the lengths. A segment that one CTA has whole is written at
// once; else its CTAs write (max, sum, sum p v) and a second kernel joins them in order, so results
// do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kernels.h"

namespace mxk {
namespace {

constexpr int kRows = 16;            // rows of a tile
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 32;           // keys a warp takes at once: always inside one page
constexpr int kStep = kChunk * kWarps;
constexpr int kMaxRequests = 4096;
constexpr int kStages = 3;

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

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// The weight of a partial result with maximum m and sum l under the common maximum mx. A part that
// saw no key has m = -inf and l = 0; one that met a NaN score keeps it.
__device__ __forceinline__ float part_weight(float m, float l, float mx) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return exp2f(m - mx);
}

struct Work {
  float* acc;   // [2 * grid][kRows][hd]
  float* ml;    // [2 * grid][kRows][2]
  int* prefix;  // [R + 1] steps before each request
};
__host__ __device__ inline Work work_of(float* w, int grid, int hd) {
  Work k;
  k.acc = w;
  k.ml = w + 2L * grid * kRows * hd;
  k.prefix = reinterpret_cast<int*>(k.ml + 2L * grid * kRows * 2);
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

template <int HD>
__global__ void __launch_bounds__(kThreads, 2) attention_kernel(Kv8Cache c, Kv8Attention a) {
  constexpr int KS = HD / 16;              // k steps of q . k
  constexpr int NT = HD / 8;               // 8-column tiles of the output
  constexpr int kStageBytes = 2 * kChunk * HD;
  constexpr int kLoads = kChunk * HD / 16 / 32;  // 16-byte copies a lane, keys or values
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int warp_sums[kWarps];
  __shared__ float sh_m[kWarps][kRows], sh_l[kWarps][kRows];
  int* prefix = reinterpret_cast<int*>(smem + kWarps * kStages * kStageBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rep = a.H / c.hkv;
  const Work w = work_of(a.work, a.grid, HD);

  // Steps before each request. Ascending starts keep the sum below the host's bound; with any other
  // nothing is computed.
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

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * kStages * kStageBytes;
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

    // rows g and g + 8 of the tile: which row of q, which head, which last position
    const int rows_here = min(kRows, n_new * rep - tile * kRows);
    int pos[2];
    const __nv_bfloat16* qp[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int y = g + 8 * i, x = tile * kRows + y;
      pos[i] = y < rows_here ? len_in - n_new + x / rep : -1;
      qp[i] = y < rows_here ? (const __nv_bfloat16*)a.q + (row0 + x / rep) * a.q_tok + (long)(kh * rep + x % rep) * HD
                            : nullptr;
    }
    // lane t holds the dims 64 s + 16 t .. + 15 of its rows: four k steps of four dims, the order in
    // which the lanes read the keys' codes (16 bytes at a time)
    uint32_t qf[KS][4];
    float qs[2];
    {
      uint4 raw[2][KS / 2];
      float big[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int s = 0; s < KS / 2; ++s) {
          raw[i][s] = qp[i] ? *reinterpret_cast<const uint4*>(qp[i] + 64 * (s / 2) + 16 * t + 8 * (s & 1))
                            : make_uint4(0, 0, 0, 0);
          const uint32_t u[4] = {raw[i][s].x, raw[i][s].y, raw[i][s].z, raw[i][s].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            big[i] = fmaxf(big[i], fmaxf(fabsf(__uint_as_float(u[j] << 16)), fabsf(__uint_as_float(u[j] & 0xffff0000u))));
        }
        big[i] = quad_max(big[i]);
        // 2^-e brings the largest to [2^13, 2^14); infinities and zeros stay
        int e = ((__float_as_int(big[i]) >> 23) & 0xff) - 127 - 13;
        if (!(big[i] > 0.f) || big[i] == INFINITY) e = 0;
        e = max(-126, e);
        const float up = __int_as_float((127 - e) << 23);
        qs[i] = __int_as_float((127 + e) << 23) * (a.scale * 1.4426950408889634f);
#pragma unroll
        for (int s = 0; s < KS / 2; ++s) {
          const uint32_t u[4] = {raw[i][s].x, raw[i][s].y, raw[i][s].z, raw[i][s].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t h = pack_f16(__uint_as_float(u[j] << 16) * up, __uint_as_float(u[j] & 0xffff0000u) * up);
            qf[2 * s + j / 2][i + 2 * (j & 1)] = h;
          }
        }
      }
    }

    float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[j][x] = 0.f;

    // this warp's chunks of the segment: first + kWarps * i, i < count
    const int tile_last = len_in - n_new + (tile * kRows + rows_here - 1) / rep;    // last position any row sees
    const int tile_first = len_in - n_new + tile * kRows / rep;                     // last position every row sees
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
    auto load = [&](int i) {  // chunk i into its stage; page ids of its block of 32 are in page_id
      const int key0 = (first + i * kWarps) * kChunk;
      const int pg = __shfl_sync(0xffffffffu, page_id, i & 31);
      const uint32_t kd = ring + (i % kStages) * kStageBytes, vd = kd + kChunk * HD;
      const long off = (((long)max(pg, 0) * c.hkv + kh) * c.page + key0 % c.page) * HD;
      const uint8_t* kp = (const uint8_t*)c.k + off;
      const uint8_t* vp = (const uint8_t*)c.v + off;
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        const int byte = (x * 32 + lane) * 16, key = byte / HD, col = byte % HD / 16;
        const bool in = pg >= 0 && key0 + key < seen;  // what lies behind the last key is not read
        int kc, vc;
        if (HD == 128) {
          kc = col ^ ((key & 1) << 2);
          vc = col ^ (((key >> 1) & 3) << 1);
        } else {
          kc = col;
          vc = col ^ (((key >> 1) & 1) << 1);
        }
        cp16(kd + key * HD + kc * 16, kp + byte, in);
        cp16(vd + key * HD + vc * 16, vp + byte, in);
      }
    };
    // Stages are filled in order and a lane-parallel block of page ids serves 32 chunks, so the ids
    // of the block being loaded and the scales of the block being used are kept apart.
    float ks_use = 0.f, vs_use = 0.f;
    if (count > 0) {
      fetch_pages(0);
      ks_use = ks_all;
      vs_use = vs_all;
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (i < count) load(i);
      cp_commit();
    }
    for (int i = 0; i < count; ++i) {
      const int nx = i + kStages - 1;
      if (nx < count && (nx & 31) == 0) fetch_pages(nx);
      __syncwarp();  // all lanes are done with the stage that is filled next
      if (nx < count) load(nx);
      cp_commit();
      cp_wait<kStages - 1>();
      __syncwarp();
      if (i > 0 && (i & 31) == 0) {  // fetched above, at most kStages - 1 chunks ago
        ks_use = ks_all;
        vs_use = vs_all;
      }
      float ks = __shfl_sync(0xffffffffu, ks_use, i & 31);
      const float vs = __shfl_sync(0xffffffffu, vs_use, i & 31);
      if (too_long) ks = NAN;
      const int key0 = (first + i * kWarps) * kChunk;
      const uint32_t kb = ring + (i % kStages) * kStageBytes, vb = kb + kChunk * HD;

      // scores of 16 rows x 32 keys
      float s[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s[n][x] = 0.f;
        const int key = 8 * n + g;
#pragma unroll
        for (int b = 0; b < HD / 64; ++b) {
          const int col = 4 * b + t;
          const uint4 u = lds128(kb + key * HD + (HD == 128 ? col ^ ((key & 1) << 2) : col) * 16);
          mma(s[n], qf[4 * b + 0], f16_lo(u.x), f16_hi(u.x));
          mma(s[n], qf[4 * b + 1], f16_lo(u.y), f16_hi(u.y));
          mma(s[n], qf[4 * b + 2], f16_lo(u.z), f16_hi(u.z));
          mma(s[n], qf[4 * b + 3], f16_lo(u.w), f16_hi(u.w));
        }
      }
      const bool diag = key0 + kChunk > min(len, tile_first + 1);  // some row does not see some key
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float v = s[n][x] * (qs[x >> 1] * ks);
          if (diag && key0 + 8 * n + 2 * t + (x & 1) > pos[x >> 1]) v = -INFINITY;
          s[n][x] = v;
          top[x >> 1] = fmaxf(top[x >> 1], v);
        }
      float alpha[2], sub[2];
#pragma unroll
      for (int i2 = 0; i2 < 2; ++i2) {
        const float mn = fmaxf(m[i2], quad_max(top[i2]));
        const float ref = mn == -INFINITY ? 0.f : mn;
        alpha[i2] = exp2f(m[i2] - ref);
        sub[i2] = ref - 15.f;
        m[i2] = mn;
        l[i2] *= alpha[i2];
      }
      uint32_t pf[2][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float p[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          p[x] = exp2f(s[n][x] - sub[x >> 1]);
          l[x >> 1] += p[x];
        }
        pf[n >> 1][2 * (n & 1) + 0] = pack_f16(p[0], p[1]);
        pf[n >> 1][2 * (n & 1) + 1] = pack_f16(p[2], p[3]);
      }
      // sum p v: lane g has the dims g * NT .. + NT - 1 of the values, column g of NT tiles
      constexpr int VW = NT / 4;  // words a lane reads of a value row
      uint32_t vw[2][4][VW];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int key = 16 * h + 2 * t + (q & 1) + 8 * (q >> 1);
          if constexpr (HD == 128) {
            const uint4 u = lds128(vb + key * HD + ((g ^ (((key >> 1) & 3) << 1)) * 16));
            vw[h][q][0] = u.x; vw[h][q][1] = u.y; vw[h][q][2] = u.z; vw[h][q][3] = u.w;
          } else {
            const uint2 u = lds64(vb + key * HD + (((g >> 1) ^ (((key >> 1) & 1) << 1)) * 16) + (g & 1) * 8);
            vw[h][q][0] = u.x; vw[h][q][1] = u.y;
          }
        }
      if (diag) {
        // A NaN in a value that a row does not see must not reach it through 0 * NaN, and one that it
        // sees must: count the NaN codes each row sees, take them out, and mark the columns.
        uint32_t nan_any = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int x = 0; x < VW; ++x) nan_any |= ((vw[h][q][x] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        if (__any_sync(0xffffffffu, nan_any != 0)) {
          uint32_t see[2][4];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
              const int k0 = key0 + 8 * n + 2 * t;
              see[n >> 1][2 * (n & 1) + i2] = (k0 <= pos[i2] ? 0x3c00u : 0u) | (k0 + 1 <= pos[i2] ? 0x3c000000u : 0u);
            }
#pragma unroll
          for (int x = 0; x < VW; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              float hit[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t b[2] = {0, 0};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const uint32_t code = (vw[h][q][x] >> (8 * y)) & 0x7f;
                  if (code == 0x7f) {
                    b[q >> 1] |= 0x3c00u << (16 * (q & 1));
                    vw[h][q][x] &= ~(0xffu << (8 * y));
                  }
                }
                mma(hit, see[h], b[0], b[1]);
              }
#pragma unroll
              for (int z = 0; z < 4; ++z)
                if (hit[z] > 0.f) o[4 * x + y][z] = NAN;
            }
        }
      }
#pragma unroll
      for (int x = 0; x < VW; ++x) {
        float part[4][4];
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int z = 0; z < 4; ++z) part[y][z] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // bytes of keys (2t, 2t + 1) and (2t + 8, 2t + 9) side by side, for four dims
          const uint32_t a0 = __byte_perm(vw[h][0][x], vw[h][1][x], 0x5140), a1 = __byte_perm(vw[h][0][x], vw[h][1][x], 0x7362);
          const uint32_t b0 = __byte_perm(vw[h][2][x], vw[h][3][x], 0x5140), b1 = __byte_perm(vw[h][2][x], vw[h][3][x], 0x7362);
          mma(part[0], pf[h], f16_lo(a0), f16_lo(b0));
          mma(part[1], pf[h], f16_hi(a0), f16_hi(b0));
          mma(part[2], pf[h], f16_lo(a1), f16_lo(b1));
          mma(part[3], pf[h], f16_hi(a1), f16_hi(b1));
        }
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int z = 0; z < 4; ++z) o[4 * x + y][z] = o[4 * x + y][z] * alpha[z >> 1] + part[y][z] * vs;
      }
    }
    cp_wait<0>();

    // join the warps: through shared memory, which the ring no longer needs
    __syncthreads();
    l[0] = quad_sum(l[0]);
    l[1] = quad_sum(l[1]);
    if (t == 0) {
      sh_m[warp][g] = m[0];
      sh_m[warp][g + 8] = m[1];
      sh_l[warp][g] = l[0];
      sh_l[warp][g + 8] = l[1];
    }
    float* so = reinterpret_cast<float*>(smem) + warp * kRows * HD;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int z = 0; z < 4; ++z) so[(g + 8 * (z >> 1)) * HD + (2 * t + (z & 1)) * NT + j] = o[j][z];
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

// Joins the segments that several CTAs shared. One warp for each output row and head.
template <int HD>
__global__ void __launch_bounds__(128) combine_kernel(Kv8Cache c, Kv8Attention a) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const long i = blockIdx.x * 4L + (threadIdx.x >> 5);
  if (i >= (long)a.rows * a.H) return;
  const int row = (int)(i / a.H), h = (int)(i % a.H);
  const Work w = work_of(a.work, a.grid, HD);
  const int rep = a.H / c.hkv;
  int r = row;
  if (a.starts != nullptr) {
    if (row >= a.starts[a.R]) return;
    r = owner(a.starts, a.R, row);
  } else if (row >= a.R) {
    return;
  }
  int row0;
  if (row - (a.starts ? a.starts[r] : r) >= new_rows(a, r, row0)) return;
  const int total = w.prefix[a.R];
  if (total == 0) return;
  const int steps = steps_of(a, c.page, a.lens[r]);
  const int x = (row - row0) * rep + h % rep, tile = x / kRows, y = x % kRows;
  const int s0 = w.prefix[r] + (tile * c.hkv + h / rep) * steps, s1 = s0 + steps;
  const int used = min(a.grid, total);
  const int c0 = cta_of(s0, total, used), c1 = cta_of(s1 - 1, total, used);
  if (c0 == c1) return;  // written by its CTA
  float mx = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int b = c0; b <= c1; ++b) mx = fmaxf(mx, w.ml[((2 * b + (b == c0)) * kRows + y) * 2]);
  for (int b = c0; b <= c1; ++b) {
    const int slot = 2 * b + (b == c0);
    const float l = w.ml[(slot * kRows + y) * 2 + 1];
    const float f = part_weight(w.ml[(slot * kRows + y) * 2], l, mx);
    sum += l * f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += w.acc[((long)slot * kRows + y) * HD + e * 32 + lane] * f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    ((__nv_bfloat16*)a.out)[((long)row * a.H + h) * HD + e * 32 + lane] =
        __float2bfloat16(sum == 0.f ? 0.f : acc[e] / sum);
}

template <int HD>
int launch(const Kv8Cache& c, const Kv8Attention& a, cudaStream_t st) {
  const int smem = kWarps * kStages * 2 * kChunk * HD + (a.R + 1) * 4;
  static_assert(kWarps * kRows * HD * 4 <= kWarps * kStages * 2 * kChunk * HD, "the join fits the ring");
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<bool> raised[64];
  if (dev < 0 || dev >= 64) return kErrBadArgsHost;
  if (!raised[dev].load()) {
    if (cudaFuncSetAttribute(attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kWarps * kStages * 2 * kChunk * HD + (kMaxRequests + 1) * 4) != cudaSuccess)
      return kErrBadArgsHost;
    raised[dev].store(true);
  }
  count_launch();
  attention_kernel<HD><<<a.grid, kThreads, smem, st>>>(c, a);
  count_launch();
  combine_kernel<HD><<<(unsigned)(((long)a.rows * a.H + 3) / 4), 128, 0, st>>>(c, a);
  return cudaGetLastError() == cudaSuccess ? 0 : kErrBadArgsHost;
}

}  // namespace

int kv8_attention_grid(int rows, int H, int hkv, int R, int width, int page, int sms) {
  if (R < 1 || R > kMaxRequests || rows < 0 || hkv < 1 || H % hkv || (long)width * page > 0x7fffffffL) return -1;
  const long tiles = ((long)rows * (H / hkv) + kRows - 1) / kRows + R;  // each request rounds up at most once
  const long steps = ((long)width * page + kStep - 1) / kStep;
  if ((double)tiles * hkv * (steps < 1 ? 1 : steps) > 2.0e9) return -1;
  const long most = tiles * hkv * (steps < 1 ? 1 : steps), ctas = 2L * sms;
  return (int)(most < ctas ? (most < 1 ? 1 : most) : ctas);
}

long kv8_attention_work(int grid, int R, int hd) { return 2L * grid * kRows * (hd + 2) + R + 1; }

int launch_kv8_attention(const Kv8Cache& c, const Kv8Attention& a, cudaStream_t st) {
  if (a.rows < 1) return 0;
  if (c.page % kChunk || a.grid < 1) return kErrBadArgsHost;
  if (c.hd == 64) return launch<64>(c, a, st);
  if (c.hd == 128) return launch<128>(c, a, st);
  return kErrBadArgsHost;
}

}  // namespace mxk
