// Products with 4-bit weights: y[t, n] = sum_k x[t, k] * code[n, k] * scale[n, k / group], for the few
// rows (1 to 32; w4_wide.cu has 33 to 64) of a decode step, with the residual added or the SwiGLU applied before the one
// rounding to bf16.
//
// Layout: int32 words [N][K / 8]. Within each 128 values of a row word 4 t + i of the 16 holds values
// 32 i + 8 t .. + 7, and a word holds values 0 2 4 6 1 3 5 7 from its lowest bits up, each as code + 8.
// So a lane's 16-byte load (words 4 t .. 4 t + 3) gives it, for each 32 values of the row, the eight
// that mma.sync.m16n8k16 takes from lane t in two k steps, and word >> 4 j & 0x000f000f is the pair
// (2 j, 2 j + 1) in the halves of a register. The k order inside a step is free as long as x has the
// same: lane t reads x at the same eight places, 16 bytes at once.
//
// Exactness: 0x4300 | c is the bf16 number 128 + c, so one bf16x2 subtraction of 136 gives the code
// exactly; x is bf16 as it stands; products and sums are fp32, and the scale multiplies the group's
// fp32 sum.
//
// What bounds it: at 151936 x 4096 nearly the N * K / 2 bytes of weights (5.1 TB/s); else shared memory,
// which gives 512 bytes of x to every 16 x 32 weights and takes and gives their words (64 weights a clock
// and SM at most; 42 reached) next to the conversions' issue slots; at a few MB a matrix also the start
// and one round trip to memory.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "kernels.h"
#include "pdl.cuh"
#include "w4.cuh"

namespace mxk {
namespace {

constexpr int kWarps = 16;
constexpr int kFew = 32;    // rows of x that these kernels take; w4_wide.cu takes more (times of both there)
constexpr int kStages = 2;  // units of a warp on their way
// Blocks of 128 values of K in a unit: 256 bytes of a row, or 128 where x needs the shared memory.
__host__ __device__ constexpr int blocks_of(int nt) { return nt == 1 ? 4 : 2; }
constexpr int kMaxSmem = 226 * 1024;  // of 227 KB; part_tile is static
constexpr double kSliceCost = 0.1;  // of one more slice, in units
constexpr int kThreads = kWarps * 32;

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The first product of a sum.
__device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Pitch of x's rows in shared memory: 64 bytes off a multiple of 128, so that the two rows that eight
// lanes read at once lie in different banks.
__host__ __device__ inline int x_pitch_of(int units, int bu) { return units * bu * 128 + 32; }

// The scales of a row in one unit of BU blocks, two to a word.
template <int BU, int GW>
struct Scales {
  static constexpr int kWords = BU * 2 / GW;
  uint32_t v[kWords];
  __device__ __forceinline__ float at(int i) const {
    return __uint_as_float(i & 1 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
  }
  // `n` of them are there; `aligned`: all, and at a multiple of their size (16 bytes at most)
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int n, bool aligned) {
    if (aligned) {
      if constexpr (kWords == 1) v[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
      if constexpr (kWords == 2) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        v[0] = u.x, v[1] = u.y;
      }
      if constexpr (kWords >= 4) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
          v[i] = u.x, v[i + 1] = u.y, v[i + 2] = u.z, v[i + 3] = u.w;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2 * kWords; ++i) {
        const uint32_t h = i < n ? __ldg(reinterpret_cast<const uint16_t*>(p) + i) : 0;
        v[i / 2] = i & 1 ? v[i / 2] | h << 16 : h;
      }
    }
  }
};

// One CTA of 16 warps on each SM. Its slice of x stays in shared memory. A tile is 16 rows of W (with
// GLU 8 gate rows and the 8 up rows of the same units). The CTA's tiles one after the other, each cut
// into units of BU blocks of 128 values of K, are shared evenly among its warps: a warp walks along
// rows, so that it reads BU * 64 bytes of a row at once (16 rows x 256 bytes: 6.5 TB/s, 16 x 128: 5.7),
// and has at most two tiles in part, whose sums meet in shared memory at the end. The words arrive
// through a ring that each lane fills and reads alone (cp.async, kStages units ahead, across tiles),
// the scales through registers with them, so the stream of weights waits for no barrier. Where x is
// too large for one SM, K is cut into slices with CTAs of their own, and slices_kernel adds their parts.
// NT: tiles of 8 rows of x. GW: words of a lane in one scale group (group / 32).
template <int NT, int GW, bool GLU>
__global__ void __launch_bounds__(kThreads, 1) stream_kernel(const __grid_constant__ W4Args a) {
  constexpr int BU = blocks_of(NT), kUnitBytes = BU * 1024, kPitch = NT * 8 + 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int part_tile[2 * kWarps];  // the tile whose sums in part a place holds
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int slice = blockIdx.y, cta = blockIdx.x;
  const int blocks = a.K / 128, all = (blocks + BU - 1) / BU;  // units of K, the last perhaps of fewer blocks
  int u0 = 0, units = all;
  if (a.slices > 1) {
    u0 = (int)((long)all * slice / a.slices);
    units = (int)((long)all * (slice + 1) / a.slices) - u0;
  }
  const int b0 = BU * u0, nb = min(BU * units, blocks - b0);
  const bool aligned = blocks % BU == 0;
  // shared memory: rings, x, sums of tiles in part (two a warp)
  uint8_t* ring = smem + warp * kStages * kUnitBytes + lane * 16;
  const int x_pitch = x_pitch_of(units, BU);
  __nv_bfloat16* xs = reinterpret_cast<__nv_bfloat16*>(smem + kWarps * kStages * kUnitBytes);
  float* sums = reinterpret_cast<float*>(xs + a.T * x_pitch);

  const int n_tiles = a.per + (cta < a.more), tile0 = cta * a.per + min(cta, a.more);
  auto start_of = [&](int w) {  // of warp w's share, in units of the CTA's tiles
    return a.whole ? (int)((long)n_tiles * w / kWarps) * units : (int)((long)n_tiles * units * w / kWarps);
  };
  int pos = start_of(warp);
  const int end = start_of(warp + 1);
  int tile = pos / units, u = pos - tile * units;

  // the walk ahead
  int ahead = pos, f_tile = tile, f_u = u, put = 0;
  const uint32_t* w_row[2];
  const __nv_bfloat16* s_row[2];
  auto set_rows = [&]() {  // rows g and g + 8 of f_tile
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int n;
      if (GLU) {
        const int unit = (tile0 + f_tile) * 8 + g;
        n = unit / kGlu * 2 * kGlu + unit % kGlu + i * kGlu;
      } else {
        n = (tile0 + f_tile) * 16 + g + 8 * i;
      }
      n = min(n, a.N - 1);  // rows past N repeat the last and are not stored
      w_row[i] = a.codes + (long)n * (a.K / 8) + b0 * 16 + 4 * t;
      s_row[i] = a.scales + ((long)n * blocks + b0) * (4 / GW);
    }
  };
  auto fetch = [&](Scales<BU, GW> (&s)[2]) {
    if (ahead < end) {
      const int have = nb - BU * f_u;  // blocks
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int h = 0; h < BU; ++h)
          if (aligned || h < have) cp16(ring + put + (h * 2 + i) * 512, w_row[i] + (f_u * BU + h) * 16);
        s[i].load(s_row[i] + f_u * (BU * 4 / GW), have * (4 / GW), aligned);
      }
      put = put + kUnitBytes == kStages * kUnitBytes ? 0 : put + kUnitBytes;
      ++ahead;
      if (++f_u == units) {
        f_u = 0;
        ++f_tile;
        if (ahead < end) set_rows();
      }
    }
    cp_commit();
  };
  if (pos < end) set_rows();
  for (int i = tid; i < 2 * kWarps; i += kThreads) part_tile[i] = -1;
  // launched early: the kernel before may still be writing x (or the weights)
  wait_for_previous();
  // The next kernel's CTAs may take this kernel's places as they come free, and do there what needs no
  // memory (4096 x 4096, one row, in a row: 4.85 -> 4.56 us a product; 24576 x 4096, 16 rows: 22.4 -> 21.3).
  let_next_start();
  // x before the weights, which would keep the memory busy for longer than it waits.
  // Blocks that the last unit lacks meet zeros (their codes are what the ring held).
  for (int c = tid; c < units * BU * 16; c += kThreads) {
    const __nv_bfloat16* from = a.x + b0 * 128 + c * 8;
    __nv_bfloat16* to = xs + c * 8;
    if (c < nb * 16) {
#pragma unroll 8
      for (int r = 0; r < a.T; ++r) cp16(to + r * x_pitch, from + r * a.x_tok);
    } else {
      for (int r = 0; r < a.T; ++r) *reinterpret_cast<uint4*>(to + r * x_pitch) = make_uint4(0, 0, 0, 0);
    }
  }
  cp_commit();
  Scales<BU, GW> s_ring[kStages][2];
#pragma unroll
  for (int i = 0; i < kStages; ++i) fetch(s_ring[i]);
  const __nv_bfloat16* xp[NT];  // columns past T repeat the last row and are not stored
#pragma unroll
  for (int n = 0; n < NT; ++n) xp[n] = xs + min(n * 8 + g, a.T - 1) * x_pitch + t * 8;
  cp_wait<kStages>();
  __syncthreads();

  // in registers, so that the conversions take them as operands
  uint32_t magic = 0x43004300u, bias = 0x43084308u;
  asm volatile("" : "+r"(magic), "+r"(bias));
  int get = 0;
#pragma unroll 1
  while (pos < end) {
    const int from = u, to = min(units, u + (end - pos));
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int z = 0; z < 4; ++z) acc[n][z] = 0.f;
#pragma unroll 1
    for (; u < to; ++u) {
      cp_wait<kStages - 1>();
      uint4 w[BU][2];
#pragma unroll
      for (int h = 0; h < BU; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) w[h][i] = *reinterpret_cast<const uint4*>(ring + get + (h * 2 + i) * 512);
      get = get + kUnitBytes == kStages * kUnitBytes ? 0 : get + kUnitBytes;
      Scales<BU, GW> s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = s_ring[0][i];
#pragma unroll
        for (int k = 0; k + 1 < kStages; ++k) s_ring[k][i] = s_ring[k + 1][i];
      }
      fetch(s_ring[kStages - 1]);  // into the place just read, by the lane that read it
#pragma unroll
      for (int h = 0; h < BU; ++h) {
        const uint32_t w0[4] = {w[h][0].x, w[h][0].y, w[h][0].z, w[h][0].w};
        const uint32_t w1[4] = {w[h][1].x, w[h][1].y, w[h][1].z, w[h][1].w};
#pragma unroll
        for (int gi = 0; gi < 4 / GW; ++gi) {
          float part[NT][4];
#pragma unroll
          for (int i = gi * GW; i < (gi + 1) * GW; ++i) {
            uint32_t p0[4], p1[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              p0[j] = pair_of(w0[i], j, magic, bias);
              p1[j] = pair_of(w1[i], j, magic, bias);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (NT > 1 && n >= NT / 2 && n * 8 >= a.T) break;  // columns that T does not reach
              const uint4 y = *reinterpret_cast<const uint4*>(xp[n] + (u * BU + h) * 128 + i * 32);
              if (i == gi * GW) mma0(part[n], p0[0], p1[0], p0[1], p1[1], y.x, y.y);
              else mma(part[n], p0[0], p1[0], p0[1], p1[1], y.x, y.y);
              mma(part[n], p0[2], p1[2], p0[3], p1[3], y.z, y.w);
            }
          }
          const float f0 = s[0].at(h * (4 / GW) + gi), f1 = s[1].at(h * (4 / GW) + gi);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (NT > 1 && n >= NT / 2 && n * 8 >= a.T) break;
#pragma unroll
            for (int z = 0; z < 4; ++z) acc[n][z] += part[n][z] * (z < 2 ? f0 : f1);
          }
        }
      }
    }
    if (from == 0 && to == units) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int tok = n * 8 + 2 * t + z;
          if (tok >= a.T) continue;
          store<GLU>(a, slice, tile0 + tile, g, tok, acc[n][z], acc[n][z + 2]);
          if (!GLU) store<GLU>(a, slice, tile0 + tile, g + 8, tok, acc[n][z + 2], 0.f);
        }
    } else {  // the warp's first tile, begun by others, or its last
      const int place = 2 * warp + (from == 0);
      float* mine = sums + place * 16 * kPitch;
      if (lane == 0) part_tile[place] = tile;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int z = 0; z < 4; ++z) mine[(g + 8 * (z >> 1)) * kPitch + n * 8 + 2 * t + (z & 1)] = acc[n][z];
    }
    pos += to - from;
    u = 0;
    ++tile;
  }
  if (a.whole) return;
  __syncthreads();
  // Tiles that several warps had, one warp at each: their parts in the order of K, which is that of
  // the places.
  constexpr int kOut = GLU ? 8 : 16;
  const int holds = part_tile[lane];
  for (int j = warp; j < n_tiles; j += kWarps) {
    const uint32_t places = __ballot_sync(0xffffffffu, holds == j);
    if (places == 0) continue;
    for (int i = lane; i < kOut * a.T; i += 32) {
      const int r = i % kOut, tok = i / kOut;
      float y = 0.f, up = 0.f;
      for (uint32_t left = places; left; left &= left - 1) {
        const float* p = sums + (__ffs(left) - 1) * 16 * kPitch;
        y += p[r * kPitch + tok];
        if (GLU) up += p[(r + 8) * kPitch + tok];
      }
      store<GLU>(a, slice, tile0 + j, r, tok, y, up);
    }
  }
}

// The weights as bf16 [N][K] (code * scale rounded), for products of many rows on the dense GEMM.
__global__ void __launch_bounds__(256) dequant_kernel(const uint32_t* __restrict__ codes,
                                                      const __nv_bfloat16* __restrict__ scales,
                                                      __nv_bfloat16* __restrict__ out, long words, int K, int group) {
  for (long i = blockIdx.x * 256L + threadIdx.x; i < words; i += gridDim.x * 256L) {
    const int per = K / 8;
    const long n = i / per;
    const int p = (int)(i % per), k = p / 16 * 128 + p % 4 * 32 + p % 16 / 4 * 8;
    const float s = __bfloat162float(scales[n * (K / group) + k / group]);
    const uint32_t w = codes[i];
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float lo = (float)((int)((w >> (4 * j)) & 15) - 8) * s, hi = (float)((int)((w >> (4 * j + 16)) & 15) - 8) * s;
      const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
      o[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(out + n * K + k) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

bool bad_shape(int N, int K, int group) {
  return N < 1 || K < 128 || K % 128 || (group != 32 && group != 64 && group != 128);
}

int smem_of(int T, int units, bool whole, int nt) {
  return kWarps * kStages * blocks_of(nt) * 1024 + T * x_pitch_of(units, blocks_of(nt)) * 2 +
         (whole ? 0 : 2 * kWarps * 16 * (nt * 8 + 1) * 4);
}

int tiles_of_x(int T) { return T <= 8 ? 1 : T <= 16 ? 2 : 4; }
int units_of(const W4Args& a) {
  const int bu = blocks_of(tiles_of_x(a.T)), all = (a.K / 128 + bu - 1) / bu;
  return (all + a.slices - 1) / a.slices;
}

// Slices of K: the fewest whose x fits an SM, or some more if that shares the work better, whose time
// is the units that the warp with most of them takes. Returns the CTAs of a slice.
int plan(W4Args& a, int sms) {
  const int nt = tiles_of_x(a.T), tiles = (a.N + 15) / 16;
  double best = 0;
  W4Args b = a;
  int ctas = 1, least = 1;
  for (b.slices = 1; b.slices <= 2 * least + 2; ++b.slices) {
    const int units = units_of(b);
    if (smem_of(a.T, units, true, nt) > kMaxSmem) {
      if (units == 1) break;
      least = b.slices + 1;
      continue;
    }
    const int n = std::min(tiles, std::max(1, sms / b.slices));
    b.per = tiles / n;
    b.more = tiles % n;
    b.whole = smem_of(a.T, units, false, nt) > kMaxSmem;
    const long most = b.per + (b.more > 0);
    const double cost = (b.whole ? (most + kWarps - 1) / kWarps * units : (most * units + kWarps - 1) / kWarps) +
                        (b.slices > least ? kSliceCost * (b.slices - least) : 0.) + (b.slices > 1 ? 1. : 0.);
    if (best == 0 || cost < best) {
      best = cost;
      a = b;
      ctas = n;
    }
    if (units == 1) break;
  }
  return best == 0 ? 0 : ctas;
}

template <int NT, int GW, bool GLU>
int run(const W4Args& a, int ctas, cudaStream_t st) {
  const int smem = smem_of(a.T, units_of(a), a.whole, NT);
  static std::atomic<bool> raised[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return kErrBadArgsHost;
  if (!raised[dev].load()) {
    if (cudaFuncSetAttribute(stream_kernel<NT, GW, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) !=
        cudaSuccess)
      return kErrBadArgsHost;
    raised[dev].store(true);
  }
  count_launch();
  if (launch_early(stream_kernel<NT, GW, GLU>, dim3(ctas, a.slices), kThreads, smem, st, 1, a) != cudaSuccess)
    return kErrBadArgsHost;
  if (a.slices == 1) return 0;
  count_launch();
  const long outputs = (long)a.T * (GLU ? a.N / 2 : a.N);
  return launch_early(slices_kernel<GLU>, dim3((unsigned)((outputs + 255) / 256)), 256, 0, st, 1, a) == cudaSuccess
             ? 0
             : kErrBadArgsHost;
}
template <int NT>
int run_group(const W4Args& a, int group, bool glu, int ctas, cudaStream_t st) {
  if (group == 32) return glu ? run<NT, 1, true>(a, ctas, st) : run<NT, 1, false>(a, ctas, st);
  if (group == 64) return glu ? run<NT, 2, true>(a, ctas, st) : run<NT, 2, false>(a, ctas, st);
  return glu ? run<NT, 4, true>(a, ctas, st) : run<NT, 4, false>(a, ctas, st);
}

}  // namespace

long linear_w4_work(int T, int N, int K, int glu, int sms) {
  if (T < 1 || T > 64 || bad_shape(N, K, 32)) return 0;
  const long wide = (N + 15) / 16 * 16L;
  if (T > kFew) {
    const int slices = wide_slices(T, N, K, sms);
    return slices > 1 || glu ? slices * T * wide : 0;
  }
  W4Args a{};
  a.T = T, a.N = N, a.K = K;
  return plan(a, sms) == 0 || a.slices == 1 ? 0 : (long)a.slices * T * wide;
}

int launch_linear_w4(const void* x, long x_tok, const void* codes, const void* scales, const void* residual, long r_tok,
                     void* out, int T, int N, int K, int group, int glu, int sms, float* work, int* err,
                     cudaStream_t st) {
  if (bad_shape(N, K, group) || T > 64 || (glu && N % (2 * kGlu))) return kErrBadArgsHost;
  if (T < 1) return 0;
  W4Args a{};
  a.x = (const __nv_bfloat16*)x, a.x_tok = x_tok;
  a.codes = (const uint32_t*)codes, a.scales = (const __nv_bfloat16*)scales;
  a.residual = (const __nv_bfloat16*)residual, a.r_tok = r_tok;
  a.out = (__nv_bfloat16*)out, a.parts = work;
  a.T = T, a.N = N, a.K = K;
  if (T > kFew) {
    a.slices = wide_slices(T, N, K, sms);
    return launch_wide(a, group, glu, err, st);
  }
  const int ctas = plan(a, sms);
  if (ctas == 0) return kErrBadArgsHost;
  switch (tiles_of_x(T)) {
    case 1: return run_group<1>(a, group, glu, ctas, st);
    case 2: return run_group<2>(a, group, glu, ctas, st);
    default: return run_group<4>(a, group, glu, ctas, st);
  }
}

int launch_dequant_w4(const void* codes, const void* scales, void* out, int N, int K, int group, cudaStream_t st) {
  if (bad_shape(N, K, group)) return kErrBadArgsHost;
  const long words = (long)N * (K / 8);
  const long grid = (words + 255) / 256;
  count_launch();
  dequant_kernel<<<(unsigned)(grid < 148 * 16 ? grid : 148 * 16), 256, 0, st>>>(
      (const uint32_t*)codes, (const __nv_bfloat16*)scales, (__nv_bfloat16*)out, words, K, group);
  return cudaGetLastError() == cudaSuccess ? 0 : kErrBadArgsHost;
}

}  // namespace mxk
