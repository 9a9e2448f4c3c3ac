// Products with 4-bit weights: y[t, n] = sum_k x[t, k] * code[n, k] * scale[n, k / group], for the few
// rows (1 to 64) of a decode step, with the residual added or the SwiGLU applied before the one
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
// What bounds it: N * K / 2 bytes of weights against 2 * T * N * K operations, so memory for T up to
// 64; at a few MB a matrix the launch, one round trip to memory and the sum over the warps count as
// much. The 8 warps of a CTA share K (each takes every eighth block of 128, so a row is read in
// 512-byte runs) and join their sums in shared memory in a fixed order.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kernels.h"

namespace mxk {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kGlu = 128;  // rows of a gate (or up) block

__device__ __forceinline__ uint32_t pair_of(uint32_t w, int j) {
  const uint32_t u = ((w >> (4 * j)) & 0x000f000fu) | 0x43004300u;
  __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&u);
  h = __hsub2(h, __nv_bfloat162(__float2bfloat16(136.f), __float2bfloat16(136.f)));
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_once(const uint32_t* p) {  // weights: no second use
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

struct W4Args {
  const __nv_bfloat16* x;
  long x_tok;
  const uint32_t* codes;
  const __nv_bfloat16* scales;
  const __nv_bfloat16* residual;
  long r_tok;
  __nv_bfloat16* out;
  int T, N, K;
};

// NT: tiles of 8 rows of x. GW: words of a lane in one group (group / 32). A CTA makes 16 rows of W;
// with GLU these are 8 gate rows and the 8 up rows of the same units.
template <int NT, int GW, bool GLU>
__global__ void __launch_bounds__(kThreads) linear_kernel(W4Args a) {
  __shared__ float red[kWarps][16][NT * 8 + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int tile = blockIdx.x;
  int row[2];  // of W
  if (GLU) {
    const int unit = tile * 8 + g;
    row[0] = unit / kGlu * 2 * kGlu + unit % kGlu;
    row[1] = row[0] + kGlu;
  } else {
    row[0] = tile * 16 + g;
    row[1] = row[0] + 8;
  }
  const int blocks = a.K / 128, groups = a.K / (GW * 32);
  const uint32_t* wp[2];
  const __nv_bfloat16* sp[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = min(row[i], a.N - 1);  // rows past N repeat the last and are not stored
    wp[i] = a.codes + (long)r * (a.K / 8) + 4 * t;
    sp[i] = a.scales + (long)r * groups;
  }
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int z = 0; z < 4; ++z) acc[n][z] = 0.f;

#pragma unroll 2
  for (int b = warp; b < blocks; b += kWarps) {
    uint4 u[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) u[i] = load_once(wp[i] + (long)b * 16);
    const uint32_t w0[4] = {u[0].x, u[0].y, u[0].z, u[0].w}, w1[4] = {u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
    for (int gi = 0; gi < 4 / GW; ++gi) {
      const float s0 = __bfloat162float(sp[0][b * (4 / GW) + gi]), s1 = __bfloat162float(sp[1][b * (4 / GW) + gi]);
      float part[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int z = 0; z < 4; ++z) part[n][z] = 0.f;
#pragma unroll
      for (int i = gi * GW; i < (gi + 1) * GW; ++i) {
        uint32_t p0[4], p1[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p0[j] = pair_of(w0[i], j);
          p1[j] = pair_of(w1[i], j);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int tok = n * 8 + g;
          uint4 xv = make_uint4(0, 0, 0, 0);
          if (tok < a.T) xv = *reinterpret_cast<const uint4*>(a.x + tok * a.x_tok + b * 128 + i * 32 + t * 8);
          mma(part[n], p0[0], p1[0], p0[1], p1[1], xv.x, xv.y);
          mma(part[n], p0[2], p1[2], p0[3], p1[3], xv.z, xv.w);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[n][0] += part[n][0] * s0;
        acc[n][1] += part[n][1] * s0;
        acc[n][2] += part[n][2] * s1;
        acc[n][3] += part[n][3] * s1;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int z = 0; z < 4; ++z) red[warp][g + 8 * (z >> 1)][n * 8 + 2 * t + (z & 1)] = acc[n][z];
  __syncthreads();
  if (GLU) {
    const int cols = a.N / 2;
    for (int i = tid; i < 8 * NT * 8; i += kThreads) {
      const int r = i % 8, tok = i / 8;
      if (tok >= a.T || tile * 8 + r >= cols) continue;
      float gate = 0.f, up = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        gate += red[w][r][tok];
        up += red[w][r + 8][tok];
      }
      a.out[(long)tok * cols + tile * 8 + r] = __float2bfloat16(gate / (1.f + expf(-gate)) * up);
    }
  } else {
    for (int i = tid; i < 16 * NT * 8; i += kThreads) {
      const int r = i % 16, tok = i / 16, n = tile * 16 + r;
      if (tok >= a.T || n >= a.N) continue;
      float y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) y += red[w][r][tok];
      if (a.residual) y += __bfloat162float(a.residual[(long)tok * a.r_tok + n]);
      a.out[(long)tok * a.N + n] = __float2bfloat16(y);
    }
  }
}

template <int NT, int GW>
void run(const W4Args& a, bool glu, cudaStream_t st) {
  count_launch();
  if (glu) linear_kernel<NT, GW, true><<<a.N / 16, kThreads, 0, st>>>(a);
  else linear_kernel<NT, GW, false><<<(a.N + 15) / 16, kThreads, 0, st>>>(a);
}
template <int NT>
void run_group(const W4Args& a, int group, bool glu, cudaStream_t st) {
  if (group == 32) run<NT, 1>(a, glu, st);
  else if (group == 64) run<NT, 2>(a, glu, st);
  else run<NT, 4>(a, glu, st);
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

}  // namespace

int launch_linear_w4(const void* x, long x_tok, const void* codes, const void* scales, const void* residual, long r_tok,
                     void* out, int T, int N, int K, int group, int glu, cudaStream_t st) {
  if (bad_shape(N, K, group) || T > 64 || (glu && N % (2 * kGlu))) return kErrBadArgsHost;
  if (T < 1) return 0;
  const W4Args a{(const __nv_bfloat16*)x, x_tok, (const uint32_t*)codes, (const __nv_bfloat16*)scales,
                 (const __nv_bfloat16*)residual, r_tok, (__nv_bfloat16*)out, T, N, K};
  if (T <= 8) run_group<1>(a, group, glu, st);
  else if (T <= 16) run_group<2>(a, group, glu, st);
  else if (T <= 32) run_group<4>(a, group, glu, st);
  else run_group<8>(a, group, glu, st);
  return cudaGetLastError() == cudaSuccess ? 0 : kErrBadArgsHost;
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
