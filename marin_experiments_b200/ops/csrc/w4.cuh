// What the kernels of 4-bit weights share: their arguments, the conversion of codes, and the results.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pdl.cuh"

namespace mxk {

struct W4Args {
  const __nv_bfloat16* x;
  long x_tok;
  const uint32_t* codes;
  const __nv_bfloat16* scales;
  const __nv_bfloat16* residual;
  long r_tok;
  __nv_bfloat16* out;
  int T, N, K;
  // blockIdx.y is the slice of K. The CTAs of a slice take `per` tiles each, the first `more` one more;
  // `whole`: their warps take whole tiles.
  int slices, per, more, whole;
  float* parts;  // [slices][T][N rounded up to 16], where there are several slices
};

namespace {

constexpr int kGlu = 128;  // rows of a gate (or up) block

// (2 j, 2 j + 1) of a word, as bf16 codes. The mask and the exponent go in by one lop3; the compiler
// makes two of the expression.
__device__ __forceinline__ uint32_t pair_of(uint32_t w, int j, uint32_t magic, uint32_t bias) {
  uint32_t u, d;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(u) : "r"(w >> (4 * j)), "r"(magic));
  asm("sub.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(u), "r"(bias));
  return d;
}

// One output of a tile's row r (with GLU a unit, whose gate is y), or this slice's part of it.
template <bool GLU>
__device__ __forceinline__ void store(const W4Args& a, int slice, int tile, int r, int tok, float y, float up) {
  if (a.slices > 1) {
    float* p = a.parts + ((long)slice * a.T + tok) * ((a.N + 15) / 16 * 16L) + tile * 16 + r;
    p[0] = y;
    if (GLU) p[8] = up;
    return;
  }
  const int cols = GLU ? a.N / 2 : a.N, n = tile * (GLU ? 8 : 16) + r;
  if (n >= cols) return;
  if (GLU) y = y / (1.f + expf(-y)) * up;
  if (a.residual) y += __bfloat162float(a.residual[(long)tok * a.r_tok + n]);
  a.out[(long)tok * cols + n] = __float2bfloat16(y);
}

// The result from the slices' parts, in their order.
template <bool GLU>
__global__ void __launch_bounds__(256) slices_kernel(const __grid_constant__ W4Args a) {
  const int cols = GLU ? a.N / 2 : a.N;
  const long wide = (a.N + 15) / 16 * 16L, i = blockIdx.x * 256L + threadIdx.x;
  wait_for_previous();
  let_next_start();
  if (i >= (long)a.T * cols) return;
  const int tok = (int)(i / cols), n = (int)(i % cols);
  const float* p = a.parts + tok * wide + (GLU ? n / 8 * 16 + n % 8 : n);
  float y = 0.f, up = 0.f;
  for (int s = 0; s < a.slices; ++s, p += a.T * wide) {
    y += p[0];
    if (GLU) up += p[8];
  }
  if (GLU) y = y / (1.f + expf(-y)) * up;
  if (a.residual) y += __bfloat162float(a.residual[(long)tok * a.r_tok + n]);
  a.out[i] = __float2bfloat16(y);
}

}  // namespace

// Products of 33 to 64 rows of x (w4_wide.cu): CTAs' slices of K for these sizes, and the launch.
int wide_slices(int T, int N, int K, int sms);
int launch_wide(const W4Args& a, int group, bool glu, int* err, cudaStream_t st);

}  // namespace mxk
