// 4-bit products of 33 to 64 rows on the tcgen05 tensor cores.
//
// A CTA takes 128 rows of W and a slice of K. Eight warps turn the words into bf16 codes (exact, no
// scale) and write them as the K-major 128-byte-swizzled A operand; x comes by TMA as B; one thread
// issues the MMAs. Each scale group of a stage (128 values of K) has accumulator columns of its own in
// TMEM, and four warps, a row of W a thread, add them to fp32 registers times the group's scale: as
// exact as the kernel for fewer rows, where a scale folded into bf16 operands would round each weight.
//
// What bounds it: the steps of a stage, each a wait of a warp: codes written, a fence, products issued,
// sums read, about 0.45 us with four stages in flight. Without the products, the stores, the loads or the
// sums it is 2 to 13 % faster, without all of them 30 %. More warps for the codes (16: 33 us where 8 take
// 22), two issuing warps, stages of 256 values and a fifth stage were no faster. One thread found by
// elect.sync with descriptors built once issues 20 % faster than lane 0 with descriptors built each time.
//
// The kernel for fewer rows (mma.sync) against this one, B200, device time in us (24576 with SwiGLU):
//   rows, N x K, group      mma.sync  this      rows, N x K, group      mma.sync  this
//   32, 4096 x 4096, 128        11.3  10.5      33, 4096 x 12288, 32        30.0  20.9
//   32, 24576 x 4096, 128       33.7    44      64, 4096 x 12288, 128       36.8  22.4
//   32, 4096 x 12288, 32        20.3    21      64, 24576 x 4096, 64        76.6  50.9
// so up to 32 rows stay there: what this one gives at small N (8 %) is less than what it costs at large (30 %).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "kernels.h"
#include "pdl.cuh"
#include "sm100_primitives.cuh"
#include "w4.cuh"

namespace mxk {

bool make_tmap_bf16_2d(CUtensorMap* m, const void* ptr, int64_t inner, int64_t outer, int64_t ld, int box_inner,
                       int box_outer);

namespace {

constexpr int kRowsW = 128;              // rows of W of a CTA: M of the MMA
constexpr int kStages = 4;
constexpr int kCodeWarps = 8, kSumWarps = 4;
constexpr int kCodes0 = 2, kSums0 = kCodes0 + kCodeWarps;
constexpr int kAhead = 4;                // stages whose words a thread loads ahead
constexpr int kThreads = 32 * (kSums0 + kSumWarps);
constexpr int kABytes = kRowsW * 256;    // two tiles of 64 values of K
constexpr int kErrX = 61, kErrCodes = 62, kErrMma = 63, kErrSums = 64;

__host__ __device__ constexpr int stage_bytes(int n) { return kABytes + n * 256; }
constexpr int kAccCols = 64;             // of one scale group's accumulator
// Accumulators of a stage, used while the next fill.
__host__ __device__ constexpr int slots(int gw) { return 4 * (4 / gw) * kAccCols <= 512 ? 4 : 2; }
__host__ __device__ constexpr int tmem_cols(int gw) { return slots(gw) * (4 / gw) * kAccCols; }  // 256 or 512

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// a += x f in two sums by one instruction.
__device__ __forceinline__ void fma2(float& a0, float& a1, float x0, float x1, float f) {
  asm("{\n\t.reg .b64 a, x, g;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 x, {%2, %3};\n\tmov.b64 g, {%4, %4};\n\t"
      "fma.rn.f32x2 a, x, g, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(x0), "f"(x1), "f"(f));
}

// The scales of a row in a stage.
template <int GW>
struct RowScales;
template <>
struct RowScales<4> {
  uint16_t v;
  __device__ __forceinline__ float at(int) const { return __uint_as_float((uint32_t)v << 16); }
};
template <>
struct RowScales<2> {
  uint32_t v;
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i ? v & 0xffff0000u : v << 16); }
};
template <>
struct RowScales<1> {
  uint2 v;
  __device__ __forceinline__ float at(int i) const {
    const uint32_t w = i < 2 ? v.x : v.y;
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
};

// N: columns of the product, rows of x rounded up. GW: words of a lane in one scale group (group / 32).
template <int N, int GW, bool GLU>
__global__ void __launch_bounds__(kThreads, 1)
    wide_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ W4Args a, int* err) {
  constexpr int G = 4 / GW;  // scale groups of a stage
  constexpr int kSlots = slots(GW);
  constexpr uint32_t kCols = tmem_cols(GW);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);  // a cast of the address would make generic stores
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], sum_full[kSlots], sum_empty[kSlots], drain;
  __shared__ uint32_t tmem_slot;
  __shared__ int aborted;
  volatile int* abort_flag = &aborted;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int blocks = a.K / 128, slice = blockIdx.y, row0 = blockIdx.x * kRowsW;
  const int b0 = (int)((long)blocks * slice / a.slices), n_stages = (int)((long)blocks * (slice + 1) / a.slices) - b0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], kCodeWarps + 1);
      mbar_init(&empty[s], 1);
    }
    for (int d = 0; d < kSlots; ++d) {
      mbar_init(&sum_full[d], 1);
      mbar_init(&sum_empty[d], kSumWarps);
    }
    mbar_init(&drain, 1);
    fence_barrier_init();
    prefetch_tmap(&tm_x);
    aborted = 0;
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  wait_for_previous();
  let_next_start();

  if (warp == 0) {  // x
    if (lane == 0) {
      bool ok = true;
      int it = 0;
      for (; it < n_stages; ++it) {
        const int s = it % kStages;
        ok = mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, err, kErrX, abort_flag);
        if (!ok) break;
        mbar_arrive_expect_tx(&full[s], N * 256);
        uint8_t* dst = smem + s * stage_bytes(N) + kABytes;
        tma_load_2d(&tm_x, &full[s], dst, (b0 + it) * 128, 0);
        tma_load_2d(&tm_x, &full[s], dst + N * 128, (b0 + it) * 128 + 64, 0);
      }
      if (!ok) {  // bounded: the loads in flight have about 10 ms to land before the memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < (1ll << 24)) {}
      }
    }
  } else if (warp < kCodes0) {  // products
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_bf16(kRowsW, N, false, false);
      const uint64_t codes0 = make_sdesc(smem_u32(smem), 16, 1024), x0 = codes0 + kABytes / 16;
      bool ok = true, issued = false;
      for (int it = 0; it < n_stages; ++it) {
        const int s = it % kStages, d = it % kSlots;
        ok = mbar_wait(&sum_empty[d], ((it / kSlots) & 1) ^ 1, err, kErrMma, abort_flag) &&
             mbar_wait(&full[s], (it / kStages) & 1, err, kErrMma, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint64_t codes = codes0 + (uint32_t)(s * stage_bytes(N) / 16), x = x0 + (uint32_t)(s * stage_bytes(N) / 16);
        const uint32_t to = tmem + d * G * kAccCols;
#pragma unroll
        for (int k = 0; k < 8; ++k)  // 16 values of K
          umma_bf16(to + k / (2 * GW) * kAccCols, codes + ((k / 4) * (kRowsW * 128) + (k % 4) * 32) / 16,
                    x + ((k / 4) * (N * 128) + (k % 4) * 32) / 16, idesc, k % (2 * GW) != 0 ? 1u : 0u);
        issued = true;
        umma_commit(&empty[s]);
        umma_commit(&sum_full[d]);
      }
      if (!ok && issued) {  // bounded: every product has ended before TMEM is freed
        umma_commit(&drain);
        const long long t0 = clock64();
        while (!mbar_try_wait(&drain, 0) && clock64() - t0 < (1ll << 26)) {}
      }
    }
  } else if (warp < kSums0) {  // codes
    // A thread has a quarter (16 bytes of words) of a block in rows r and r + 64. Rows of eight lanes
    // differ in bit 2, so that their swizzled 16-byte columns are all of the 128-byte row.
    const int id = threadIdx.x - 32 * kCodes0, t = id & 3, q = id >> 2;
    const int r = (q & ~7) | (q & 1) << 2 | (q >> 1 & 3);
    const uint32_t* p[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) p[i] = a.codes + (long)min(row0 + r + 64 * i, a.N - 1) * (a.K / 8) + (long)b0 * 16 + 4 * t;
    uint4 w[kAhead][2];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[k][i] = k < n_stages ? __ldg(reinterpret_cast<const uint4*>(p[i] + k * 16)) : make_uint4(0, 0, 0, 0);
    uint32_t magic = 0x43004300u, bias = 0x43084308u;
    asm volatile("" : "+r"(magic), "+r"(bias));
    // Column 4 (k & 1) + t of the row's eight; rows 64 apart have the same swizzle.
    const uint32_t mine_at = smem_u32(smem) + r * 128 + ((t ^ (r & 7)) << 4);
    bool mine = true;
    for (int first = 0; first < n_stages && mine; first += kAhead) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {  // unrolled: moving a register waits for the load that fills it
        const int it = first + j, s = it % kStages;
        if (it >= n_stages) break;
        mine = lane != 0 || mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, err, kErrCodes, abort_flag);
        mine = __all_sync(0xffffffffu, mine);
        if (!mine) break;
        const uint32_t dst = mine_at + s * stage_bytes(N);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t words[4] = {w[j][i].x, w[j][i].y, w[j][i].z, w[j][i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // values 32 k + 8 t .. + 7
            sts128((k & 1 ? dst ^ 64 : dst) + (k >> 1) * (kRowsW * 128) + i * 64 * 128,
                   pair_of(words[k], 0, magic, bias), pair_of(words[k], 1, magic, bias),
                   pair_of(words[k], 2, magic, bias), pair_of(words[k], 3, magic, bias));
          }
          if (it + kAhead < n_stages) w[j][i] = __ldg(reinterpret_cast<const uint4*>(p[i] + (it + kAhead) * 16));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
      }
    }
  } else {  // sums: one row of W a thread
    const int quad = warp & 3;  // the lanes of TMEM that this warp reaches
    const int row = row0 + quad * 32 + lane;
    const RowScales<GW>* sp =
        reinterpret_cast<const RowScales<GW>*>(a.scales) + (long)min(row, a.N - 1) * blocks + b0;
    float acc[N];
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = 0.f;
    RowScales<GW> next = sp[0];
    bool ok = true;
    for (int it = 0; it < n_stages; ++it) {
      const int d = it % kSlots;
      const RowScales<GW> sc = next;
      if (it + 1 < n_stages) next = sp[it + 1];
      ok = lane != 0 || mbar_wait(&sum_full[d], (it / kSlots) & 1, err, kErrSums, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const float f = sc.at(gi);
        const uint32_t at = tmem + ((uint32_t)(quad * 32) << 16) + (d * G + gi) * kAccCols;
#pragma unroll
        for (int c = 0; c < N; c += 16) {
          float v[16];
          tmem_ld16(at + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int n = 0; n < 16; n += 2) fma2(acc[c + n], acc[c + n + 1], v[n], v[n + 1], f);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sum_empty[d]);
    }
    if (row < a.N) {
      if (a.slices > 1 || GLU) {
        int at = row;
        if (GLU) {  // tiles of 8 gate rows and the 8 up rows of the same units
          const int u = row / (2 * kGlu) * kGlu + row % kGlu;
          at = u / 8 * 16 + u % 8 + (row / kGlu % 2) * 8;
        }
        float* o = a.parts + (long)slice * a.T * ((a.N + 15) / 16 * 16L) + at;
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (n < a.T) o[n * ((a.N + 15) / 16 * 16L)] = acc[n];
      } else {
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (n < a.T) {
            float y = acc[n];
            if (a.residual) y += __bfloat162float(a.residual[(long)n * a.r_tok + row]);
            a.out[(long)n * a.N + row] = __float2bfloat16(y);
          }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

template <int N, int GW, bool GLU>
int run(const W4Args& a, int* err, cudaStream_t st) {
  constexpr int kSmem = kStages * stage_bytes(N) + 1024;
  static std::atomic<bool> raised[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return kErrBadArgsHost;
  if (!raised[dev].load()) {
    if (cudaFuncSetAttribute(wide_kernel<N, GW, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return kErrBadArgsHost;
    raised[dev].store(true);
  }
  CUtensorMap tm;
  if (!make_tmap_bf16_2d(&tm, a.x, a.K, a.T, a.x_tok, 64, N)) return kErrBadArgsHost;
  count_launch();
  if (launch_early(wide_kernel<N, GW, GLU>, dim3((a.N + kRowsW - 1) / kRowsW, a.slices), kThreads, kSmem, st, 1, tm, a,
                   err) != cudaSuccess)
    return kErrBadArgsHost;
  if (a.slices == 1 && !GLU) return 0;
  count_launch();
  const long outputs = (long)a.T * (GLU ? a.N / 2 : a.N);
  return launch_early(slices_kernel<GLU>, dim3((unsigned)((outputs + 255) / 256)), 256, 0, st, 1, a) == cudaSuccess
             ? 0
             : kErrBadArgsHost;
}
template <int N>
int run_group(const W4Args& a, int group, bool glu, int* err, cudaStream_t st) {
  if (group == 32) return glu ? run<N, 1, true>(a, err, st) : run<N, 1, false>(a, err, st);
  if (group == 64) return glu ? run<N, 2, true>(a, err, st) : run<N, 2, false>(a, err, st);
  return glu ? run<N, 4, true>(a, err, st) : run<N, 4, false>(a, err, st);
}

}  // namespace

// The slices for which the rounds of CTAs end first: a CTA's time in stages, kStart for its start and
// end, and what the slices' parts cost.
int wide_slices(int T, int N, int K, int sms) {
  const int blocks = K / 128, tiles = (N + kRowsW - 1) / kRowsW;
  constexpr double kStart = 8., kStageUs = 0.35;
  double best = 0;
  int slices = 1;
  for (int s = 1; s <= blocks && s <= 32; ++s) {
    const long rounds = ((long)tiles * s + sms - 1) / sms;
    double cost = rounds * ((blocks + s - 1) / s + kStart);
    if (s > 1) cost += kStart + (double)s * T * N * 8 / 4e6 / kStageUs;  // written and read at 4 TB/s
    if (s == 1 || cost < best) {
      best = cost;
      slices = s;
    }
  }
  return slices;
}

int launch_wide(const W4Args& a, int group, bool glu, int* err, cudaStream_t st) {
  if (err == nullptr || (glu && a.parts == nullptr)) return kErrBadArgsHost;
  if (a.T <= 48) return run_group<48>(a, group, glu, err, st);
  return run_group<64>(a, group, glu, err, st);
}

}  // namespace mxk
