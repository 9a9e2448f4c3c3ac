// Paged KV cache in 8 bits: its format, and the append of new keys and values (kv8_attention.cu has the
// attention over it).
//
// A page holds `page` tokens of one kv head as e4m3 codes, [pages][hkv][page][hd], with one fp32
// scale for each page and head, keys and values apart. A value is code * scale. Scales are powers of
// two: the least 2^e with max|x| <= 448 * 2^e. e4m3 keeps 4 significant bits wherever a value lies in
// its 2^-6 .. 448 range, so a scale that is up to twice too large costs no precision, while a power
// of two makes x / scale exact (one rounding in all, to the nearest code, ties to even) and lets the
// scale of a page grow as tokens arrive: its older codes are multiplied by 2^-j, exact again but for
// those that become subnormal. Values that are not finite are stored as e4m3's NaN, and the sign of a
// page's v_scale says that it holds one: the attention converts values without a look for NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kernels.h"
#include "pdl.cuh"

namespace mxk {
namespace {

constexpr int kMinExp = -110, kMaxExp = 120;  // 2^e and 2^-e are both normal fp32 numbers

__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

// Least e in [kMinExp, kMaxExp] with amax <= 448 * 2^e = 0.875 * 2^(e + 9).
__device__ __forceinline__ int need_exponent(float amax) {
  if (!(amax > 0.f)) return kMinExp;
  int p;
  const float m = frexpf(amax, &p);
  const int e = m <= 0.875f ? p - 9 : p - 8;
  return min(kMaxExp, max(kMinExp, e));
}

// Largest magnitudes of the low and the high halves of 8 bf16 values, two 16-bit numbers (0x7f80 and
// above: not finite); `most` before.
__device__ __forceinline__ uint32_t amax8(const uint4& u, uint32_t most) {
  most = __vmaxu2(most, u.x & 0x7fff7fffu);
  most = __vmaxu2(most, u.y & 0x7fff7fffu);
  most = __vmaxu2(most, u.z & 0x7fff7fffu);
  return __vmaxu2(most, u.w & 0x7fff7fffu);
}
// The same of the finite ones alone.
__device__ __forceinline__ uint32_t finite8(uint4 u, uint32_t most) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
    if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0xffffu;
  }
  return amax8(make_uint4(w[0], w[1], w[2], w[3]), most);
}

__device__ __forceinline__ float or_nan(float x) { return fabsf(x) < INFINITY ? x : NAN; }

// 8 bf16 values times inv, as 8 codes. CHECK: what is not finite becomes NaN.
template <bool CHECK>
__device__ __forceinline__ uint2 codes8(const uint4& u, float inv) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w}, c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    if (CHECK) f = make_float2(or_nan(f.x), or_nan(f.y));
    f.x *= inv;
    f.y *= inv;
    c[i] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// 8 codes times a power of two <= 1, rounded to codes again.
__device__ __forceinline__ uint2 rescale8(uint2 u, float ratio) {
  uint32_t w[2] = {u.x, u.y}, o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((w[i] >> (16 * j)) & 0xffffu), __NV_E4M3);
      float2 f = __half22float2(__half2(h));
      f.x *= ratio;
      f.y *= ratio;
      r |= (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3) << (16 * j);
    }
    o[i] = r;
  }
  return make_uint2(o[0], o[1]);
}

// ------------------------------------------------------------------------------------- append
//
// Rows whose slots follow one another inside a page form a run, and a run is written by the threads
// that handle its first row, so a page's scale has one writer. A CTA (8 warps) takes a window of
// rows, one head, keys or values. Few runs start in a window of prompt tokens: the CTA takes each
// together, with the run's values in registers between the maximum and the rounding (one read). Many
// start in a window of decode tokens: each warp takes its own.
//
// What bounds it: in prompts the bytes, 2 in and 1 out a value; in decode two dependent loads. A run's
// values are loaded while its length is still looked for (they are masked when it is known).
constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kManyRows = 64;  // of a window: a prompt's

// Pages of 128 hold 8 pieces a thread: held to 3 CTAs an SM (16000 rows 24.3 -> 19.1 us then),
// the others to 4 (8000 rows in pages of 64 15 us then; 23 at one, where registers are not held back).
template <int HD, int PAGE>
__global__ void __launch_bounds__(kAppendThreads, PAGE == 128 ? 3 : 4)
    append_kernel(const __grid_constant__ Kv8Cache c, const __nv_bfloat16* __restrict__ k_new,
                  const __nv_bfloat16* __restrict__ v_new, long k_tok, long v_tok, const int* __restrict__ slots,
                  int rows, int window) {
  constexpr int LPT = HD / 8;  // 16-byte pieces of a row
  constexpr int kHeld = (PAGE * LPT + kAppendThreads - 1) / kAppendThreads;  // that a thread holds of a full run
  __shared__ uint32_t sh_max[kAppendWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // heads first: the CTAs at work read whole rows and write whole pages between them (15.8 -> 14.9 us)
  const int at = blockIdx.x / c.hkv, head = blockIdx.x - at * c.hkv;
  const bool is_v = blockIdx.y;
  const __nv_bfloat16* src = (is_v ? v_new : k_new) + (long)head * HD;
  const long tok = is_v ? v_tok : k_tok;
  uint8_t* cache = (uint8_t*)(is_v ? c.v : c.k);
  float* scales = is_v ? c.v_scale : c.k_scale;
  const int limit = c.pages * PAGE;  // below 2^31 by the host's check
  wait_for_previous();
  const int stop = (int)min((long)rows, (at + 1L) * window);
  // A prompt's rows come to L2 while their slots are looked at (8000 rows 14.9 -> 13.5 us; a decode step's
  // few are slower for it, 256 rows 3.75 -> 3.82).
  constexpr int kLines = HD / 64;
  if (window >= kManyRows)
    for (int p = tid; p < (stop - at * window) * kLines; p += kAppendThreads)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(src + (at * window + p / kLines) * tok + p % kLines * 64));
  int slot_ahead, prev_ahead;  // of this lane's row and the row before
  auto look = [&](int r0) {
    const int row = r0 + lane;
    slot_ahead = row < stop ? slots[row] : -1;
    prev_ahead = row < stop && row > 0 ? slots[row - 1] : -2;
  };
  look(at * window);
  for (int r0 = at * window; r0 < stop; r0 += 32) {
    // runs that start in these 32 rows
    const int slot = slot_ahead, prev = prev_ahead;
    look(r0 + 32);
    const bool first = slot >= 0 && slot < limit && (slot % PAGE == 0 || prev != slot - 1);
    const uint32_t runs = __ballot_sync(0xffffffffu, first);
    const bool together = __popc(runs) <= 2;
    int index = 0;
    for (uint32_t left = runs; left; left &= left - 1, ++index) {
      if (!together && (index % kAppendWarps) != warp) continue;
      const int l = __ffs(left) - 1;
      const int s0 = __shfl_sync(0xffffffffu, slot, l);
      const int page = s0 / PAGE, off = s0 % PAGE, r = r0 + l;
      const int most = min(PAGE - off, rows - r);  // rows that the run may have
      const long base = ((long)page * c.hkv + head) * PAGE * HD;
      float* sp = scales + (long)page * c.hkv + head;
      const float was = off == 0 ? 0.f : *sp, old = fabsf(was);
      auto piece = [&](int p) { return *reinterpret_cast<const uint4*>(src + (r + p / LPT) * tok + (p % LPT) * 8); };
      uint4 held[kHeld];
      if (together) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          const int p = tid + i * kAppendThreads;
          held[i] = p < most * LPT ? piece(p) : make_uint4(0, 0, 0, 0);
        }
      }
      int n = 0;  // rows that it has
      bool on = true;
#pragma unroll
      for (int b = 0; b < PAGE; b += 32) {
        const bool in = b + lane < most && slots[r + b + lane] == s0 + b + lane;
        const uint32_t m = __ballot_sync(0xffffffffu, in);
        if (on) n += m == 0xffffffffu ? 32 : __ffs(~m) - 1;
        on = on && m == 0xffffffffu;
      }
      const int step = together ? kAppendThreads : 32, me = together ? tid : lane;
      uint32_t big = 0;
      auto largest = [&](auto of) {  // over the run's threads
        uint32_t v = 0;
        if (together) {
#pragma unroll
          for (int i = 0; i < kHeld; ++i)
            if (tid + i * kAppendThreads < n * LPT) v = of(held[i], v);
        } else {
          for (int p = lane; p < n * LPT; p += 32) v = of(piece(p), v);
        }
        v = __reduce_max_sync(0xffffffffu, max(v & 0xffffu, v >> 16));
        if (together) {  // the same for the whole CTA
          if (lane == 0) sh_max[warp] = v;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < kAppendWarps; ++w) v = max(v, sh_max[w]);
          __syncthreads();
        }
        return v;
      };
      big = largest([](const uint4& u, uint32_t v) { return amax8(u, v); });
      const bool bad = big >= 0x7f80u;  // something is not finite
      if (bad) big = largest([](const uint4& u, uint32_t v) { return finite8(u, v); });
      const float now = fmaxf(exp2_int(need_exponent(__uint_as_float(big << 16))), old);
      const float inv = 1.f / now;  // exact: a power of two
      if (old > 0.f && now > old) {
        uint2* older = reinterpret_cast<uint2*>(cache + base);
        for (int p = me; p < off * LPT; p += step) older[p] = rescale8(older[p], old * inv);
      }
      uint2* dst = reinterpret_cast<uint2*>(cache + base) + (long)off * LPT;
      if (together) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          const int p = tid + i * kAppendThreads;
          if (p < n * LPT) dst[p] = bad ? codes8<true>(held[i], inv) : codes8<false>(held[i], inv);
        }
      } else {
        for (int p = lane; p < n * LPT; p += 32) dst[p] = codes8<true>(piece(p), inv);
        __syncwarp();
      }
      // every thread has read `was`: the maxima met in between
      if (me == 0) *sp = is_v && (bad || was < 0.f) ? -now : now;
    }
  }
}

template <int HD>
int launch_append(const Kv8Cache& c, const void* k, const void* v, long k_tok, long v_tok, const int* slots, int rows,
                  int window, cudaStream_t st) {
  const long ctas = ((long)rows + window - 1) / window * c.hkv;
  if (ctas > 0x7fffffffL) return kErrBadArgsHost;
  const dim3 grid((unsigned)ctas, 2);
  auto kernel = c.page == 32 ? append_kernel<HD, 32> : c.page == 64 ? append_kernel<HD, 64> : append_kernel<HD, 128>;
  count_launch();
  return launch_early(kernel, grid, kAppendThreads, 0, st, 1, c, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_tok,
                      v_tok, slots, rows, window) == cudaSuccess
             ? 0
             : kErrBadArgsHost;
}

}  // namespace

int launch_kv8_append(const Kv8Cache& c, const void* k, const void* v, long k_tok, long v_tok, const int* slots,
                      int rows, cudaStream_t st) {
  if (rows < 1) return 0;
  if (c.page != 32 && c.page != 64 && c.page != 128) return kErrBadArgsHost;
  // Few rows are a decode step's, whose runs of one row want a warp each; many are a prompt's, whose runs
  // want a CTA each and no CTA without one (us at windows of 8, 16, 32, 64; 8 kv heads of 128 dims: 256
  // runs of a row 3.7, 4.7, 7.3, 13; a prompt of 700 rows 4.5, 3.7, 3.4, 3.6; 1000 runs of a row 10.5, 10.0,
  // 10.3, 14; 8000 rows of prompts at 16, 32, 64, 128, before they were fetched ahead: 21, 15.9, 14.9,
  // 15.6).
  const int window = rows <= 256 ? 8 : rows <= 2048 ? 16 : kManyRows;
  if (c.hd == 64) return launch_append<64>(c, k, v, k_tok, v_tok, slots, rows, window, st);
  if (c.hd == 128) return launch_append<128>(c, k, v, k_tok, v_tok, slots, rows, window, st);
  return kErrBadArgsHost;
}

}  // namespace mxk
