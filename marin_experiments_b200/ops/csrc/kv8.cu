// Paged KV cache in 8 bits: append of new keys and values, and attention over the cache.
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

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Largest finite magnitude of 8 bf16 values; `bad` if one is not finite.
__device__ __forceinline__ float amax8(const uint4& u, bool& bad) {
  float a = 0.f;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __uint_as_float((w[i] << 16) & 0x7fffffffu), hi = __uint_as_float(w[i] & 0x7fff0000u);
    const bool lo_in = lo < INFINITY, hi_in = hi < INFINITY;
    a = fmaxf(a, lo_in ? lo : 0.f);
    a = fmaxf(a, hi_in ? hi : 0.f);
    bad |= !(lo_in && hi_in);
  }
  return a;
}

__device__ __forceinline__ float or_nan(float x) { return fabsf(x) < INFINITY ? x : NAN; }

// 8 bf16 values times inv, as 8 codes.
__device__ __forceinline__ uint2 codes8(const uint4& u, float inv) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w}, c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    f.x = or_nan(__uint_as_float(w[i] << 16)) * inv;
    f.y = or_nan(__uint_as_float(w[i] & 0xffff0000u)) * inv;
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
constexpr int kAppendThreads = 256;
constexpr int kMaxPage = 128;

template <int HD>
__global__ void __launch_bounds__(kAppendThreads)
    append_kernel(Kv8Cache c, const __nv_bfloat16* __restrict__ k_new, const __nv_bfloat16* __restrict__ v_new,
                  long k_tok, long v_tok, const int* __restrict__ slots, int rows, int window) {
  constexpr int LPT = HD / 8;                        // lanes a token (8 values each)
  constexpr int kHeld = kMaxPage * HD / 8 / kAppendThreads;  // 16-byte pieces a thread holds of a full run
  __shared__ float sh_max[kAppendThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y;
  const bool is_v = blockIdx.z;
  const __nv_bfloat16* src = (is_v ? v_new : k_new) + (long)head * HD;
  const long tok = is_v ? v_tok : k_tok;
  uint8_t* cache = (uint8_t*)(is_v ? c.v : c.k);
  float* scales = is_v ? c.v_scale : c.k_scale;
  const int r0 = blockIdx.x * window, row = r0 + lane;
  const int limit = c.pages * c.page;  // below 2^31 by the host's check
  // runs that start in this window
  int slot = -1, prev = -2;
  if (lane < window && row < rows) {
    slot = slots[row];
    if (row > 0) prev = slots[row - 1];
  }
  const bool first = slot >= 0 && slot < limit && (slot % c.page == 0 || prev != slot - 1);
  const uint32_t runs = __ballot_sync(0xffffffffu, first);
  const bool together = __popc(runs) <= 2;
  int index = 0;
  for (uint32_t left = runs; left; left &= left - 1, ++index) {
    if (!together && (index % (kAppendThreads / 32)) != warp) continue;
    const int l = __ffs(left) - 1;
    const int s0 = __shfl_sync(0xffffffffu, slot, l);
    const int page = s0 / c.page, off = s0 % c.page, r = r0 + l;
    // length of the run: to the end of the page, the rows or the sequence of slots
    const int most = min(c.page - off, rows - r);
    int n = 0;
    for (int b = 0; b < most; b += 32) {
      const bool in = b + lane < most && slots[r + b + lane] == s0 + b + lane;
      const uint32_t m = __ballot_sync(0xffffffffu, in);
      n += m == 0xffffffffu ? 32 : __ffs(~m) - 1;
      if (m != 0xffffffffu) break;
    }
    const long base = ((long)page * c.hkv + head) * c.page * HD;
    float* sp = scales + (long)page * c.hkv + head;
    const float was = off == 0 ? 0.f : *sp, old = fabsf(was);
    const int step = together ? kAppendThreads : 32, me = together ? tid : lane;
    float amax = 0.f;
    bool bad = false;
    uint4 held[kHeld];
    if (together) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int p = me + i * kAppendThreads;
        held[i] = p < n * LPT ? *reinterpret_cast<const uint4*>(src + (r + p / LPT) * tok + (p % LPT) * 8)
                              : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kHeld; ++i) amax = fmaxf(amax, amax8(held[i], bad));
      amax = warp_max(amax);
      if (lane == 0) sh_max[warp] = amax;
      bad = __syncthreads_or(bad);  // `together` is the same for the whole CTA
#pragma unroll
      for (int w = 0; w < kAppendThreads / 32; ++w) amax = fmaxf(amax, sh_max[w]);
      __syncthreads();
    } else {
      for (int p = me; p < n * LPT; p += 32)
        amax = fmaxf(amax, amax8(*reinterpret_cast<const uint4*>(src + (r + p / LPT) * tok + (p % LPT) * 8), bad));
      amax = warp_max(amax);
      bad = __any_sync(0xffffffffu, bad);
    }
    const int need = need_exponent(amax);
    const float now = fmaxf(exp2_int(need), old);
    const float inv = 1.f / now;  // exact: a power of two
    if (old > 0.f && now > old) {
      uint2* older = reinterpret_cast<uint2*>(cache + base);
      for (int p = me; p < off * LPT; p += step) older[p] = rescale8(older[p], old * inv);
    }
    uint2* dst = reinterpret_cast<uint2*>(cache + base) + (long)off * LPT;
    if (together) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int p = me + i * kAppendThreads;
        if (p < n * LPT) dst[p] = codes8(held[i], inv);
      }
    } else {
      for (int p = me; p < n * LPT; p += 32)
        dst[p] = codes8(*reinterpret_cast<const uint4*>(src + (r + p / LPT) * tok + (p % LPT) * 8), inv);
    }
    // every thread has read `was` before the barrier above
    if (me == 0) *sp = is_v && (bad || was < 0.f) ? -now : now;
  }
}

}  // namespace

int launch_kv8_append(const Kv8Cache& c, const void* k, const void* v, long k_tok, long v_tok, const int* slots,
                      int rows, cudaStream_t st) {
  if (rows < 1) return 0;
  if (c.page < 1 || c.page > kMaxPage) return kErrBadArgsHost;
  const int window = rows <= 2048 ? 8 : 32;
  dim3 grid((rows + window - 1) / window, c.hkv, 2);
  count_launch();
  if (c.hd == 64)
    append_kernel<64><<<grid, kAppendThreads, 0, st>>>(c, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_tok, v_tok,
                                                       slots, rows, window);
  else if (c.hd == 128)
    append_kernel<128><<<grid, kAppendThreads, 0, st>>>(c, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_tok,
                                                        v_tok, slots, rows, window);
  else
    return kErrBadArgsHost;
  return cudaGetLastError() == cudaSuccess ? 0 : kErrBadArgsHost;
}

}  // namespace mxk
