// The 8-bit paged KV cache: quantised as it is written, read back as bf16.
//   codes int8 [pages, kv_heads, page, D] (K and V), scales f32 [pages, kv_heads]; value = code * scale
// A write puts tokens at positions len - n .. len - 1 of each sequence.  For each touched page and head:
//   a = max |x| over the call's tokens there;  s' = max(s, a / 127), with s = 0 if the call begins the page
//   s' below the smallest normal float becomes 0 (its tokens read as 0); a value that is not finite makes s' NaN
//   code = rint(x * (1 / s'));  older codes of the page become rint(code * (s / s'))
// Every step is one fp32 operation, so the result does not depend on the launch.
#pragma once

#include "common.cuh"

namespace gguf_b200 {

// Loads of what an earlier kernel of the same chain may have written: through the L2 (a line of the read-only path may be
// older than a programmatic launch's predecessor), and volatile, since the compiler moves an ordinary cached-load intrinsic
// across the wait for that predecessor.
__device__ __forceinline__ int32_t ld_cg(const int32_t* p) {
  int32_t v;
  asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cg(const float* p) {
  float v;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cg(const float2* p) {
  float2 v;
  asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cg(const float4* p) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld_cg64(const void* p) {
  uint2 v;
  asm volatile("ld.global.cg.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_cg128(const void* p) {
  uint4 v;
  asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

struct KvPages {
  const int32_t* table;  // [B, table_cols] page of each sequence's i-th stretch of `page` tokens
  int64_t pages;
  int table_cols, kv_heads, log2_page, D;
};

// Whether a table entry names a page of the cache; recorded where it does not.
__device__ __forceinline__ bool kv_page_ok(const KvPages& c, int entry) {
  if (entry >= 0 && entry < c.pages) return true;
  record_device_error(kSiteBadCachePage);
  return false;
}
// Page of stretch i of sequence b, or -1 (recorded) where the table or the page is out of range.
__device__ __forceinline__ int64_t kv_page(const KvPages& c, int b, int i) {
  int p = -1;
  if (i < c.table_cols) p = ld_cg(c.table + static_cast<int64_t>(b) * c.table_cols + i);
  return kv_page_ok(c, p) ? p : -1;
}

struct KvWriteArgs {
  KvPages c;
  const bf16* x[2];  // K and V: [B, R, kv_heads, D], strides in values
  int8_t* codes[2];
  float* scales[2];
  const int32_t *lens, *news;  // news may be null: R
  int64_t stride_b[2], stride_r[2];
  int R;
};

constexpr int kKvWriteThreads = 128;
constexpr int kKvWriteRegs = 8;  // 16-byte pieces of the call's tokens that a thread keeps between the two passes

// The four codes of x0..x3: adding 1.5 * 2^23 rounds the fp32 product to the nearest whole number
// (ties to even) and leaves its two's complement in the low byte.
__device__ __forceinline__ uint32_t kv_codes4(float x0, float x1, float x2, float x3, float inv) {
  constexpr float kMagic = 12582912.0f;
  const uint32_t u0 = __float_as_uint(__fadd_rn(__fmul_rn(x0, inv), kMagic));
  const uint32_t u1 = __float_as_uint(__fadd_rn(__fmul_rn(x1, inv), kMagic));
  const uint32_t u2 = __float_as_uint(__fadd_rn(__fmul_rn(x2, inv), kMagic));
  const uint32_t u3 = __float_as_uint(__fadd_rn(__fmul_rn(x3, inv), kMagic));
  return __byte_perm(__byte_perm(u0, u1, 0x0040), __byte_perm(u2, u3, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t kv_rescale4(uint32_t w, float ratio) {
  return kv_codes4(static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8)),
                   static_cast<float>(static_cast<int8_t>(w >> 16)), static_cast<float>(static_cast<int8_t>(w >> 24)),
                   ratio);
}
__device__ __forceinline__ uint32_t abs_max_bf16x2(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7FFF7FFFu); }

// One CTA per (touched page, head, K or V) of a sequence: blockIdx = (page of the call * 2 + which, head, sequence).
__global__ void __launch_bounds__(kKvWriteThreads) kv_write_kernel(const KvWriteArgs a) {
  __shared__ uint32_t red[kKvWriteThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, h = blockIdx.y, which = blockIdx.x & 1, tid = threadIdx.x;
  const int len = ld_cg(a.lens + b);
  const int n = min(a.news ? ld_cg(a.news + b) : a.R, min(a.R, len));
  const int first = len - n;
  const int lg = a.c.log2_page, i = (first >> lg) + (blockIdx.x >> 1);
  const int begin = i << lg;
  if (n <= 0 || begin >= len) return;
  const int64_t page = kv_page(a.c, b, i);
  if (page < 0) return;
  const int t0 = max(first, begin), t1 = min(len, begin + (1 << lg));
  const int per = a.c.D >> 3, pieces = (t1 - t0) * per;
  const bf16* x = a.x[which] + b * a.stride_b[which] + (t0 - first) * a.stride_r[which] + h * a.c.D;
  const int64_t rs = a.stride_r[which];
  const int64_t at = page * a.c.kv_heads + h;
  int8_t* codes = a.codes[which] + ((at << lg) * a.c.D);
  float* scale_p = a.scales[which] + at;

  uint4 keep[kKvWriteRegs];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < kKvWriteRegs; ++j) {
    const int p = tid + j * kKvWriteThreads;
    keep[j] = make_uint4(0, 0, 0, 0);
    if (p < pieces) keep[j] = ld_cg128(x + (p / per) * rs + (p % per) * 8);
  }
#pragma unroll
  for (int j = 0; j < kKvWriteRegs; ++j)
    m = abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(m, keep[j].x), keep[j].y), keep[j].z), keep[j].w);
  for (int p = tid + kKvWriteRegs * kKvWriteThreads; p < pieces; p += kKvWriteThreads) {
    const uint4 v = ld_cg128(x + (p / per) * rs + (p % per) * 8);
    m = abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(m, v.x), v.y), v.z), v.w);
  }
  m = max(m & 0xFFFFu, m >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
  const bool older = t0 > begin;
  const float was = older ? *scale_p : 0.f;
  __syncthreads();  // also: every thread has read the old scale
#pragma unroll
  for (int w = 0; w < kKvWriteThreads / 32; ++w) m = max(m, red[w]);
  const float amax = __uint_as_float(m << 16);
  float scale = __fdiv_rn(amax, 127.0f);
  if (!(was <= scale)) scale = was;  // was larger, or NaN
  if (m >= 0x7F80u) scale = __uint_as_float(0x7FC00000u);
  if (scale < 1.17549435e-38f) scale = 0.f;
  const float inv = scale > 0.f ? __fdiv_rn(1.0f, scale) : 0.f;
  if (tid == 0) *scale_p = scale;

  if (older && scale != was) {
    const float ratio = scale > 0.f ? __fdiv_rn(was, scale) : 0.f;
    const int old_pieces = (t0 - begin) * a.c.D >> 4;
    uint4* o = reinterpret_cast<uint4*>(codes);
    for (int p = tid; p < old_pieces; p += kKvWriteThreads) {
      uint4 v = o[p];
      v.x = kv_rescale4(v.x, ratio), v.y = kv_rescale4(v.y, ratio);
      v.z = kv_rescale4(v.z, ratio), v.w = kv_rescale4(v.w, ratio);
      o[p] = v;
    }
  }
  uint2* o = reinterpret_cast<uint2*>(codes + static_cast<int64_t>(t0 - begin) * a.c.D);
  auto put = [&](int p, uint4 v) {
    o[p] = make_uint2(kv_codes4(bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y), inv),
                      kv_codes4(bf16_lo(v.z), bf16_hi(v.z), bf16_lo(v.w), bf16_hi(v.w), inv));
  };
#pragma unroll
  for (int j = 0; j < kKvWriteRegs; ++j)
    if (tid + j * kKvWriteThreads < pieces) put(tid + j * kKvWriteThreads, keep[j]);
  for (int p = tid + kKvWriteRegs * kKvWriteThreads; p < pieces; p += kKvWriteThreads)
    put(p, ld_cg128(x + (p / per) * rs + (p % per) * 8));
}

struct KvReadArgs {
  KvPages c;
  const int8_t* codes[2];
  const float* scales[2];
  bf16* y[2];  // [B, rows, kv_heads, D]
  const int32_t* lens;
  int rows;
};

constexpr int kKvReadThreads = 256;

// bf16(code * scale) of the 4 codes of w.
__device__ __forceinline__ uint2 kv_values4(uint32_t w, float s) {
  const uint32_t u = w ^ 0x80808080u;  // code + 128
  auto f = [&](int sel) { return (__uint_as_float(__byte_perm(u, 0x4B000000u, sel)) - 8388736.0f) * s; };
  return make_uint2(pack_bf16x2(f(0x7440), f(0x7441)), pack_bf16x2(f(0x7442), f(0x7443)));
}

// Row i of the output is position len - rows + i (0 where that is negative).  One thread moves 16 codes.
__global__ void __launch_bounds__(kKvReadThreads) kv_read_kernel(const KvReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.y, which = blockIdx.z;
  const int per = a.c.D >> 4;
  const int64_t p = static_cast<int64_t>(blockIdx.x) * kKvReadThreads + threadIdx.x;
  const int64_t all = static_cast<int64_t>(a.rows) * a.c.kv_heads * per;
  if (p >= all) return;
  const int d = static_cast<int>(p % per);
  const int64_t rh = p / per;
  const int h = static_cast<int>(rh % a.c.kv_heads), r = static_cast<int>(rh / a.c.kv_heads);
  const int pos = ld_cg(a.lens + b) - a.rows + r;
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (pos >= 0) {
    const int64_t page = kv_page(a.c, b, pos >> a.c.log2_page);
    if (page >= 0) {
      const int64_t at = page * a.c.kv_heads + h;
      const float s = ld_cg(a.scales[which] + at);
      const int in = pos & ((1 << a.c.log2_page) - 1);
      const uint4 w = ld_cg128(a.codes[which] + ((at << a.c.log2_page) + in) * a.c.D + d * 16);
      const uint2 v0 = kv_values4(w.x, s), v1 = kv_values4(w.y, s), v2 = kv_values4(w.z, s), v3 = kv_values4(w.w, s);
      lo = make_uint4(v0.x, v0.y, v1.x, v1.y);
      hi = make_uint4(v2.x, v2.y, v3.x, v3.y);
    }
  }
  uint4* y = reinterpret_cast<uint4*>(a.y[which] + static_cast<int64_t>(b) * all * 16 + p * 16);
  y[0] = lo;
  y[1] = hi;
}

}  // namespace gguf_b200
