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

// Predicated forms, which leave the registers alone where `on` is false: behind a branch the compiler merges the two
// values with moves, which wait for the load.
__device__ __forceinline__ void ld_cg32_if(uint32_t& w, const void* p, bool on) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %2, 0;\n @p ld.global.cg.u32 %0, [%1];\n}\n" : "+r"(w) : "l"(p), "r"(on ? 1u : 0u) : "memory");
}
__device__ __forceinline__ void ld_cg64_if(uint2& v, const void* p, bool on) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %3, 0;\n @p ld.global.cg.v2.u32 {%0, %1}, [%2];\n}\n" : "+r"(v.x), "+r"(v.y)
               : "l"(p), "r"(on ? 1u : 0u) : "memory");
}
__device__ __forceinline__ void ld_cg128_if(uint4& v, const void* p, bool on) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %5, 0;\n @p ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];\n}\n"
               : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "l"(p), "r"(on ? 1u : 0u) : "memory");
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

// One CTA per (touched page, head, K or V) of a sequence: blockIdx = (page of the call * 2 + which, head, sequence).  The
// call's tokens of the page stay in registers between the maximum and the codes (16 KB at 64 tokens of 128 values); loads
// that do not depend on one another are issued before any is used: what is left in turn is lens, table entry, page.
template <int kD>
__global__ void __launch_bounds__(kKvWriteThreads) kv_write_kernel(const KvWriteArgs a) {
  constexpr int kPer = kD / 8;  // 16-byte pieces of a token
  __shared__ uint32_t red[kKvWriteThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, h = blockIdx.y, which = blockIdx.x & 1, tid = threadIdx.x;
  int len = ld_cg(a.lens + b), n = a.R;
  if (a.news) n = ld_cg(a.news + b);
  n = min(n, min(a.R, len));
  const int first = len - n;
  const int lg = a.c.log2_page, i = (first >> lg) + (blockIdx.x >> 1);
  const int begin = i << lg;
  if (n <= 0 || begin >= len) return;
  int entry = -1;
  if (i < a.c.table_cols) entry = ld_cg(a.c.table + static_cast<int64_t>(b) * a.c.table_cols + i);
  const int t0 = max(first, begin), t1 = min(len, begin + (1 << lg));
  const int pieces = (t1 - t0) * kPer;
  const int64_t rs = which ? a.stride_r[1] : a.stride_r[0];
  const bf16* x = (which ? a.x[1] : a.x[0]) + b * (which ? a.stride_b[1] : a.stride_b[0]) + (t0 - first) * rs + h * kD;

  uint4 keep[kKvWriteRegs];
#pragma unroll
  for (int j = 0; j < kKvWriteRegs; ++j) {
    const int p = tid + j * kKvWriteThreads;
    keep[j] = make_uint4(0, 0, 0, 0);
    ld_cg128_if(keep[j], x + (p / kPer) * rs + (p % kPer) * 8, p < pieces);
  }
  if (!kv_page_ok(a.c, entry)) return;
  const int64_t at = static_cast<int64_t>(entry) * a.c.kv_heads + h;
  int8_t* codes = (which ? a.codes[1] : a.codes[0]) + ((at << lg) * kD);
  float* scale_p = (which ? a.scales[1] : a.scales[0]) + at;
  const bool older = t0 > begin;
  float was = 0.f;
  if (older) was = ld_cg(scale_p);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < kKvWriteRegs; ++j)
    m = abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(m, keep[j].x), keep[j].y), keep[j].z), keep[j].w);
  for (int p = tid + kKvWriteRegs * kKvWriteThreads; p < pieces; p += kKvWriteThreads) {
    const uint4 v = ld_cg128(x + (p / kPer) * rs + (p % kPer) * 8);
    m = abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(m, v.x), v.y), v.z), v.w);
  }
  m = max(m & 0xFFFFu, m >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
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
    const int old_pieces = (t0 - begin) * kD >> 4;
    uint4* o = reinterpret_cast<uint4*>(codes);
    for (int p = tid; p < old_pieces; p += kKvWriteThreads) {
      uint4 v = ld_cg128(o + p);
      v.x = kv_rescale4(v.x, ratio), v.y = kv_rescale4(v.y, ratio);
      v.z = kv_rescale4(v.z, ratio), v.w = kv_rescale4(v.w, ratio);
      o[p] = v;
    }
  }
  uint2* o = reinterpret_cast<uint2*>(codes + static_cast<int64_t>(t0 - begin) * kD);
  auto put = [&](int p, uint4 v) {
    o[p] = make_uint2(kv_codes4(bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y), inv),
                      kv_codes4(bf16_lo(v.z), bf16_hi(v.z), bf16_lo(v.w), bf16_hi(v.w), inv));
  };
#pragma unroll
  for (int j = 0; j < kKvWriteRegs; ++j)
    if (tid + j * kKvWriteThreads < pieces) put(tid + j * kKvWriteThreads, keep[j]);
  for (int p = tid + kKvWriteRegs * kKvWriteThreads; p < pieces; p += kKvWriteThreads)
    put(p, ld_cg128(x + (p / kPer) * rs + (p % kPer) * 8));
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

// Row i of the output is position len - rows + i (0 where that is negative).  A thread moves kKvReadPieces times 16 codes,
// with all its table entries, then all its codes on their way at once, and stores 32 bytes at a time: 16-byte stores at
// 32-byte steps cost a third more (15k tokens of 8 heads of 128: 25 us).  blockIdx = (pieces, K or V, sequence).
constexpr int kKvReadPieces = 2;
template <int kD>
__global__ void __launch_bounds__(kKvReadThreads) kv_read_kernel(const KvReadArgs a) {
  constexpr int kPer = kD / 16, kN = kKvReadPieces;
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, which = blockIdx.y, lg = a.c.log2_page;
  const uint32_t all = static_cast<uint32_t>(a.rows) * a.c.kv_heads * kPer;  // fits: checked on the host
  const uint32_t p0 = blockIdx.x * (kKvReadThreads * kN) + threadIdx.x;
  const int begin = ld_cg(a.lens + b) - a.rows;
  const int32_t* table = a.c.table + static_cast<int64_t>(b) * a.c.table_cols;
  const int8_t* codes = which ? a.codes[1] : a.codes[0];
  const float* scales = which ? a.scales[1] : a.scales[0];
  bf16* out = which ? a.y[1] : a.y[0];
  uint32_t entry[kN];
  int pos[kN], h[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const uint32_t rh = (p0 + j * kKvReadThreads) / kPer, r = rh / a.c.kv_heads;
    h[j] = rh - r * a.c.kv_heads;
    pos[j] = p0 + j * kKvReadThreads < all ? begin + static_cast<int>(r) : -1;
    entry[j] = 0xFFFFFFFFu;
    ld_cg32_if(entry[j], table + (pos[j] >> lg), pos[j] >= 0 && (pos[j] >> lg) < a.c.table_cols);
  }
  uint4 w[kN];
  uint32_t s[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const bool on = pos[j] >= 0 && kv_page_ok(a.c, static_cast<int>(entry[j]));
    const int64_t at = static_cast<int64_t>(on ? entry[j] : 0u) * a.c.kv_heads + h[j];
    w[j] = make_uint4(0, 0, 0, 0);
    s[j] = 0;
    ld_cg32_if(s[j], scales + at, on);
    ld_cg128_if(w[j], codes + ((at << lg) + (pos[j] & ((1 << lg) - 1))) * kD + (p0 + j * kKvReadThreads) % kPer * 16, on);
  }
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const uint32_t p = p0 + j * kKvReadThreads;
    if (p >= all) break;
    const float sc = __uint_as_float(s[j]);
    const uint2 v0 = kv_values4(w[j].x, sc), v1 = kv_values4(w[j].y, sc), v2 = kv_values4(w[j].z, sc), v3 = kv_values4(w[j].w, sc);
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + (static_cast<int64_t>(b) * all + p) * 16),
                 "r"(v0.x), "r"(v0.y), "r"(v1.x), "r"(v1.y), "r"(v2.x), "r"(v2.y), "r"(v3.x), "r"(v3.y) : "memory");
  }
}

}  // namespace gguf_b200
