// Head norms of queries and keys with the position rotation in the same pass.
//   y = x * rsqrt(mean(x^2) + eps) * gamma      (per head; no gamma: y = x)
//   half layout:        (y[i], y[i + r/2]) -> (y[i] c_i - y[i + r/2] s_i, y[i + r/2] c_i + y[i] s_i)
//   interleaved layout: the same on (y[2i], y[2i + 1]);   values at r and above are not rotated
// fp32 throughout, one rounding to bf16.
//
// A group of kGL lanes owns one head: lane l holds eight of its values as two 8-byte pieces, chosen so that both members of
// a pair sit in the same lane (no shuffles beyond the sum of squares), and the same two pieces of every head of a token use
// the same four cos and sin values, which are loaded once for the kHeads heads that a group works on.  Bound by memory: 8191
// tokens of 32 + 8 heads of 128 take 33 to 34 us (5.2 TB/s); one head a group 43 us, 16-byte pieces on half the lanes 34.6 us.
#pragma once

#include "kv_cache.cuh"

namespace gguf_b200 {

struct RopeArgs {
  const bf16* x;  // [T] rows of (heads + 2 kv_heads) * D values, row_stride values apart
  const float *gq, *gk, *cos, *sin;
  const int32_t* pos;
  bf16 *q, *k;
  int64_t row_stride, T;
  int heads, kv_heads, D, rot, max_pos;
  float eps;
};

constexpr int kRopeThreads = 128;

__device__ __forceinline__ void rope_floats(float (&f)[4], const float* p) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(p));
  f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}

template <int kGL, int kHeads, bool kInter>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const RopeArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int l = threadIdx.x % kGL;
  const int nq = (a.heads + kHeads - 1) / kHeads, nk = (a.kv_heads + kHeads - 1) / kHeads;
  const uint32_t unit = blockIdx.x * (kRopeThreads / kGL) + threadIdx.x / kGL;  // (fits: checked on the host)
  const uint32_t t = unit / (nq + nk);
  const bool live = t < a.T && 8 * l < a.D;  // idle lanes still take part in the shuffles
  const int part = static_cast<int>(unit - t * (nq + nk));
  const bool is_q = part < nq;
  const int h0 = (is_q ? part : part - nq) * kHeads, hn = is_q ? a.heads : a.kv_heads;
  const bool turns = 8 * l < a.rot;
  const int oa = (turns && !kInter) ? 4 * l : 8 * l;
  const int ob = (turns && !kInter) ? a.rot / 2 + 4 * l : 8 * l + 4;

  uint2 va[kHeads], vb[kHeads];
  const bf16* xr = a.x + t * a.row_stride + static_cast<int64_t>(is_q ? h0 : a.heads + h0) * a.D;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    va[i] = vb[i] = make_uint2(0, 0);
    ld_cg64_if(va[i], xr + i * a.D + oa, live && h0 + i < hn);
    ld_cg64_if(vb[i], xr + i * a.D + ob, live && h0 + i < hn);
  }
  float c[4], s[4], ga[4], gb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = ga[i] = gb[i] = 1.f, s[i] = 0.f;
  if (live && turns) {
    int p = ld_cg(a.pos + t);
    if (p < 0 || p >= a.max_pos) {
      record_device_error(kSiteBadPosition);
      p = 0;
    }
    const int64_t at = static_cast<int64_t>(p) * (a.rot / 2) + 4 * l;
    rope_floats(c, a.cos + at);
    rope_floats(s, a.sin + at);
  }
  const float* gamma = is_q ? a.gq : a.gk;
  if (gamma && live) {
    rope_floats(ga, gamma + oa);
    rope_floats(gb, gamma + ob);
  }
  // A warp holds groups of queries and of keys: where only one of the two has a norm, all its lanes still take part in the
  // sums (the others' factor is 1), since the shuffles name the whole warp.
  const bool norms = a.gq || a.gk;
  const float rd = 1.0f / static_cast<float>(a.D);
  bf16* out = (is_q ? a.q : a.k) + (static_cast<int64_t>(t) * hn + h0) * a.D;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    float x[4] = {bf16_lo(va[i].x), bf16_hi(va[i].x), bf16_lo(va[i].y), bf16_hi(va[i].y)};
    float z[4] = {bf16_lo(vb[i].x), bf16_hi(vb[i].x), bf16_lo(vb[i].y), bf16_hi(vb[i].y)};
    if (norms) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) ss += x[j] * x[j] + z[j] * z[j];
#pragma unroll
      for (int o = kGL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = gamma ? rsqrtf(ss * rd + a.eps) : 1.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] *= r * ga[j], z[j] *= r * gb[j];
    }
    uint2 wa, wb;
    if (kInter) {
      wa.x = pack_bf16x2(x[0] * c[0] - x[1] * s[0], x[1] * c[0] + x[0] * s[0]);
      wa.y = pack_bf16x2(x[2] * c[1] - x[3] * s[1], x[3] * c[1] + x[2] * s[1]);
      wb.x = pack_bf16x2(z[0] * c[2] - z[1] * s[2], z[1] * c[2] + z[0] * s[2]);
      wb.y = pack_bf16x2(z[2] * c[3] - z[3] * s[3], z[3] * c[3] + z[2] * s[3]);
    } else {
      wa.x = pack_bf16x2(x[0] * c[0] - z[0] * s[0], x[1] * c[1] - z[1] * s[1]);
      wa.y = pack_bf16x2(x[2] * c[2] - z[2] * s[2], x[3] * c[3] - z[3] * s[3]);
      wb.x = pack_bf16x2(z[0] * c[0] + x[0] * s[0], z[1] * c[1] + x[1] * s[1]);
      wb.y = pack_bf16x2(z[2] * c[2] + x[2] * s[2], z[3] * c[3] + x[3] * s[3]);
    }
    if (live && h0 + i < hn) {
      *reinterpret_cast<uint2*>(out + i * a.D + oa) = wa;
      *reinterpret_cast<uint2*>(out + i * a.D + ob) = wb;
    }
  }
}

}  // namespace gguf_b200
