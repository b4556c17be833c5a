// Head norms of queries and keys with the position rotation in the same pass.
//   y = x * rsqrt(mean(x^2) + eps) * gamma      (per head; no gamma: y = x)
//   half layout:        (y[i], y[i + r/2]) -> (y[i] c_i - y[i + r/2] s_i, y[i + r/2] c_i + y[i] s_i)
//   interleaved layout: the same on (y[2i], y[2i + 1]);   values at r and above are not rotated
// fp32 throughout, one rounding to bf16.
//
// A group of kGL lanes owns one head: lane l holds eight of its values as two 8-byte pieces chosen so
// that both members of a pair sit in the same lane (no shuffles beyond the sum of squares), and the
// same two pieces of every head of a token use the same four cos and sin values, which are loaded once
// for the kHeads heads that a group works on.
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

template <int kGL, int kHeads, bool kInter>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const RopeArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int l = threadIdx.x % kGL;
  const int nq = (a.heads + kHeads - 1) / kHeads, nk = (a.kv_heads + kHeads - 1) / kHeads;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kRopeThreads / kGL) + threadIdx.x / kGL;
  const int64_t t = unit / (nq + nk);
  const bool live = t < a.T && 8 * l < a.D;  // idle lanes still take part in the shuffles
  const int part = static_cast<int>(unit % (nq + nk));
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
    if (live && h0 + i < hn) {
      va[i] = ld_cg64(xr + i * a.D + oa);
      vb[i] = ld_cg64(xr + i * a.D + ob);
    }
  }
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live && turns) {
    int p = ld_cg(a.pos + t);
    if (p < 0 || p >= a.max_pos) {
      record_device_error(kSiteBadPosition);
      p = 0;
    }
    const int64_t at = static_cast<int64_t>(p) * (a.rot / 2) + 4 * l;
    c = __ldg(reinterpret_cast<const float4*>(a.cos + at));
    s = __ldg(reinterpret_cast<const float4*>(a.sin + at));
  }
  const float* gamma = is_q ? a.gq : a.gk;
  float4 ga = make_float4(1.f, 1.f, 1.f, 1.f), gb = ga;
  if (gamma && live) {
    ga = __ldg(reinterpret_cast<const float4*>(gamma + oa));
    gb = __ldg(reinterpret_cast<const float4*>(gamma + ob));
  }
  const float rd = 1.0f / static_cast<float>(a.D);
  bf16* out = (is_q ? a.q : a.k) + (t * hn + h0) * a.D;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    float x0 = bf16_lo(va[i].x), x1 = bf16_hi(va[i].x), x2 = bf16_lo(va[i].y), x3 = bf16_hi(va[i].y);
    float z0 = bf16_lo(vb[i].x), z1 = bf16_hi(vb[i].x), z2 = bf16_lo(vb[i].y), z3 = bf16_hi(vb[i].y);
    if (gamma) {
      float ss = x0 * x0 + x1 * x1 + x2 * x2 + x3 * x3 + z0 * z0 + z1 * z1 + z2 * z2 + z3 * z3;
#pragma unroll
      for (int o = kGL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * rd + a.eps);
      x0 *= r * ga.x, x1 *= r * ga.y, x2 *= r * ga.z, x3 *= r * ga.w;
      z0 *= r * gb.x, z1 *= r * gb.y, z2 *= r * gb.z, z3 *= r * gb.w;
    }
    uint2 wa, wb;
    if (kInter) {
      wa.x = pack_bf16x2(x0 * c.x - x1 * s.x, x1 * c.x + x0 * s.x);
      wa.y = pack_bf16x2(x2 * c.y - x3 * s.y, x3 * c.y + x2 * s.y);
      wb.x = pack_bf16x2(z0 * c.z - z1 * s.z, z1 * c.z + z0 * s.z);
      wb.y = pack_bf16x2(z2 * c.w - z3 * s.w, z3 * c.w + z2 * s.w);
    } else {
      wa.x = pack_bf16x2(x0 * c.x - z0 * s.x, x1 * c.y - z1 * s.y);
      wa.y = pack_bf16x2(x2 * c.z - z2 * s.z, x3 * c.w - z3 * s.w);
      wb.x = pack_bf16x2(z0 * c.x + x0 * s.x, z1 * c.y + x1 * s.y);
      wb.y = pack_bf16x2(z2 * c.z + x2 * s.z, z3 * c.w + x3 * s.w);
    }
    if (live && h0 + i < hn) {
      *reinterpret_cast<uint2*>(out + i * a.D + oa) = wa;
      *reinterpret_cast<uint2*>(out + i * a.D + ob) = wb;
    }
  }
}

}  // namespace gguf_b200
