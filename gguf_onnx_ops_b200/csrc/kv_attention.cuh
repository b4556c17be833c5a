// Attention of a few query rows over the 8-bit paged KV cache (kv_cache.cuh), streaming kernel.
//   o = sum_j softmax_j(scale q . k_j) v_j over the positions j that a row sees
// Rows: query row r of sequence b (r < n) sits at position t = len - n + r and sees max(0, t - window + 1) .. t.
// The rows of one kv head (R query tokens x heads / kv_heads) share its K and V, which are read once for up to
// 8 kNT of them.
//
// Mathematics.  Codes enter the tensor cores as exact f16 integers; a row of q enters as f16 scaled by the power of two
// that puts its largest value in [2^14, 2^15), so its bf16 values are exact down to 2^-28 of the largest.  Scores, the
// running maximum, the sum and the output accumulators are fp32.  With s_j the base-2 logit and a_j the V scale of
// token j's page, the kernel keeps m = max_j (s_j + log2 a_j) and w_j = 2^(s_j + log2 a_j - m + 15) <= 2^15: the page
// scale of V is part of the exponent, so w_j in f16 multiplies the integer codes, O = sum w_j code_j, L = sum w_j / a_j,
// o = O / L.  L is kept times 2^-20: for V scales from 2^-112 to 2^106 neither it nor 2^-20 / a_j leaves fp32's normal numbers.
// A smaller scale counts as 2^-112 in w and L (0 as 2^-80, so that it does not push the others' weights out of f16's range),
// and its weights are multiplied by what is missing (0) for O.  w_j's rounding to f16 is the only one
// besides the final bf16: 2^-12 of w_j, averaged over the tokens; 2^-40 of the largest weight for weights below 2^-29
// of it, which is what the factor 2^15 is for (2^-26 of it where all V scales are below 2^-112, values below 2.5e-32).
//
// Work.  The cache positions of all (sequence, kv head, row tile) units are laid out in one line of 16-token tiles, with a
// stretch for each unit's own cost before them, and cut into equal slices, one per CTA, whatever the lengths are; lengths
// are read on the device, so a captured graph serves any of them.  The eight warps of a CTA take its tiles in turn, each with its own statistics, and meet at the end of
// the unit; a unit cut between CTAs leaves its pieces in the workspace, and the CTA that finishes last (a counter per
// unit) joins them in order, so results do not depend on timing.
//
// Bound.  Memory for many sequences (64 of 131 to 8009 tokens, 8 kv heads of 128: 101 us one call after the other, 5.3 TB/s;
// 111 us by itself, when nothing fills the ragged end).  For one of 131071 tokens (58 us, 4.7 TB/s) no unit is full (issue
// slots 49 %, ALU pipe 46 % busy): with one tile ahead, a warp's loads and its 390 instructions a tile take turns.  Few tokens
// are a chain of loads (lens, table, page, rows, pieces: 10 us for 777 tokens).  16 rows take half as long again as 8 (85 us
// against 57).  Other widths, 16 sequences of 801 to 9001 tokens, 8 rows a kv head, in us and of the bytes' time: 96 values 36
// (1.9x), 128 57 (2.3x), 192 62 (1.7x), 256 67 (1.4x).  Many rows of 96, 192 and 256 values are taken 16 at a time too: a chunk of
// 128 tokens, 64 heads over 8 kv heads, 9001 positions 254 / 386 / 492 us (96 / 192 / 256).
//
// A tile's fragments: S^T (16 tokens x 8 rows) = K (A operand) q^T (B), so that K goes straight from global memory
// into the A fragment: lane (g, t) loads 16 consecutive bytes of rows g and g + 8, and the order of the head's values
// inside the product is permuted alike in q.  exp of S^T, transposed by movmatrix, is the B operand of
// O^T (values x rows) = V^T (A) w, where lane (g, t) holds V bytes g D/8 .. of tokens 2t, 2t+1, 2t+8, 2t+9 and the bytes of
// two tokens are interleaved by a permute.  No shared memory is used for K and V.
#pragma once

#include "common.cuh"
#include "kv_cache.cuh"

namespace gguf_b200 {

struct KvAttnArgs {
  KvPages c;
  const int8_t *k, *v;
  const float *ks, *vs;
  const bf16* q;  // [B, R, heads, D], strides in values
  bf16* o;        // [B, R, heads, D]
  float* lse;     // [B, R, heads] or null
  const int32_t *lens, *news;
  int64_t q_stride_b, q_stride_r;
  float scale_log2;  // softmax scale * log2(e)
  int B, R, heads, group, window, row_tiles;
  int32_t* counters;  // one per unit, zero between calls
  float4* part;       // [2 grid][kNT D/16][32] pieces
  float2* ml;         // [2 grid][8 kNT]
};

constexpr int kKvWarps = 8;
constexpr int kKvThreads = kKvWarps * 32;
constexpr int kKvTile = 16;
// What a unit costs besides its tiles (rows read, warps joined, a result written), in tiles: the slices count it, or the CTAs
// that meet many short sequences end last (64 sequences of 131 to 8009 tokens, 8 rows of 128 values: 129 us without, 119 with 6,
// 101 with 24; the other widths use the same number, which was not measured for them).
constexpr int kKvUnitCost = 32;
constexpr int kKvMaxBatch = 4096;
constexpr float kKvTop = 15.f;  // the largest weight is 2^15, the top of f16's range
constexpr float kKvNone = 0x1p-80f, kKvLeast = 0x1p-112f;  // V scales in w and L: in place of 0, and the least
constexpr float kKvSum = 0x1p-20f, kKvSumLog2 = -20.f;      // of L

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t hsub2_u32(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2_u32(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// f16 pairs of bytes 0, 1 and of bytes 2, 3 of u (code + 128): 0x6400 | u is 1024 + u, less 1152.
__device__ __forceinline__ uint32_t codes_lo_f16x2(uint32_t u) { return hsub2_u32(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u); }
__device__ __forceinline__ uint32_t codes_hi_f16x2(uint32_t u) { return hsub2_u32(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What stands for the V scale v in w and L (NaN: the least), and its log2: NaN where v is not finite, so that every logit of
// the page is.
__device__ __forceinline__ float kv_counts_as(float v) { return v == 0.f ? kKvNone : fmaxf(v, kKvLeast); }
__device__ __forceinline__ float kv_log2(float v, float counts) { return fmaf(v, 0.f, lg2(counts)); }
// A K scale, NaN where it is not finite (an infinite one would make -inf of a negative score, and hide its token).
__device__ __forceinline__ float kv_finite(float k) { return fmaf(k, 0.f, k); }
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t scale_f16x2(uint32_t w, float by) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pack_f16x2(f.x * by, f.y * by);
}

// kBytes consecutive bytes (4, 8 or 16 at a time) of a cache page into words (predicated as ld_cg32_if); read
// once, kept out of L1.
template <int kBytes>
__device__ __forceinline__ void load_codes_if(uint32_t* w, const int8_t* p, bool on) {
  const uint32_t c = on ? 1u : 0u;
  if constexpr (kBytes % 16 == 0) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i)
      asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %5, 0;\n @p ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n}\n"
                   : "+r"(w[4 * i]), "+r"(w[4 * i + 1]), "+r"(w[4 * i + 2]), "+r"(w[4 * i + 3]) : "l"(p + 16 * i), "r"(c) : "memory");
  } else if constexpr (kBytes % 8 == 0) {
#pragma unroll
    for (int i = 0; i < kBytes / 8; ++i)
      asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %3, 0;\n @p ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];\n}\n"
                   : "+r"(w[2 * i]), "+r"(w[2 * i + 1]) : "l"(p + 8 * i), "r"(c) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i)
      asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %2, 0;\n @p ld.global.L1::no_allocate.u32 %0, [%1];\n}\n"
                   : "+r"(w[i]) : "l"(p + 4 * i), "r"(c) : "memory");
  }
}

// What the rows of sequence b see: positions lo .. len - 1 in all, len - n .. len - 1 are the rows' own.
struct KvSpan {
  int len, n, lo, t0, t1;  // tiles t0 .. t1 - 1
};
__device__ __forceinline__ KvSpan kv_span(const KvAttnArgs& a, int b) {
  KvSpan s;
  s.len = max(0, ld_cg(a.lens + b));
  const int cap = a.c.table_cols << a.c.log2_page;
  if (s.len > cap) {
    record_device_error(kSiteBadCachePage);
    s.len = cap;
  }
  s.n = max(0, min(a.news ? ld_cg(a.news + b) : a.R, min(a.R, s.len)));
  s.lo = a.window > 0 ? max(0, s.len - s.n + 1 - a.window) : 0;
  s.t0 = s.lo / kKvTile;
  s.t1 = s.n > 0 ? (s.len + kKvTile - 1) / kKvTile : s.t0;
  return s;
}

template <int kD, int kNT>
struct KvAttnPlan {
  static constexpr int kRows = 8 * kNT;
  static constexpr int kSteps = kD / 16;            // k16 steps of S, and value tiles of O
  static constexpr int kFrags = kNT * kSteps;       // O fragments (float4 per lane)
  static constexpr int kKPiece = kD % 64 == 0 ? 16 : 8;
  static constexpr int kQBytes = kNT * kSteps * 32 * 8;
  static constexpr int kOBytes = kKvWarps * kFrags * 32 * 16;
  static constexpr int kRowBytes = kRows * (4 + 4 + 4) + kKvWarps * kRows * 8;
  static constexpr int smem(int B) { return kQBytes + kOBytes + kRowBytes + 64 + (B + 1) * 4; }
  // CTAs per SM: two where 128 registers a thread are enough (96 values and 16 rows do not fit: one sequence of 131071
  // tokens 106 us with two, 81 with one; three for 64 values and 8 rows spill: 44.7 us against 40.9).
  static constexpr int kCtas = kD > 128 || (kD == 96 && kNT == 2) ? 1 : 2;
};

template <int kD, int kNT>
__global__ void __launch_bounds__(kKvThreads, KvAttnPlan<kD, kNT>::kCtas) kv_attention_kernel(const KvAttnArgs a) {
  using P = KvAttnPlan<kD, kNT>;
  extern __shared__ __align__(16) uint8_t smem[];
  uint2* qf = reinterpret_cast<uint2*>(smem);                       // [kNT][steps][32]
  float4* ob = reinterpret_cast<float4*>(smem + P::kQBytes);        // [warps][frags][32]
  float2* wml = reinterpret_cast<float2*>(smem + P::kQBytes + P::kOBytes);  // [warps][rows]
  float* row_scale = reinterpret_cast<float*>(wml + kKvWarps * P::kRows);
  int* row_hi = reinterpret_cast<int*>(row_scale + P::kRows);
  int* row_lo = row_hi + P::kRows;
  int* scratch = row_lo + P::kRows;  // 16 words
  int* prefix = scratch + 16;        // tiles of sequences before b

  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

  // Tiles of every sequence, summed (a sequence without any counts one, so that its rows are written).
  if (tid == 0) prefix[0] = 0;
  int carry = 0;
  for (int b0 = 0; b0 < a.B; b0 += kKvThreads) {
    int n = 0;
    if (b0 + tid < a.B) {
      const KvSpan s = kv_span(a, b0 + tid);
      n = kKvUnitCost + max(1, s.t1 - s.t0);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += x;
    }
    if (lane == 31) scratch[warp] = n;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < kKvWarps; ++w) {
      if (w < warp) before += scratch[w];
      carry += scratch[w];
    }
    if (b0 + tid < a.B) prefix[b0 + tid + 1] = before + n;
    __syncthreads();
  }
  const int per_seq = a.c.kv_heads * a.row_tiles;
  const int64_t total = static_cast<int64_t>(carry) * per_seq;
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), (total + 15) / 16);  // (no less than a tile a warp, on the whole)
  if (blockIdx.x >= ctas) return;
  int64_t at = total * blockIdx.x / ctas;
  const int64_t end = total * (blockIdx.x + 1) / ctas;

  while (at < end) {
    // The unit that holds tile `at`.
    int b = 0;
    for (int hi = a.B; hi - b > 1;) {
      const int mid = (b + hi) >> 1;
      if (static_cast<int64_t>(prefix[mid]) * per_seq <= at) b = mid; else hi = mid;
    }
    const KvSpan sp = kv_span(a, b);
    const int tiles = max(1, sp.t1 - sp.t0), span = kKvUnitCost + tiles;
    const int64_t in_seq = at - static_cast<int64_t>(prefix[b]) * per_seq;
    const int hr = static_cast<int>(in_seq / span), in_unit = static_cast<int>(in_seq % span);
    const int h = hr / a.row_tiles, rt = hr % a.row_tiles;
    const int64_t first_tile = at - in_unit + kKvUnitCost;  // where the unit's tiles begin in the line
    const int taken = static_cast<int>(min(static_cast<int64_t>(span - in_unit), end - at));
    const int ta = max(0, in_unit - kKvUnitCost), tb = in_unit + taken - kKvUnitCost;
    at += taken;
    if (tb <= ta) continue;  // the slice ends within the unit's cost

    // The warp's first tile on its way.
    uint32_t kw[2][P::kSteps] = {}, vw[4][kD / 32] = {};
    uint32_t ks = 0, vs = 0;  // bits of the tile's scales
    const int stop = min(sp.t0 + tb, sp.t1);
    int tile = sp.t0 + ta + warp;
    const int lg = a.c.log2_page, in_page = (1 << lg) - 1;
    const int32_t* table = a.c.table + static_cast<int64_t>(b) * a.c.table_cols;  // (positions below len lie in it)
    uint32_t entry = 0, entry_next = 0;  // pages of `tile` and of this warp's next tile
    // -1: not in the cache; nothing is loaded then, and the tile is hidden from every row
    auto page_of = [&](uint32_t e) { return kv_page_ok(a.c, static_cast<int>(e)) ? static_cast<int>(e) : -1; };
    auto row0 = [&](int page, int tl) {
      return (((static_cast<int64_t>(page) * a.c.kv_heads + h) << lg) + ((tl * kKvTile) & in_page)) * kD;
    };
    auto load_k = [&](int page, int tl, bool on) {
      const int8_t* p = a.k + row0(page, tl) + t * P::kKPiece;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < kD / (4 * P::kKPiece); ++j)
          load_codes_if<P::kKPiece>(&kw[r][j * (P::kKPiece / 4)], p + (g + 8 * r) * kD + j * 4 * P::kKPiece, on);
      ld_cg32_if(ks, a.ks + static_cast<int64_t>(page) * a.c.kv_heads + h, on);
      ld_cg32_if(vs, a.vs + static_cast<int64_t>(page) * a.c.kv_heads + h, on);
    };
    auto load_v = [&](int page, int tl, bool on) {
      const int8_t* p = a.v + row0(page, tl) + g * (kD / 8);
#pragma unroll
      for (int r = 0; r < 4; ++r) load_codes_if<kD / 8>(vw[r], p + (2 * t + (r & 1) + 8 * (r >> 1)) * kD, on);
    };
    ld_cg32_if(entry, table + ((tile * kKvTile) >> lg), tile < stop);
    ld_cg32_if(entry_next, table + (((tile + kKvWarps) * kKvTile) >> lg), tile + kKvWarps < stop);
    int page = page_of(entry);
    load_k(page, tile, tile < stop && page >= 0);
    load_v(page, tile, tile < stop && page >= 0);

    // Rows: q as f16 fragments, their limits.
    for (int n = warp; n < P::kRows; n += kKvWarps) {
      const int rr = rt * P::kRows + n, r = rr / a.group;
      const bool on = r < sp.n;
      const bf16* qr = a.q + b * a.q_stride_b + r * a.q_stride_r + static_cast<int64_t>(h * a.group + rr % a.group) * kD;
      constexpr int kPer = (kD / 4 + 31) / 32;
      uint2 w[kPer];
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        w[i] = make_uint2(0, 0);
        if (on && (lane + 32 * i) * 4 < kD) w[i] = ld_cg64(qr + (lane + 32 * i) * 4);
        m = abs_max_bf16x2(abs_max_bf16x2(m, w[i].x), w[i].y);
      }
      m = __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16));
      const int e = m ? min(127, 14 - (static_cast<int>(m >> 7) - 127)) : 0;
      const float up = pow2i(e);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int d = (lane + 32 * i) * 4;
        if (d < kD) {
          const int j = d / (4 * P::kKPiece), tt = d % (4 * P::kKPiece) / P::kKPiece, s = d % P::kKPiece / 4;
          const int step = j * (P::kKPiece / 4) + s;
          qf[((n >> 3) * P::kSteps + step) * 32 + (n & 7) * 4 + tt] =
              make_uint2(pack_f16x2(bf16_lo(w[i].x) * up, bf16_hi(w[i].x) * up),
                         pack_f16x2(bf16_lo(w[i].y) * up, bf16_hi(w[i].y) * up));
        }
      }
      if (lane == 0) {
        row_scale[n] = pow2i(-e) * a.scale_log2;
        const int last = sp.len - sp.n + r + 1;
        row_hi[n] = on ? last : sp.len;  // rows past the sequence's see everything and are written as zeros
        row_lo[n] = on && a.window > 0 ? max(0, last - a.window) : 0;
      }
    }
    __syncthreads();

    float m[kNT][2], l[kNT][2], o[kNT][P::kSteps][4], qs[kNT][2];
    int lo[kNT][2], hi[kNT][2], all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = nt * 8 + 2 * t + i;
        m[nt][i] = -INFINITY, l[nt][i] = 0.f;
        qs[nt][i] = row_scale[n];
        lo[nt][i] = row_lo[n], hi[nt][i] = row_hi[n];
        all_lo = max(all_lo, lo[nt][i]), all_hi = min(all_hi, hi[nt][i]);
      }
#pragma unroll
      for (int i = 0; i < P::kSteps; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }
    all_lo = __reduce_max_sync(0xffffffffu, all_lo);
    all_hi = __reduce_min_sync(0xffffffffu, all_hi);

    while (tile < stop) {
      const int next = tile + kKvWarps;
      float s[kNT][4];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int i = 0; i < P::kSteps; ++i) {
        const uint32_t u0 = kw[0][i] ^ 0x80808080u, u1 = kw[1][i] ^ 0x80808080u;
        const uint32_t a0 = codes_lo_f16x2(u0), a2 = codes_hi_f16x2(u0), a1 = codes_lo_f16x2(u1), a3 = codes_hi_f16x2(u1);
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const uint2 q2 = qf[(nt * P::kSteps + i) * 32 + lane];
          mma_f16_16816(s[nt], a0, a1, a2, a3, q2.x, q2.y);
        }
      }
      const float ks_now = kv_finite(__uint_as_float(ks)), vs_now = __uint_as_float(vs);
      const bool more = next < stop, here = page >= 0;
      page = page_of(entry_next);  // (read a tile ahead; page 0 where there is no next tile)
      const bool loads = more && page >= 0;
      load_k(page, next, loads);
      entry_next = more ? entry_next : 0;
      ld_cg32_if(entry_next, table + (((next + kKvWarps) * kKvTile) >> lg), next + kKvWarps < stop);

      // (the reciprocal is finite whatever the page's scale is: a row that the mask hides from the page adds 0 times it)
      const float av = kv_counts_as(vs_now), lv = kv_log2(vs_now, av), inv_v = __fdividef(kKvSum, av);
      const int p0 = tile * kKvTile;
      const bool whole = p0 >= all_lo && p0 + kKvTile <= all_hi && here;
      uint32_t pb[kNT][2];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        const float c0 = qs[nt][0] * ks_now, c1 = qs[nt][1] * ks_now;
        float x[4] = {fmaf(s[nt][0], c0, lv), fmaf(s[nt][1], c1, lv), fmaf(s[nt][2], c0, lv), fmaf(s[nt][3], c1, lv)};
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = p0 + g + 8 * (i >> 1);
            if (pos < lo[nt][i & 1] || pos >= hi[nt][i & 1] || !here) x[i] = -INFINITY;
          }
        }
        float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], sh));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], sh));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[nt][0] || mx[1] > m[nt][1])) {
          float f[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float mn = fmaxf(m[nt][i], mx[i]);
            f[i] = mn == -INFINITY ? 1.f : ex2(m[nt][i] - mn);
            m[nt][i] = mn;
            l[nt][i] *= f[i];
          }
#pragma unroll
          for (int i = 0; i < P::kSteps; ++i) {
            o[nt][i][0] *= f[0], o[nt][i][1] *= f[1], o[nt][i][2] *= f[0], o[nt][i][3] *= f[1];
          }
        }
        const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0] - kKvTop, m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1] - kKvTop;
        const float w0 = ex2(x[0] - m0), w1 = ex2(x[1] - m1), w2 = ex2(x[2] - m0), w3 = ex2(x[3] - m1);
        l[nt][0] = fmaf(w0 + w2, inv_v, l[nt][0]);
        l[nt][1] = fmaf(w1 + w3, inv_v, l[nt][1]);
        pb[nt][0] = movmatrix_trans(pack_f16x2(w0, w1));
        pb[nt][1] = movmatrix_trans(pack_f16x2(w2, w3));
      }
      if (vs_now < kKvLeast) {
        const float by = vs_now * (1.f / kKvLeast);
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) pb[nt][0] = scale_f16x2(pb[nt][0], by), pb[nt][1] = scale_f16x2(pb[nt][1], by);
      }
#pragma unroll
      for (int j = 0; j < kD / 32; ++j) {
        const uint32_t x0 = vw[0][j] ^ 0x80808080u, x1 = vw[1][j] ^ 0x80808080u;
        const uint32_t y0 = vw[2][j] ^ 0x80808080u, y1 = vw[3][j] ^ 0x80808080u;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t px = __byte_perm(x0, x1, k ? 0x7362 : 0x5140), py = __byte_perm(y0, y1, k ? 0x7362 : 0x5140);
          const uint32_t a0 = codes_lo_f16x2(px), a1 = codes_hi_f16x2(px), a2 = codes_lo_f16x2(py), a3 = codes_hi_f16x2(py);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) mma_f16_16816(o[nt][2 * j + k], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
        }
      }
      load_v(page, next, loads);
      tile = next;
    }

    // The warps meet.
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) {
        l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], sh);
        l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], sh);
      }
      if (g == 0) {
        wml[warp * P::kRows + nt * 8 + 2 * t] = make_float2(m[nt][0], l[nt][0]);
        wml[warp * P::kRows + nt * 8 + 2 * t + 1] = make_float2(m[nt][1], l[nt][1]);
      }
#pragma unroll
      for (int i = 0; i < P::kSteps; ++i)
        ob[(warp * P::kFrags + nt * P::kSteps + i) * 32 + lane] =
            make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
    }
    __syncthreads();

    // Piece or whole?  A piece goes to slot 0 of this CTA when its unit began in an earlier one, else to slot 1.
    const int64_t c_first = ((first_tile + 1) * ctas - 1) / total;
    const int64_t c_last = ((first_tile + tiles) * ctas - 1) / total;
    const int pieces = static_cast<int>(c_last - c_first) + 1;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (ta > 0 ? 0 : 1);
    const int64_t unit = (static_cast<int64_t>(b) * a.c.kv_heads + h) * a.row_tiles + rt;
    auto finish = [&](int n, int d, float v0, float v1, float sum, float mx) {  // values d, d + 1 of row n
      const int rr = rt * P::kRows + n, r = rr / a.group;
      if (r >= a.R) return;
      const bool some = r < sp.n;
      const float inv = some ? (sum == 0.f ? 0.f : 1.0f / sum) : 0.f;
      const int64_t row = (static_cast<int64_t>(b) * a.R + r) * a.heads + h * a.group + rr % a.group;
      *reinterpret_cast<uint32_t*>(a.o + row * kD + d) = some ? pack_bf16x2(v0 * kKvSum * inv, v1 * kKvSum * inv) : 0u;
      if (a.lse && d == 0) a.lse[row] = some && sum != 0.f ? (mx - kKvTop - kKvSumLog2 + lg2(sum)) * 0.69314718055994531f : -INFINITY;
    };
    for (int f = warp; f < P::kFrags; f += kKvWarps) {
      const int nt = f / P::kSteps, i = f % P::kSteps, n = nt * 8 + 2 * t;
      float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kKvWarps; ++w) {
        mx[0] = fmaxf(mx[0], wml[w * P::kRows + n].x);
        mx[1] = fmaxf(mx[1], wml[w * P::kRows + n + 1].x);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kKvWarps; ++w) {
        const float2 u0 = wml[w * P::kRows + n], u1 = wml[w * P::kRows + n + 1];
        const float f0 = u0.x == -INFINITY ? 0.f : ex2(u0.x - mx[0]), f1 = u1.x == -INFINITY ? 0.f : ex2(u1.x - mx[1]);
        const float4 v = ob[(w * P::kFrags + f) * 32 + lane];
        sum[0] = fmaf(u0.y, f0, sum[0]), sum[1] = fmaf(u1.y, f1, sum[1]);
        acc.x = fmaf(v.x, f0, acc.x), acc.y = fmaf(v.y, f1, acc.y);
        acc.z = fmaf(v.z, f0, acc.z), acc.w = fmaf(v.w, f1, acc.w);
      }
      if (pieces == 1) {
        const int d = g * (kD / 8) + 2 * i;
        finish(n, d, acc.x, acc.z, sum[0], mx[0]);
        finish(n + 1, d, acc.y, acc.w, sum[1], mx[1]);
      } else {
        __stcg(a.part + (slot * P::kFrags + f) * 32 + lane, acc);
        if (i == 0 && g == 0) {
          __stcg(a.ml + slot * P::kRows + n, make_float2(mx[0], sum[0]));
          __stcg(a.ml + slot * P::kRows + n + 1, make_float2(mx[1], sum[1]));
        }
      }
    }
    if (pieces > 1) {
      __threadfence();
      __syncthreads();
      if (tid == 0) scratch[8] = atomicAdd(a.counters + unit, 1);
      __syncthreads();
      if (scratch[8] == pieces - 1) {  // the last of the unit's CTAs joins the pieces
        __threadfence();
        if (tid == 0) a.counters[unit] = 0;
        for (int f = warp; f < P::kFrags; f += kKvWarps) {
          const int nt = f / P::kSteps, i = f % P::kSteps, n = nt * 8 + 2 * t;
          float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
          for (int p = 0; p < pieces; ++p) {
            const int64_t sl = 2 * (c_first + p) + (p == 0 ? 1 : 0);
            mx[0] = fmaxf(mx[0], ld_cg(a.ml + sl * P::kRows + n).x);
            mx[1] = fmaxf(mx[1], ld_cg(a.ml + sl * P::kRows + n + 1).x);
          }
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int p = 0; p < pieces; ++p) {
            const int64_t sl = 2 * (c_first + p) + (p == 0 ? 1 : 0);
            const float2 u0 = ld_cg(a.ml + sl * P::kRows + n), u1 = ld_cg(a.ml + sl * P::kRows + n + 1);
            const float4 v = ld_cg(a.part + (sl * P::kFrags + f) * 32 + lane);
            const float f0 = u0.x == -INFINITY ? 0.f : ex2(u0.x - mx[0]), f1 = u1.x == -INFINITY ? 0.f : ex2(u1.x - mx[1]);
            sum[0] = fmaf(u0.y, f0, sum[0]), sum[1] = fmaf(u1.y, f1, sum[1]);
            acc.x = fmaf(v.x, f0, acc.x), acc.y = fmaf(v.y, f1, acc.y);
            acc.z = fmaf(v.z, f0, acc.z), acc.w = fmaf(v.w, f1, acc.w);
          }
          const int d = g * (kD / 8) + 2 * i;
          finish(n, d, acc.x, acc.z, sum[0], mx[0]);
          finish(n + 1, d, acc.y, acc.w, sum[1], mx[1]);
        }
      }
    }
    __syncthreads();  // shared memory is reused by the next unit
  }
}

}  // namespace gguf_b200
