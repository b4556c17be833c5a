// Attention of many query rows over the 8-bit paged KV cache: 128-row tiles on tcgen05 (the formulas, the scaling of q
// and the use of V's page scale are those of kv_attention.cuh; w_j <= 2^15 here too, kept so by a running maximum that moves
// only when it has grown by more than 2^4, with weights scaled to 2^11: f16 rounds a weight by 2^-12 of it, or by 2^-36 of the
// largest for weights below 2^-25 of it, 2^-22 where all V scales are below 2^-112).
//
// Why.  R * heads / kv_heads rows share the K and V of a kv head.  The streaming kernel converts the codes once per 16
// rows and multiplies on mma.sync; from 17 rows on that work, not the bytes, is its time (48 rows, 16 sequences of 801 to 9001
// tokens: 144 us for 25 us of bytes, 79 us here).  Here a CTA converts each 128-token tile of codes once, to f16 in shared
// memory, for up to 256 rows, and the products run on the 5th-generation tensor cores.
//
// One CTA per SM, seven warp groups; the tokens go by in steps of 64:
//   warps 0-7, 8-15  softmax of stream 0 and 1: two threads per row, scores and O in tensor memory
//   warps 16-19, 20-23  K and V codes to f16, stored swizzled for the MMAs: three buffers each; and a unit's q
//   warp 27          page scales
//   warp 25          copies codes into a ring of steps (bulk copies, a page each: loads through the L1 stop at what the
//                    28 KB beside this much shared memory hold, 2 us a tile)
//   warps 24 and 26  issue the MMAs of a stream: S = q K^T (128 x 64), then O += w V with w (f16) in the columns of its S.
//                    Every stream has two S, so that the next scores are there before this step's weights are done (one S
//                    and two places for weights: a step of a chunk 5 % longer)
// A stream is a 128-row tile against every step when a unit has two row tiles (256 rows share the converted codes), or
// one row tile against every second step when it has one (two accumulators, joined at the end).
// The line of all units' 128-token tiles is cut into equal slices as in the streaming kernel; a second kernel joins the pieces.
//
// Bound.  A step of two streams takes about 2300 cycles: the softmax warps' instructions (issue slots 60 % used, the exp unit
// 40 %) and the round of waits between them and the MMAs (tensor pipe 39 %).  A chunk of 1001 tokens, 32 heads over 8 kv
// heads of 128, 9001 positions: 187 us, 745 TFLOP/s, 16 us of it the joining kernel.  A unit's begin and end take 5000
// cycles each, a launch 15000 before the first step, which is what few tokens cost.  With parts left out (of 195 us before
// the last steps): 172 us without exponentials, 180 with an eighth of S's products, no less without the conversion of the codes.
#pragma once

#include <type_traits>

#include "kv_attention.cuh"
#include "tcgen05.cuh"

namespace gguf_b200 {

constexpr int kTileSoftmax = 512, kTileConvert = 256, kTileThreads = kTileSoftmax + kTileConvert + 128;
constexpr int kTileConvertWarp = kTileSoftmax / 32, kTileConvertWarps = kTileConvert / 32, kTileMmaWarp = (kTileSoftmax + kTileConvert) / 32;
// Registers a thread: the kernel is launched with at least kTileLaunchRegs (checked on the host), 64512 in all; the
// softmax groups then take 88, the converting ones 40 and the last group 72: 45056 + 10240 + 9216 = 64512.
constexpr int kTileLaunchRegs = 72, kTileSoftmaxRegs = 88, kTileConvertRegs = 40, kTileOtherRegs = 72;
static_assert(kTileSoftmax * kTileSoftmaxRegs + kTileConvert * kTileConvertRegs + 128 * kTileOtherRegs <= kTileThreads * kTileLaunchRegs,
              "the shares must fit what the CTA is launched with");
constexpr int kTileTokens = 128;          // what the work is cut by
constexpr int kTileStep = 64;             // tokens of a step
constexpr int kTileMaxBatch = 2048;       // what the shared memory leaves room for (a larger batch is streamed)
constexpr int kTileBufs = 3;              // K and V buffers
constexpr int kTileUnitCost = 4;          // of a unit besides its tiles, in tiles (kKvUnitCost)
constexpr int kTileRows = 128;            // of one stream
constexpr int kTileUnitRows = 2 * kTileRows;
constexpr float kTileTop = 11.f, kTileGrow = 4.f;  // weights start at 2^11 and may grow to 2^15

template <int kD>
struct KvTilePlan {
  static constexpr int kQTile = kTileRows * kD * 2;      // f16 bytes of a q tile
  static constexpr int kOperand = kTileStep * kD * 2;    // f16 bytes of a step of K or V
  static constexpr int kBlock = kTileStep * 128;         // of which each 64 values of a head take this much
  static constexpr int kPieces = kTileStep * kD / 8 / 128;  // 8-code pieces per converting thread
  static constexpr int kRaw = kTileStep * kD;            // bytes of a staged step of codes
  static constexpr int kRing = kD == 128 ? 6 : 12;       // staged steps, K and V in turn: 48 KB
  static constexpr int kVAt = kTileBufs * kOperand, kQAt = 2 * kVAt, kRingAt = kQAt + 2 * kQTile, kCtrlAt = kRingAt + kRing * kRaw;
  static constexpr int kCtrl = 8304;                     // scales, barriers, small shared state
  static constexpr int smem(int B) { return 1024 + kCtrlAt + kCtrl + (B + 1) * 4; }
  // Tensor memory columns of stream s: its two S (the f16 weights over their S), O.
  __host__ __device__ static constexpr uint32_t s_at(int s, int buf) { return 128u * s + 64u * buf; }
  __host__ __device__ static constexpr uint32_t o_at(int s) { return 256u + kD * s; }
  static_assert(smem(kTileMaxBatch) <= 227 * 1024, "shared memory");
};

struct KvTileCtrl {
  // By step % 8 and group of 16 tokens.  A V scale below kKvLeast turns the sign of inv_v[0] or [2] (the softmax threads take two
  // groups each and look at the first one's sign alone); weights are then multiplied by mul (f16 twice, a power of two or 0).
  alignas(16) float scale_k[8][4], lv[8][4], inv_v[8][4];
  uint32_t mul[8][4];
  uint64_t k_full[kTileBufs], k_empty[kTileBufs], v_full[kTileBufs], v_empty[kTileBufs], raw_full[12], raw_empty[12];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], q_full[2], q_free;  // [stream][item % 2]: an item is a stream's step
  uint32_t tmem;
  int scan[28];
  float2 hand[kTileRows];   // maximum and sum of stream 1, handed to stream 0
  float swap[2][2][2][kTileRows];  // [maxima of items, else][stream][half][row]: what a row's two threads tell each other
  float row_scale[2][2][kTileRows];  // [unit % 2][row tile][row]: of the scores
};
static_assert(sizeof(KvTileCtrl) <= 8304, "control block");

// The token tiles of the 256-row unit rt of a sequence: t0 .. t1 - 1.
__device__ __forceinline__ void kv_tile_range(const KvAttnArgs& a, const KvSpan& s, int rt, int& t0, int& t1) {
  const int r0 = rt * kTileUnitRows / a.group;
  if (r0 >= s.n) {
    t0 = t1 = 0;
    return;
  }
  const int r1 = min(s.n - 1, ((rt + 1) * kTileUnitRows - 1) / a.group);
  const int hi = s.len - s.n + r1 + 1;
  const int lo = a.window > 0 ? max(0, s.len - s.n + r0 + 1 - a.window) : 0;
  t0 = lo / kTileTokens;
  t1 = (hi + kTileTokens - 1) / kTileTokens;
}

__device__ __forceinline__ int kv_tile_cost(const KvAttnArgs& a, const KvSpan& s, int rt) {
  int t0, t1;
  kv_tile_range(a, s, rt, t0, t1);
  return kTileUnitCost + max(1, t1 - t0);
}
// Of row tiles 0 .. n - 1, by a whole warp (one thread takes 5500 cycles for 16 row tiles).
__device__ __forceinline__ int kv_tile_cost_sum(const KvAttnArgs& a, const KvSpan& s, int n) {
  int c = 0;
  for (int rt = threadIdx.x & 31; rt < n; rt += 32) c += kv_tile_cost(a, s, rt);
  return __reduce_add_sync(0xffffffffu, c);
}
// 32-bit where the numbers allow it: a 64-bit division is some hundred instructions.
__device__ __forceinline__ int64_t kv_div(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

struct KvTileUnit {
  KvSpan sp;
  int b, h, rt, t0, ta, tb, tiles;  // token tiles t0 + ta .. t0 + tb - 1 of this CTA, of `tiles`
  int taken;                        // how far the slice has come with it
  bool mine, work, two;             // mine: tiles are this CTA's; work: rows see something; two: two row tiles
};
// The unit that holds place `at` of the line (called by whole warps).
__device__ __forceinline__ KvTileUnit kv_tile_unit(const KvAttnArgs& a, const int* prefix, int64_t at, int64_t end) {
  KvTileUnit u;
  int b = 0;
  for (int hi = a.B; hi - b > 1;) {
    const int mid = (b + hi) >> 1;
    if (static_cast<int64_t>(prefix[mid]) * a.c.kv_heads <= at) b = mid; else hi = mid;
  }
  u.b = b;
  u.sp = kv_span(a, b);
  const int per_head = prefix[b + 1] - prefix[b];
  const int64_t in_seq = at - static_cast<int64_t>(prefix[b]) * a.c.kv_heads;
  u.h = static_cast<int>(kv_div(in_seq, per_head));
  int rem = static_cast<int>(in_seq - static_cast<int64_t>(u.h) * per_head), t1 = 0;
  if (a.row_tiles == 1) {
    u.rt = 0;
    kv_tile_range(a, u.sp, 0, u.t0, t1);
  } else {
    const int lane = threadIdx.x & 31;
    for (int base = 0;; base += 32) {
      const int rt = base + lane;
      int mt0 = 0, mt1 = 0, cost = 0;
      if (rt < a.row_tiles) {
        kv_tile_range(a, u.sp, rt, mt0, mt1);
        cost = kTileUnitCost + max(1, mt1 - mt0);
      }
      int sum = cost;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, rem < sum || rt >= a.row_tiles - 1);
      if (hit) {
        const int f = __ffs(hit) - 1;
        u.rt = base + f;
        u.t0 = __shfl_sync(0xffffffffu, mt0, f), t1 = __shfl_sync(0xffffffffu, mt1, f);
        rem -= __shfl_sync(0xffffffffu, sum - cost, f);
        break;
      }
      rem -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  u.tiles = max(1, t1 - u.t0);
  u.taken = static_cast<int>(min(static_cast<int64_t>(kTileUnitCost + u.tiles - rem), end - at));
  u.ta = max(0, rem - kTileUnitCost);
  u.tb = rem + u.taken - kTileUnitCost;
  u.mine = u.tb > u.ta;
  u.work = u.mine && t1 > u.t0;
  u.two = a.R * a.group - u.rt * kTileUnitRows > kTileRows;
  return u;
}

// Token tiles of every sequence (all row units of one head), summed: prefix[b] before sequence b; returns the total.
template <int kThreads>
__device__ __forceinline__ int kv_tile_prefix(const KvAttnArgs& a, int* prefix, int* scan) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (a.row_tiles > 1) {
    for (int b = warp; b < a.B; b += kThreads / 32) {
      const int c = kv_tile_cost_sum(a, kv_span(a, b), a.row_tiles);
      if (lane == 0) prefix[b + 1] = c;
    }
    __syncthreads();
  }
  int carry = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    int n = 0;
    if (b0 + tid < a.B) n = a.row_tiles > 1 ? prefix[b0 + tid + 1] : kv_tile_cost(a, kv_span(a, b0 + tid), 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += x;
    }
    if (lane == 31) scan[warp] = n;
    __syncthreads();
    int before = carry;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += scan[w];
      carry += scan[w];
    }
    if (b0 + tid < a.B) prefix[b0 + tid + 1] = before + n;
    if (b0 + tid == 0) prefix[0] = 0;
    __syncthreads();
  }
  return carry;
}
__device__ __forceinline__ int64_t kv_tile_ctas(int64_t total, int grid) {
  return min(static_cast<int64_t>(grid), (total + kTileUnitCost + 1) / (kTileUnitCost + 2));
}
// Workspace slot of CTA c's piece of stream s: every CTA cuts at most one unit at its front and one at its end.
__device__ __forceinline__ int64_t kv_tile_slot(int64_t c, bool begins, int s) { return (2 * c + (begins ? 1 : 0)) * 2 + s; }

__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A wait that gives up for good after its first timeout (which is recorded).
__device__ __forceinline__ void tile_wait(uint64_t* bar, uint32_t phase, bool& dead) {
  if (!dead && !mbar_wait(bar, phase & 1u, kSiteTileWait)) dead = true;
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// The same, and whether any of the threads says so.
__device__ __forceinline__ bool bar_any(int id, int threads, bool mine) {
  uint32_t any;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n bar.red.or.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(any) : "r"(id), "r"(threads), "r"(mine ? 1u : 0u) : "memory");
  return any != 0;
}

template <int kD>
__global__ void __launch_bounds__(kTileThreads, 1) kv_attention_tile_kernel(const KvAttnArgs a) {
  using P = KvTilePlan<kD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *k_buf = smem, *v_buf = smem + P::kVAt, *q_buf = smem + P::kQAt, *ring = smem + P::kRingAt;
  KvTileCtrl* ct = reinterpret_cast<KvTileCtrl*>(smem + P::kCtrlAt);
  int* prefix = reinterpret_cast<int*>(smem + P::kCtrlAt + P::kCtrl);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (warp == kTileMmaWarp) {
    tmem_alloc(&ct->tmem, 512);
    if (lane == 0) {
      for (int i = 0; i < kTileBufs; ++i) {
        mbar_init(&ct->k_full[i], kTileConvertWarps / 2 + 1), mbar_init(&ct->v_full[i], kTileConvertWarps / 2);
        mbar_init(&ct->k_empty[i], 2), mbar_init(&ct->v_empty[i], 2);
      }
      for (int i = 0; i < 2; ++i) {
        for (int j = 0; j < 2; ++j) mbar_init(&ct->s_full[i][j], 1), mbar_init(&ct->p_full[i][j], 8), mbar_init(&ct->pv_done[i][j], 1);
        mbar_init(&ct->q_full[i], kTileConvertWarps);
      }
      mbar_init(&ct->q_free, 2);
      for (int i = 0; i < P::kRing; ++i) mbar_init(&ct->raw_full[i], 1), mbar_init(&ct->raw_empty[i], kTileConvertWarps / 2);
      fence_mbar_init();
    }
    tc_fence_before();
  }
  pdl_wait();
  pdl_launch_dependents();

  const int carry = kv_tile_prefix<kTileThreads>(a, prefix, ct->scan);
  tc_fence_after();
  // All 512 columns are this CTA's, so they begin at column 0 (KvTilePlan has their use).
  const int64_t total = static_cast<int64_t>(carry) * a.c.kv_heads, ctas = kv_tile_ctas(total, gridDim.x);
  const int64_t from = kv_div(total * blockIdx.x, max(ctas, static_cast<int64_t>(1)));
  const int64_t end = blockIdx.x < ctas ? kv_div(total * (blockIdx.x + 1), ctas) : from;
  bool dead = false;

  if (warp >= kTileConvertWarp && warp < kTileMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTileConvertRegs));
    // ---------------------------------------------------------------- codes to f16
    // Piece i of a thread: 8 codes of token tok + i * kTokStep, one 16-byte chunk of f16, stored at chunk ^ token % 8 of the
    // token's 128-byte row (tokens of a thread are alike modulo 8).  Eight lanes read 64 bytes in a row and write eight
    // different chunks: no bank conflicts on either side.
    // The first group takes K, the second V.
    constexpr int kParts = kD / 8, kTokStep = 128 / kParts;
    const int cw = warp & 3, part = lane % kParts, tok = (cw * 32 + lane) / kParts;
    const bool is_v = warp >= kTileConvertWarp + 4;
    const int dst = (part >> 3) * P::kBlock + tok * 128 + (((part & 7) ^ (tok & 7)) << 4);
    const uint8_t* raw0 = ring + tok * kD + part * 8;
    uint8_t* buf0 = (is_v ? v_buf : k_buf) + dst;
    uint64_t *full = is_v ? ct->v_full : ct->k_full, *empty = is_v ? ct->v_empty : ct->k_empty;
    uint32_t slot = is_v ? 1 : 0, slot_use = 0, buf = 0, use = 0, units = 0;
    for (int64_t at = from; at < end;) {
      const KvTileUnit u = kv_tile_unit(a, prefix, at, end);
      at += u.taken;
      if (!u.work) continue;
      // The unit's q, while the softmax is still at the unit before: the largest value of a row to [2^14, 2^15) by a power of
      // two, a negative softmax scale into its sign.  A group takes a row tile, or half of the only one; a warp a fourth
      // of that, kD / 8 lanes a row, so that its loads are whole lines.
      {
        constexpr int kLanes = kD / 8, kAtOnce = 32 / kLanes, kRound = 4;
        const int rows = u.two ? 32 : 16, qt = u.two && is_v ? 1 : 0, row0 = (u.two ? 0 : is_v ? 64 : 0) + cw * rows, c = lane % kLanes;
        const int my = u.rt * kTileUnitRows + qt * kTileRows + row0 + (lane & (rows - 1)), my_r = my / a.group;  // lane j knows where row j is
        const int64_t my_at = u.b * a.q_stride_b + my_r * a.q_stride_r + static_cast<int64_t>(u.h * a.group + my - my_r * a.group) * kD;
        const uint32_t rows_on = __ballot_sync(0xffffffffu, my_r < u.sp.n);
        uint8_t* dst_q = q_buf + qt * P::kQTile + (c >> 3) * (kTileRows * 128);
        if (units > 0) tile_wait(&ct->q_free, units - 1, dead);
#pragma unroll 1
        for (int i0 = 0; i0 < rows; i0 += kRound * kAtOnce) {
          uint4 w[kRound];
#pragma unroll
          for (int i = 0; i < kRound; ++i) {
            const int j = i0 + i * kAtOnce + lane / kLanes;
            const int64_t row_at = __shfl_sync(0xffffffffu, my_at, j);
            w[i] = make_uint4(0, 0, 0, 0);
            ld_cg128_if(w[i], a.q + row_at + c * 8, rows_on >> j & 1);
          }
#pragma unroll
          for (int i = 0; i < kRound; ++i) {
            const int j = row0 + i0 + i * kAtOnce + lane / kLanes;
            uint32_t m = abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(abs_max_bf16x2(0u, w[i].x), w[i].y), w[i].z), w[i].w);
            m = max(m & 0xFFFFu, m >> 16);
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const int e = m ? min(127, 14 - (static_cast<int>(m >> 7) - 127)) : 0;
            if (c == 0) ct->row_scale[units & 1][qt][j] = pow2i(-e) * fabsf(a.scale_log2);
            const float up = a.scale_log2 < 0.f ? -pow2i(e) : pow2i(e);
            *reinterpret_cast<uint4*>(dst_q + j * 128 + (((c & 7) ^ (j & 7)) << 4)) =
                make_uint4(pack_f16x2(bf16_lo(w[i].x) * up, bf16_hi(w[i].x) * up), pack_f16x2(bf16_lo(w[i].y) * up, bf16_hi(w[i].y) * up),
                           pack_f16x2(bf16_lo(w[i].z) * up, bf16_hi(w[i].z) * up), pack_f16x2(bf16_lo(w[i].w) * up, bf16_hi(w[i].w) * up));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ct->q_full[units & 1]);
        ++units;
      }
      for (int left = 2 * (u.tb - u.ta); left > 0; --left) {
        tile_wait(&ct->raw_full[slot], slot_use, dead);
        uint2 r[P::kPieces];
#pragma unroll
        for (int i = 0; i < P::kPieces; ++i) r[i] = *reinterpret_cast<const uint2*>(raw0 + slot * P::kRaw + i * kTokStep * kD);
        if (use > 0) tile_wait(empty + buf, use - 1, dead);
#pragma unroll
        for (int i = 0; i < P::kPieces; ++i) {
          const uint32_t x0 = r[i].x ^ 0x80808080u, x1 = r[i].y ^ 0x80808080u;
          *reinterpret_cast<uint4*>(buf0 + buf * P::kOperand + i * kTokStep * 128) =
              make_uint4(codes_lo_f16x2(x0), codes_hi_f16x2(x0), codes_lo_f16x2(x1), codes_hi_f16x2(x1));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(full + buf);
          mbar_arrive(&ct->raw_empty[slot]);
        }
        if (++buf == kTileBufs) buf = 0, ++use;
        if ((slot += 2) >= P::kRing) slot -= P::kRing, ++slot_use;
      }
    }
  } else if (warp >= kTileMmaWarp) {  // (keeps what it was launched with)
    if (warp == kTileMmaWarp + 1) {
    // ---------------------------------------------------------------- copies of codes
    const int lg = a.c.log2_page;
    const int chunk = min(1 << lg, kTileStep), chunks = kTileStep / chunk;  // tokens a copy, copies a step
    uint32_t n = 0;  // staged steps
    for (int64_t at = from; at < end;) {
      const KvTileUnit u = kv_tile_unit(a, prefix, at, end);
      at += u.taken;
      if (!u.work) continue;
      const int st_end = 2 * (u.t0 + u.tb);
      const int32_t* table = a.c.table + static_cast<int64_t>(u.b) * a.c.table_cols;  // (positions below len lie in it)
      auto wanted = [&](int st) { return lane < chunks && st < st_end && st * kTileStep + lane * chunk < u.sp.len; };
      auto entry_of = [&](int st) {
        uint32_t e = 0;
        ld_cg32_if(e, table + ((st * kTileStep + lane * chunk) >> lg), wanted(st));
        return e;
      };
      auto copy = [&](const int8_t* codes, int st, uint32_t entry, bool copies) {
        const uint32_t slot = n % P::kRing, bytes = chunk * kD;
        const int64_t src = (((static_cast<int64_t>(entry) * a.c.kv_heads + u.h) << lg) + (st * kTileStep & ((1 << lg) - 1))) * kD;
        if (n >= P::kRing) tile_wait(&ct->raw_empty[slot], n / P::kRing - 1, dead);
        const uint32_t count = __popc(__ballot_sync(0xffffffffu, copies));
        if (lane == 0) mbar_arrive_expect_tx(&ct->raw_full[slot], count * bytes);
        __syncwarp();
        if (copies && !dead) bulk_g2s(ring + slot * P::kRaw + lane * bytes, codes + src, bytes, &ct->raw_full[slot]);
        ++n;
      };
      int st = 2 * (u.t0 + u.ta);
      uint32_t next = entry_of(st), after = entry_of(st + 1);
      for (; st < st_end; ++st) {
        const uint32_t entry = next;
        next = after;
        after = entry_of(st + 2);
        const bool copies = wanted(st) && kv_page_ok(a.c, static_cast<int>(entry));
        copy(a.k, st, entry, copies);
        copy(a.v, st, entry, copies);
      }
    }
    bool late = false;  // no copy is in flight when the CTA ends
    for (uint32_t i = n > P::kRing ? n - P::kRing : 0; i < n; ++i) tile_wait(&ct->raw_full[i % P::kRing], i / P::kRing, late);
    } else if (warp == kTileMmaWarp + 3) {
    // ---------------------------------------------------------------- page scales
    // Of a step's four groups of 16 tokens (pages hold whole groups), read two steps ahead: lanes 0-3 K's, lanes 4-7 V's.
    // A page outside the cache (the copying warp records it) gets the scales 0 and log2 of 0: the logits of its tokens are
    // -inf whatever older codes the buffers hold for them.  K's buffer counts as filled when the scales are
    // there too: the softmax reads them once S is.  (Their slot was last read for the step eight before; the products with
    // K's buffer that are waited for here were issued after that step's weights had been used.)
    const int lg = a.c.log2_page;
    uint32_t steps = 0;
    for (int64_t at = from; at < end;) {
      const KvTileUnit u = kv_tile_unit(a, prefix, at, end);
      at += u.taken;
      if (!u.work) continue;
      const int st_end = 2 * (u.t0 + u.tb);
      const int32_t* table = a.c.table + static_cast<int64_t>(u.b) * a.c.table_cols;
      auto entry_of = [&](int st) {
        const int pos = st * kTileStep + (lane & 3) * 16;
        uint32_t e = 0xFFFFFFFFu;
        ld_cg32_if(e, table + (pos >> lg), st < st_end && pos < u.sp.len);
        return e;
      };
      auto scale_of = [&](uint32_t e) {
        uint32_t w = 0;
        ld_cg32_if(w, (lane < 4 ? a.ks : a.vs) + static_cast<int64_t>(static_cast<int>(e)) * a.c.kv_heads + u.h, lane < 8 && e < a.c.pages);
        return w;
      };
      int st = 2 * (u.t0 + u.ta);
      const uint32_t entry = entry_of(st);
      uint32_t scale = scale_of(entry), entry_next = entry_of(st + 1);
      bool here = entry < a.c.pages;
      for (; st < st_end; ++st, ++steps) {
        const uint32_t buf = steps % kTileBufs, use = steps / kTileBufs;
        if (use > 0) tile_wait(&ct->k_empty[buf], use - 1, dead);
        const float sv = __uint_as_float(scale);
        const uint32_t faint = __ballot_sync(0xffffffffu, sv < kKvLeast);
        if (lane < 4) {
          ct->scale_k[steps & 7][lane] = kv_finite(sv);
        } else if (lane < 8) {
          float av = kv_counts_as(sv), mul = 1.f;
          if (sv < kKvLeast) {  // its bits with kKvLeast's exponent, and the power of two that is missing
            const int up = -112 - (static_cast<int>(__float_as_uint(sv * 0x1p60f) >> 23) - 127 - 60);
            mul = sv == 0.f ? 0.f : pow2i(-up);
            if (sv != 0.f) av = sv * pow2i(up);
          }
          const float inv = __fdividef(kKvSum, av);
          ct->lv[steps & 7][lane & 3] = here ? kv_log2(sv, av) : -INFINITY;
          ct->inv_v[steps & 7][lane & 3] = (lane & 1) == 0 && (faint >> lane & 3) != 0 ? -inv : inv;
          ct->mul[steps & 7][lane & 3] = pack_f16x2(mul, mul);
        }
        scale = scale_of(entry_next);
        here = entry_next < a.c.pages;
        entry_next = entry_of(st + 2);
        __syncwarp();
        if (lane == 0) mbar_arrive(&ct->k_full[buf]);
      }
    }
    } else if (warp == kTileMmaWarp || warp == kTileMmaWarp + 2) {
    // ---------------------------------------------------------------- MMA issue, a warp per stream
    // The whole warp walks the stream's items and one elected lane issues.  What the operands depend on is broadcast, so
    // that the compiler knows it to be uniform: the MMAs take uniform registers, and moving each operand there costs more
    // than the products.
    constexpr uint32_t id_s = tc_idesc_f16(kTileRows, kTileStep, false), id_o = tc_idesc_f16(kTileRows, kD, true);
    const uint64_t q_desc = smem_desc_sw128(smem_u32(q_buf), 16, 1024), k_desc = smem_desc_sw128(smem_u32(k_buf), 16, 1024);
    const uint64_t v_desc = smem_desc_sw128(smem_u32(v_buf), P::kBlock, 1024);
    uint32_t steps = 0, done = 0, units = 0;  // of the units before: steps, items of a stream, units
    for (int64_t at = from; at < end;) {
      const KvTileUnit u = kv_tile_unit(a, prefix, at, end);
      at += u.taken;
      if (!u.work) continue;
      const int tiles = u.tb - u.ta, items = u.two ? 2 * tiles : tiles;
      tile_wait(&ct->q_full[units & 1], units >> 1, dead);
      ++units;
      auto run = [&](auto stream, auto two) {
        constexpr int s = decltype(stream)::value;
        constexpr bool both = decltype(two)::value;  // both streams take every step, else each every second
        auto score = [&](int i, uint32_t buf, uint32_t use) {  // S of item i, K in buffer buf, which is in its use-th use
          const uint32_t odd = __shfl_sync(0xffffffffu, (done + i) & 1, 0);
          buf = __shfl_sync(0xffffffffu, buf, 0);
          tile_wait(&ct->k_full[buf], use, dead);
          // The weights over this S are used: those of the item two before, of the last unit's too (its products with V were
          // issued after the last scores, which are all that q_full stands for).
          if (done + i > 1) tile_wait(&ct->pv_done[s][odd], (done + i - 2) >> 1, dead);
          tc_fence_after();
          if (elect_one()) {
            const uint64_t kd = k_desc + buf * (P::kOperand >> 4);
#pragma unroll
            for (int k = 0; k < kD / 16; ++k)
              tc_mma_ss(P::s_at(s, odd), q_desc + (((both && s == 1 ? P::kQTile : 0) + (k >> 2) * (kTileRows * 128) + (k & 3) * 32) >> 4),
                        kd + (((k >> 2) * P::kBlock + (k & 3) * 32) >> 4), id_s, k > 0);
            tc_commit(&ct->s_full[s][odd]);
            tc_commit(&ct->k_empty[buf]);
            if (!both) tc_commit(&ct->k_empty[buf]);  // for the other stream
            if (i == items - 1) tc_commit(&ct->q_free);
          }
          __syncwarp();
        };
        auto weigh = [&](int i, uint32_t buf, uint32_t use) {  // O of item i
          const uint32_t odd = __shfl_sync(0xffffffffu, (done + i) & 1, 0);
          buf = __shfl_sync(0xffffffffu, buf, 0);
          tile_wait(&ct->v_full[buf], use, dead);
          tile_wait(&ct->p_full[s][odd], (done + i) >> 1, dead);
          tc_fence_after();
          if (elect_one()) {
            const uint64_t vd = v_desc + buf * (P::kOperand >> 4);
#pragma unroll
            for (int k = 0; k < kTileStep / 16; ++k)
              tc_mma_ts(P::o_at(s), P::s_at(s, odd) + k * 8, vd + k * (2048 >> 4), id_o, k > 0 || i > 0);
            tc_commit(&ct->pv_done[s][odd]);
            tc_commit(&ct->v_empty[buf]);
            if (!both) tc_commit(&ct->v_empty[buf]);
          }
          __syncwarp();
        };
        const uint32_t st0 = steps + (both ? 0 : s);
        uint32_t buf = st0 % kTileBufs, use = st0 / kTileBufs;
        score(0, buf, use);
        for (int i = 0; i < items; ++i) {
          const uint32_t buf_v = buf, use_v = use;
          buf += both ? 1 : 2;
          if (buf >= kTileBufs) buf -= kTileBufs, ++use;
          if (i + 1 < items) score(i + 1, buf, use);
          weigh(i, buf_v, use_v);
        }
      };
      const std::integral_constant<int, 0> s0;
      const std::integral_constant<int, 1> s1;
      if (warp == kTileMmaWarp) {
        if (u.two) run(s0, std::true_type{}); else run(s0, std::false_type{});
      } else {
        if (u.two) run(s1, std::true_type{}); else run(s1, std::false_type{});
      }
      steps += 2 * tiles;
      done += items;
    }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTileSoftmaxRegs));
    // ---------------------------------------------------------------- softmax: two threads per row
    // Thread `half` of a row has 32 of a step's 64 scores and half of the row's q and O.  Four warps per scheduler: with one
    // thread per row (two warps), waits and tensor-memory latencies left the exp unit idle for two thirds of the time.
    const int s = warp >> 3, half = warp >> 2 & 1, row = tid & 127;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    // The two threads of a row are in warps w and w + 4 of the stream; a barrier of those two (64 threads) is enough.
    const int pair = 2 + s * 4 + (warp & 3);
    auto tell = [&](int place, float v) {  // place 1: maxima of items; 0: the end's sums
      ct->swap[place][s][half][row] = v;
      bar_sync(pair, 64);
      return ct->swap[place][s][half ^ 1][row];
    };
    uint32_t steps = 0, done = 0, units = 0;
    for (int64_t at = from; at < end;) {
      const KvTileUnit u = kv_tile_unit(a, prefix, at, end);
      at += u.taken;
      const int rr = u.rt * kTileUnitRows + (u.two ? s : 0) * kTileRows + row, r = rr / a.group;
      const bool on = r < u.sp.n, exists = r < a.R;
      auto out_row_of = [&] {
        const int rr = u.rt * kTileUnitRows + (u.two ? s : 0) * kTileRows + row, r = rr / a.group;
        return (static_cast<int64_t>(u.b) * a.R + r) * a.heads + u.h * a.group + (rr - r * a.group);
      };
      if (!u.work) {  // none of the unit's rows sees anything (or the slice ends before its tiles)
        if (u.mine && exists && (u.two || s == 0)) {
          const int64_t out_row = out_row_of();
          uint4* o = reinterpret_cast<uint4*>(a.o + out_row * kD) + half * (kD / 16);
          for (int i = 0; i < kD / 16; ++i) o[i] = make_uint4(0, 0, 0, 0);
          if (a.lse && half == 0) a.lse[out_row] = -INFINITY;
        }
        continue;
      }
      // Tokens that the row sees, from this half's first one of the slice on: first .. last - 1; all of the warp's rows see
      // all_first .. all_last - 1.
      const int base = (u.t0 + u.ta) * kTileTokens + half * 32, hi = u.sp.len - u.sp.n + r + 1;
      const int first = on && a.window > 0 ? max(0, hi - a.window) - base : -base, last = (on ? hi : u.sp.len) - base;
      const int all_first = __reduce_max_sync(0xffffffffu, first), all_last = __reduce_min_sync(0xffffffffu, last);
      tile_wait(&ct->q_full[units & 1], units >> 1, dead);
      const float qs = ct->row_scale[units & 1][u.two ? s : 0][row];
      ++units;
      const int tiles = u.tb - u.ta, items = u.two ? 2 * tiles : tiles;
      float m = -INFINITY, l = 0.f;
      const uint32_t to = P::o_at(s) + lane_off + half * (kD / 2);
      for (int i = 0; i < items; ++i) {
        const uint32_t g = done + i;
        const int st = u.two ? i : 2 * i + s, sl = (steps + st) & 7, g0 = half * 2;  // the half's first group of 16 tokens
        const int p0 = st * kTileStep;
        const uint32_t ts = P::s_at(s, g & 1) + lane_off;
        const bool whole = p0 >= all_first && p0 + 32 <= all_last;
        uint32_t bits = 0xFFFFFFFFu;  // bit i: token i of the half is seen
        if (!whole) {
          const int f = min(max(first - p0, 0), 32), n = min(max(last - p0, 0), 32);
          bits = n > f ? (0xFFFFFFFFu >> (32 - n)) & (0xFFFFFFFFu << f) : 0u;
        }
        tile_wait(&ct->s_full[s][g & 1], g >> 1, dead);
        tc_fence_after();
        uint32_t x[32];
        tmem_ld32(x, ts + half * 32);
        const float2 sk = *reinterpret_cast<const float2*>(&ct->scale_k[sl][g0]), lv2 = *reinterpret_cast<const float2*>(&ct->lv[sl][g0]);
        const float2 iv2 = *reinterpret_cast<const float2*>(&ct->inv_v[sl][g0]);
        const float cs[2] = {qs * sk.x, qs * sk.y}, lv[2] = {lv2.x, lv2.y}, iv[2] = {iv2.x, iv2.y};
        tmem_wait_ld(x);
        float mx = -INFINITY;
        auto largest = [&](auto cut) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float best = -INFINITY;
#pragma unroll
            for (int j = 0; j < 16; j += 2)
              best = fmaxf(best, fmaxf(!cut || bits >> (16 * k + j) & 1 ? __uint_as_float(x[16 * k + j]) : -INFINITY,
                                       !cut || bits >> (16 * k + j + 1) & 1 ? __uint_as_float(x[16 * k + j + 1]) : -INFINITY));
            if (!cut || bits >> (16 * k) & 0xFFFFu) mx = fmaxf(mx, fmaf(best, cs[k], lv[k]));
          }
        };
        if (whole) largest(std::false_type{}); else largest(std::true_type{});
        if (bar_any(pair, 64, mx > m + kTileGrow)) {  // a row's maximum moves: O and the sum shrink
          const float mn = fmaxf(m, fmaxf(mx, tell(1, mx))), f = mn == -INFINITY ? 1.f : ex2(m - mn);
          m = mn;
          l *= f;
          if (i > 0) {
            tile_wait(&ct->pv_done[s][(g - 1) & 1], (g - 1) >> 1, dead);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kD / 2; c += 8) {  // (rare: few registers and little code, or the loop around it pays)
              uint32_t y[8];
              tmem_ld8(y, to + c);
              tmem_wait_ld(y);
#pragma unroll
              for (int j = 0; j < 8; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * f);
              tmem_st8(to + c, y);
            }
          }
          tmem_ld32(x, ts + half * 32);  // (read again rather than kept over all this; weights go over them after both have)
          tmem_wait_ld(x);
          bar_sync(pair, 64);
        }
        const float top = m == -INFINITY ? 0.f : m - kTileTop;
        uint32_t w[16];
        auto weights = [&](auto cut) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint64_t lift = pack_f32x2(lv[k] - top, lv[k] - top), mul = pack_f32x2(cs[k], cs[k]);
            uint64_t sum = 0;
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float2 y = unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[16 * k + j]), __uint_as_float(x[16 * k + j + 1])), mul, lift));
              float w0 = ex2(y.x), w1 = ex2(y.y);
              if constexpr (cut) {
                w0 = bits >> (16 * k + j) & 1 ? w0 : 0.f;
                w1 = bits >> (16 * k + j + 1) & 1 ? w1 : 0.f;
              }
              sum = add_f32x2(sum, pack_f32x2(w0, w1));
              w[k * 8 + j / 2] = pack_f16x2(w0, w1);
            }
            if (!cut || bits >> (16 * k) & 0xFFFFu) l = fmaf(unpack_f32x2(sum).x + unpack_f32x2(sum).y, k == 0 ? fabsf(iv[k]) : iv[k], l);
          }
        };
        if (whole) weights(std::false_type{}); else weights(std::true_type{});
        if (iv[0] < 0.f) {
          const uint2 mul = *reinterpret_cast<const uint2*>(&ct->mul[sl][g0]);
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = hmul2_u32(w[i], i < 8 ? mul.x : mul.y);
        }
        tmem_st16(ts + half * 16, w);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ct->p_full[s][g & 1]);
      }
      steps += 2 * tiles;
      done += items;
      l += tell(0, l);  // (each of the two adds the other's: the same sum)
      tile_wait(&ct->pv_done[s][(done - 1) & 1], (done - 1) >> 1, dead);  // (the item two before is known to be done: S)
      tc_fence_after();

      // A unit that is cut leaves its pieces (O, maximum, sum) to the joining kernel.  One that is not is written here; with
      // one row tile, stream 0 adds stream 1's sums, which it reads from tensor memory.
      const bool cut_unit = u.tb - u.ta != u.tiles, joins = !cut_unit && !u.two;
      float f0 = 1.f, f1 = 0.f;
      if (joins) {
        if (s == 1 && half == 0) ct->hand[row] = make_float2(m, l);
        tc_fence_before();
        bar_sync(1, kTileSoftmax);
        tc_fence_after();
        if (s == 0) {
          const float2 o = ct->hand[row];
          const float mn = fmaxf(m, o.x);
          f0 = m == -INFINITY ? 0.f : ex2(m - mn), f1 = o.x == -INFINITY ? 0.f : ex2(o.x - mn);
          l = l * f0 + o.y * f1;
          m = mn;
        }
      }
      if (!(joins && s == 1)) {
        const int64_t out_row = out_row_of();
        const float inv = l == 0.f ? 0.f : 1.f / l;  // (kKvSum is taken out of the other factor: 1 / l may be large)
        const int64_t slot = kv_tile_slot(blockIdx.x, u.ta == 0, s);
#pragma unroll 1
        for (int c = 0; c < kD / 32; ++c) {
          uint32_t x[16];
          tmem_ld16(x, to + c * 16);
          tmem_wait_ld(x);
          if (cut_unit) {
            if (on) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                __stcg(a.part + (slot * (kD / 4) + half * (kD / 8) + c * 4 + i) * kTileRows + row,
                       make_float4(__uint_as_float(x[4 * i]), __uint_as_float(x[4 * i + 1]), __uint_as_float(x[4 * i + 2]), __uint_as_float(x[4 * i + 3])));
            }
          } else {
            if (joins) {
              uint32_t y[16];
              tmem_ld16(y, P::o_at(1) + lane_off + half * (kD / 2) + c * 16);
              tmem_wait_ld(y);
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f0 + __uint_as_float(y[i]) * f1);
            }
            if (exists) {
              uint2* o = reinterpret_cast<uint2*>(a.o + out_row * kD + half * (kD / 2) + c * 16);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                o[i] = on ? make_uint2(pack_bf16x2(__uint_as_float(x[4 * i]) * kKvSum * inv, __uint_as_float(x[4 * i + 1]) * kKvSum * inv),
                                       pack_bf16x2(__uint_as_float(x[4 * i + 2]) * kKvSum * inv, __uint_as_float(x[4 * i + 3]) * kKvSum * inv))
                          : make_uint2(0u, 0u);
            }
          }
        }
        if (half == 0) {
          if (cut_unit) __stcg(a.ml + slot * kTileRows + row, make_float2(m, l));
          else if (exists && a.lse) a.lse[out_row] = on && l != 0.f ? (m - kTileTop - kKvSumLog2 + lg2(l)) * 0.69314718055994531f : -INFINITY;
        }
      }
      tc_fence_before();
      if (joins) bar_sync(1, kTileSoftmax);  // (stream 1's sums have been read)
    }
  }
  __syncthreads();
  if (warp == kTileMmaWarp) {
    tc_fence_after();
    tmem_free(0, 512);
  }
}

// Joins the pieces that the tile kernel left, in the order of the tokens.  A launch of its own, after the tile kernel: joining
// inside it, by the CTA that finishes a unit last, took 9 us of its end (fence, counter, then one thread per row reading
// piece after piece).  A unit with few rows and many tokens has up to two pieces per CTA of the tile kernel, so the loads of
// many pieces have to be in flight at once: first the factors of up to kJoinChunk pieces, then the pieces.
// blockIdx = (kRows rows of a row tile, kv head, sequence); a thread takes one float4 of kD / 4 and every kBase-th row.
constexpr int kJoinThreads = 256, kJoinChunk = 32;
template <int kD, int kGroups>
struct KvJoinPlan {
  static constexpr int kVecs = kD / 4, kBase = kJoinThreads / kVecs, kRows = kBase * kGroups;
};
template <int kD, int kGroups>
__global__ void __launch_bounds__(kJoinThreads) kv_attention_join_kernel(const KvAttnArgs a, int grid) {
  using P = KvJoinPlan<kD, kGroups>;
  constexpr int kRows = P::kRows, kBase = P::kBase;
  extern __shared__ int prefix[];
  __shared__ float factor[kJoinChunk][kRows];
  __shared__ int scan[kJoinThreads / 32];
  __shared__ float2 part_ml[kJoinThreads / kRows][kRows];
  // (The lengths are older than the tile kernel, which begins only when its own predecessor is done.)
  const int64_t total = static_cast<int64_t>(kv_tile_prefix<kJoinThreads>(a, prefix, scan)) * a.c.kv_heads;
  const int64_t ctas = kv_tile_ctas(total, grid);
  const int tid = threadIdx.x, b = blockIdx.z, h = blockIdx.y, rr0 = blockIdx.x * kRows, rt = rr0 / kTileUnitRows;
  const KvSpan sp = kv_span(a, b);
  int t0 = 0, t1 = 0;
  const int before = kv_tile_cost_sum(a, sp, rt);
  kv_tile_range(a, sp, rt, t0, t1);
  const int tiles = max(1, t1 - t0);
  const int64_t begin = static_cast<int64_t>(prefix[b]) * a.c.kv_heads + static_cast<int64_t>(prefix[b + 1] - prefix[b]) * h + before;
  const int64_t first = begin + kTileUnitCost;  // of the unit's tiles
  const int64_t c0 = kv_div((first + 1) * ctas - 1, total), c1 = kv_div((first + tiles) * ctas - 1, total);
  const bool two = a.R * a.group - rt * kTileUnitRows > kTileRows;
  pdl_wait();
  pdl_launch_dependents();
  if (t1 <= t0 || c0 == c1) return;  // written by the tile kernel
  const int s0 = two ? rr0 % kTileUnitRows / kTileRows : 0, row0 = rr0 % kTileRows;
  const int pieces = static_cast<int>(c1 - c0 + 1) << (two ? 0 : 1);
  auto slot_of = [&](int p) { return two ? kv_tile_slot(c0 + p, p == 0, s0) : kv_tile_slot(c0 + (p >> 1), p < 2, p & 1); };

  // Maxima and factors: a thread takes a row and every kEvery-th piece.
  constexpr int kEvery = kJoinThreads / kRows;
  const int frow = tid % kRows, q = tid / kRows;
  const float2* ml0 = a.ml + row0 + frow;
  float m = -INFINITY, l = 0.f;
#pragma unroll 4
  for (int p = q; p < pieces; p += kEvery) m = fmaxf(m, ld_cg(ml0 + slot_of(p) * kTileRows).x);
  part_ml[q][frow].x = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEvery; ++i) m = fmaxf(m, part_ml[i][frow].x);

  const int c = tid / kBase, sub = tid % kBase;
  const float4* src = a.part + static_cast<int64_t>(c) * kTileRows + row0 + sub;
  float4 acc[kGroups];
#pragma unroll
  for (int j = 0; j < kGroups; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < pieces; p0 += kJoinChunk) {
    const int n = min(kJoinChunk, pieces - p0);
    __syncthreads();  // (the maxima, or the last factors, have been read)
#pragma unroll 4
    for (int p = q; p < n; p += kEvery) {
      const float2 ml = ld_cg(ml0 + slot_of(p0 + p) * kTileRows);
      const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
      factor[p][frow] = f;
      l = fmaf(ml.y, f, l);
    }
    __syncthreads();
#pragma unroll(8 / kGroups)
    for (int p = 0; p < n; ++p) {
      const float4* v0 = src + slot_of(p0 + p) * (P::kVecs * kTileRows);
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const float f = factor[p][sub + j * kBase];
        const float4 v = ld_cg(v0 + j * kBase);
        acc[j].x = fmaf(v.x, f, acc[j].x), acc[j].y = fmaf(v.y, f, acc[j].y);
        acc[j].z = fmaf(v.z, f, acc[j].z), acc[j].w = fmaf(v.w, f, acc[j].w);
      }
    }
  }
  part_ml[q][frow] = make_float2(m, l);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    const int row = sub + j * kBase, rr = rr0 + row, r = rr / a.group;
    if (r >= a.R) continue;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kEvery; ++i) sum += part_ml[i][row].y;
    const bool on = r < sp.n;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t out_row = (static_cast<int64_t>(b) * a.R + r) * a.heads + h * a.group + rr % a.group;
    reinterpret_cast<uint2*>(a.o + out_row * kD)[c] =
        on ? make_uint2(pack_bf16x2(acc[j].x * kKvSum * inv, acc[j].y * kKvSum * inv), pack_bf16x2(acc[j].z * kKvSum * inv, acc[j].w * kKvSum * inv))
           : make_uint2(0u, 0u);
    if (a.lse && c == 0) a.lse[out_row] = on && sum != 0.f ? (part_ml[0][row].x - kTileTop - kKvSumLog2 + lg2(sum)) * 0.69314718055994531f : -INFINITY;
  }
}

}  // namespace gguf_b200
