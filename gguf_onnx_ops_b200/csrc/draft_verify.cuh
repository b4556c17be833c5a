// Verification of drafted tokens against the target's probabilities, from given random numbers.
//   draft i of a sequence stands iff u_i q_i(x_i) < p_i(x_i)  (no q: u_i < p_i(x_i));  the first that does not ends the run
//   n = drafts that stand; the next token is drawn from w = max(p_n - q_n, 0) after a rejected draft (no q: p_n without
//   x_n), from w = p_n after a run that stands whole.
// The draw inverts the cumulative distribution in whole numbers: W_v = floor(min(w_v, 1) 2^38) (NaN counts as 0),
// T = sum W_v, target = floor(T floor(u 2^24) / 2^24), token = the lowest v with W_0 + .. + W_v > target.  Sums of whole
// numbers do not depend on their order, so however the row is cut the token is the same.  Where T is 0 the draw is
// made from p_n instead, and where that is empty too the token is -1.
//
// One cluster of up to eight CTAs per sequence: each sums its part of the row (two fp32 reads a token, nothing kept), the
// CTAs' totals meet through distributed shared memory, and the one warp whose stretch holds the target reads that stretch
// again (from the L2) to find the token.  Bound by memory for batches and by the chain of cluster barriers for one sequence
// (64 sequences of 7 drafts and 131072 tokens: 18 us, 3.7 TB/s, 13.4 where the L2 still holds the rows; one of 5 drafts and
// 32000 tokens: 5 us, of which a kernel that does nothing takes 2).  Rows that do not begin at 16 bytes are read 4 bytes a lane: 64
// sequences of 50257 tokens 14.9 us, of 50256 tokens 9.4.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"
#include "kv_cache.cuh"

namespace gguf_b200 {

struct DraftArgs {
  const float *p, *q;      // [B, R + 1, V], [B, R, V] or null
  const int32_t* draft;    // [B, R]
  const float *u, *us;     // [B, R], [B]
  const int32_t* drafts;   // [B] drafts of each sequence, or null: R
  int32_t *accepted, *tokens;  // [B], [B, R + 1]
  int R, V;
};

constexpr int kDraftCtas = 8;   // of a sequence, at most
constexpr int kDraftThreads = 512;
constexpr int kDraftWarps = kDraftThreads / 32;
constexpr int kDraftMax = 32;

constexpr int kDraftBatch = 4;  // steps whose loads are on their way at once

__device__ __forceinline__ float draft_weight(uint32_t p, uint32_t q) {
  return fminf(fmaxf(__fsub_rn(__uint_as_float(p), __uint_as_float(q)), 0.f), 1.f);  // NaN: 0
}
__device__ __forceinline__ unsigned long long draft_mass(float w) { return __float2ull_rz(w * 274877906944.0f); }

// kVec values per lane and load (4 needs V % 4 == 0 and 16-byte aligned rows).
template <int kVec>
__global__ void __launch_bounds__(kDraftThreads, 2) draft_verify_kernel(const DraftArgs a) {
  namespace cg = cooperative_groups;
  __shared__ unsigned long long warp_sum[kDraftWarps], cta_sum[2];
  pdl_wait();
  pdl_launch_dependents();
  auto cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
  const int b = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_drafts = a.drafts ? max(0, min(a.R, ld_cg(a.drafts + b))) : a.R;
  const int64_t V = a.V;

  // Every warp decides the run by itself: lane i looks at draft i.
  bool stands = false;
  int x = -1;
  if (lane < n_drafts) {
    x = ld_cg(a.draft + static_cast<int64_t>(b) * a.R + lane);
    if (x >= 0 && x < a.V) {
      const float p = ld_cg(a.p + (static_cast<int64_t>(b) * (a.R + 1) + lane) * V + x);
      const float q = a.q ? ld_cg(a.q + (static_cast<int64_t>(b) * a.R + lane) * V + x) : 1.f;
      stands = __fmul_rn(ld_cg(a.u + static_cast<int64_t>(b) * a.R + lane), q) < p;
    }
  }
  const int n = __ffs(~__ballot_sync(0xffffffffu, stands)) - 1 < 0 ? 32 : __ffs(~__ballot_sync(0xffffffffu, stands)) - 1;
  const bool rejected = n < n_drafts;
  const int x_n = __shfl_sync(0xffffffffu, x, n & 31);
  if (rank == 0 && warp == 0) {
    if (lane == 0) a.accepted[b] = n;
    for (int i = lane; i <= a.R; i += 32)
      if (i != n) a.tokens[static_cast<int64_t>(b) * (a.R + 1) + i] = i < n ? x : -1;
  }

  const float* p = a.p + (static_cast<int64_t>(b) * (a.R + 1) + n) * V;
  const float* q = rejected && a.q ? a.q + (static_cast<int64_t>(b) * a.R + n) * V : nullptr;
  const int skip = rejected && !a.q ? x_n : -1;  // the token a certain draft takes out of the row
  // The row in warp stretches of whole 32 kVec-value steps.
  const int step = 32 * kVec, steps = (a.V + step - 1) / step, all_warps = ctas * kDraftWarps;
  const int w_id = rank * kDraftWarps + warp;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * w_id / all_warps);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (w_id + 1) / all_warps);
  // w of this lane's values of kDraftBatch steps from s on (0 past the warp's stretch).
  auto weights = [&](int s, bool with_q, float (&w)[kDraftBatch][kVec]) {
    alignas(16) uint32_t pw[kDraftBatch][kVec] = {}, qw[kDraftBatch][kVec] = {};
#pragma unroll
    for (int k = 0; k < kDraftBatch; ++k) {
      const int v = (s + k) * step + lane * kVec;
      const bool in = s + k < s1 && v < a.V;
      if constexpr (kVec == 4) {
        ld_cg128_if(*reinterpret_cast<uint4*>(pw[k]), p + v, in);
        ld_cg128_if(*reinterpret_cast<uint4*>(qw[k]), q + v, in && q && with_q);
      } else {
        ld_cg32_if(pw[k][0], p + v, in);
        ld_cg32_if(qw[k][0], q + v, in && q && with_q);
      }
    }
#pragma unroll
    for (int k = 0; k < kDraftBatch; ++k)
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        w[k][i] = with_q && (s + k) * step + lane * kVec + i == skip ? 0.f : draft_weight(pw[k][i], qw[k][i]);
  };

  int token = -1;
  bool mine = false;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {  // pass 1: the residual is empty, draw from p_n
    const bool with_q = pass == 0;
    unsigned long long sum = 0;
    for (int s = s0; s < s1; s += kDraftBatch) {
      float w[kDraftBatch][kVec];
      weights(s, with_q, w);
#pragma unroll
      for (int k = 0; k < kDraftBatch; ++k)
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum += draft_mass(w[k][i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      unsigned long long c = 0;
      for (int w = 0; w < kDraftWarps; ++w) c += warp_sum[w];
      cta_sum[pass] = c;
    }
    cluster.sync();
    unsigned long long total = 0, before = 0;
    for (int r = 0; r < ctas; ++r) {
      const unsigned long long c = *cluster.map_shared_rank(&cta_sum[pass], r);
      total += c;
      if (r < rank) before += c;
    }
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    if (total == 0) {
      mine = rank == 0 && warp == 0 && lane == 0;
      __syncthreads();  // warp_sum is written again
      continue;
    }
    const float uf = ld_cg(a.us + b) * 16777216.0f;
    const unsigned long long u = static_cast<unsigned long long>(fminf(fmaxf(uf, 0.f), 16777215.0f));
    const unsigned long long target = (total >> 24) * u + (((total & 0xFFFFFFull) * u) >> 24);
    mine = false;
    if (before <= target && target < before + sum) {  // in this warp's stretch
      unsigned long long run = before;
      bool found = false;
      for (int s = s0; s < s1 && !found; s += kDraftBatch) {
        float w[kDraftBatch][kVec];
        weights(s, with_q, w);
#pragma unroll
        for (int k = 0; k < kDraftBatch; ++k) {
          if (found) continue;
          unsigned long long c = 0;
#pragma unroll
          for (int i = 0; i < kVec; ++i) c += draft_mass(w[k][i]);
          unsigned long long incl = c;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
          }
          const unsigned hit = __ballot_sync(0xffffffffu, run + incl > target);
          if (hit) {
            found = true;
            mine = lane == __ffs(hit) - 1;
            unsigned long long low = run + incl - c;
            bool past = false;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
              low += draft_mass(w[k][i]);
              if (!past && low > target) token = (s + k) * step + lane * kVec + i, past = true;
            }
          }
          run += __shfl_sync(0xffffffffu, incl, 31);
        }
      }
    }
    break;
  }
  if (mine) a.tokens[static_cast<int64_t>(b) * (a.R + 1) + n] = token;
  cluster.sync();  // no CTA leaves while another may still read its sum
}

}  // namespace gguf_b200
