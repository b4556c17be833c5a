// C ABI of the attention side of a decode / verify step (include/gguf_ops.h): head norms with the position
// rotation, the 8-bit paged KV cache, attention over it, and the verification of drafted tokens.  Every entry
// validates its arguments, picks a kernel by sizes alone and enqueues it on the caller's stream; nothing is allocated.
#include <atomic>
#include <algorithm>
#include <string>
#include <type_traits>

#include "host.cuh"
#include "qk_norm_rope.cuh"
#include "kv_cache.cuh"
#include "kv_attention.cuh"
#include "kv_attention_tile.cuh"
#include "draft_verify.cuh"

namespace gguf_b200 {

cudaError_t kv_device_error(int* error, int* site) {
  const int zero = 0;
  cudaError_t e;
  if ((e = cudaMemcpyFromSymbol(error, g_dev_error, sizeof(int))) != cudaSuccess) return e;
  if ((e = cudaMemcpyFromSymbol(site, g_dev_error_site, sizeof(int))) != cudaSuccess) return e;
  if ((e = cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(int))) != cudaSuccess) return e;
  return cudaMemcpyToSymbol(g_dev_error_site, &zero, sizeof(int));
}

namespace {

constexpr int64_t kMaxGridZ = 65535;

int invalid(const char* op, const std::string& what) {
  return set_error(GGUF_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

bool known_dim(int64_t d) { return d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// The cache, its table and the batch that an op is given.
int check_cache(const char* op, const GgufKvCache* c, const int32_t* table, const int32_t* lens, int64_t B,
                int64_t table_cols, KvPages* out) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || (B > 0 && (!table || !lens))) return invalid(op, "null tensor pointer");
  if (!known_dim(c->head_dim)) return invalid(op, "head_dim must be 64, 96, 128, 192 or 256");
  if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1))) return invalid(op, "page must be 16, 32, 64, 128 or 256 tokens");
  if (c->kv_heads < 1 || c->kv_heads > kMaxGridZ) return invalid(op, "bad number of kv heads");
  if (c->pages < 1 || c->pages >= (1ll << 31)) return invalid(op, "bad number of pages");
  if (B < 0 || B > kMaxGridZ) return invalid(op, "batch must be in [0, 65535]");
  if (table_cols < 1 || table_cols * c->page >= (1ll << 31)) return invalid(op, "bad page table width");
  if (!is_aligned(c->k, 16) || !is_aligned(c->v, 16)) return invalid(op, "cache tensors must be 16-byte aligned");
  int lg = 4;
  while ((1ll << lg) < c->page) ++lg;
  *out = KvPages{table, c->pages, static_cast<int>(table_cols), static_cast<int>(c->kv_heads), lg, static_cast<int>(c->head_dim)};
  return GGUF_OK;
}

// Calls f with the head width as a constant.
template <typename F>
auto by_dim(int64_t D, F&& f) {
  switch (D) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 96: return f(std::integral_constant<int, 96>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 192: return f(std::integral_constant<int, 192>{});
    default: return f(std::integral_constant<int, 256>{});
  }
}

template <int kGL, int kHeads>
cudaError_t run_rope(const RopeArgs& a, bool interleaved, cudaStream_t s) {
  const int64_t parts = (a.heads + kHeads - 1) / kHeads + (a.kv_heads + kHeads - 1) / kHeads;
  const int64_t per = kRopeThreads / kGL, blocks = (a.T * parts + per - 1) / per;
  const dim3 grid(static_cast<unsigned>(blocks)), block(kRopeThreads);
  return interleaved ? launch_kernel(qk_norm_rope_kernel<kGL, kHeads, true>, grid, block, 0, s, a)
                     : launch_kernel(qk_norm_rope_kernel<kGL, kHeads, false>, grid, block, 0, s, a);
}

// How a call's rows (query tokens x heads of one kv head) are taken: 8 or 16 at a time by the streaming kernel, or 256 at a
// time by the tile kernel, when there are many rows and much work: the streaming kernel reads a cache once per 16 rows, the
// tile kernel costs 20 us in any case (two launches, a pipeline to fill).  Work is what the streaming kernel's line would
// hold at most, from the page table's width and the window: lengths are on the device.
// Streaming / tile in us, 8 kv heads, 16 sequences of 801 to 9001 tokens, and one of 65001:
//   128 values: 16 rows 60 / 79, 58 / 70; 24 rows 101 / 79, 86 / 71; 48 rows 144 / 82, 117 / 73
//   64 values: 16 rows 36 / 68, 34 / 61; 32 rows 58 / 68, 47 / 61; 48 rows 81 / 68, 62 / 61; 96 rows 148 / 71, 106 / 62
// and by work, in tiles of the line per SM:
//   128 values: 128 rows, 3201 tokens (100) 29 / 29; 512 rows, 801 tokens (143) 32 / 37; 128 rows, 6401 tokens (187) 41 / 32;
//   512 rows, 1601 tokens (230) 44 / 38
//   64 values: 128 rows, 6401 tokens (187) 25 / 26; 512 rows, 1601 tokens (230) 28 / 32; 16 sequences, 128 rows, 201 tokens (311)
//   32 / 18; 512 rows, 3201 tokens (400) 39 / 34
// 8 rows of 128 values taken as 16: 57 -> 84 us (one sequence of 131071 tokens).
struct AttentionPlan {
  bool tile;
  int rows;            // of a unit
  int64_t row_tiles;   // units per kv head
};
int64_t tile_work(int64_t D, int sms) { return sms * (D == 64 ? 250ll : 150ll); }
bool tile_rows(int64_t B, int64_t rows, int64_t D) { return ((D == 64 && rows > 32) || (D == 128 && rows > 16)) && B <= kTileMaxBatch; }
AttentionPlan stream_plan(int64_t rows) {
  const int unit = rows <= 8 ? 8 : 16;
  return {false, unit, (rows + unit - 1) / unit};
}
AttentionPlan attention_plan(int64_t B, int64_t rows, int64_t D, int64_t kv_heads, int64_t positions, int sms) {
  const AttentionPlan p = stream_plan(rows);
  const int64_t per_unit = (positions + kKvTile - 1) / kKvTile + kKvUnitCost;
  if (!tile_rows(B, rows, D) || B * kv_heads * p.row_tiles < tile_work(D, sms) / per_unit) return p;
  return {true, kTileUnitRows, (rows + kTileUnitRows - 1) / kTileUnitRows};
}

template <typename Kernel>
int raise_smem(Kernel kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_cuda_error("KvCacheAttention", e);
  if (!(done.load() >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return set_cuda_error("KvCacheAttention", e);
    done.fetch_or(1ull << (dev & 63));
  }
  return GGUF_OK;
}

// The streaming kernel for heads of kD values and kNT * 8 rows a unit.
template <int kD, int kNT>
struct Stream {
  using P = KvAttnPlan<kD, kNT>;
  static int64_t part_bytes(int sms) { return 2ll * sms * P::kCtas * P::kFrags * 32 * 16; }
  static int64_t ml_bytes(int sms) { return 2ll * sms * P::kCtas * P::kRows * 8; }
  static int run(const KvAttnArgs& a, int sms, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    static_assert(P::smem(kKvMaxBatch) <= 227 * 1024, "shared memory");
    if (int rc = raise_smem(kv_attention_kernel<kD, kNT>, P::smem(kKvMaxBatch), done)) return rc;
    cudaError_t e = launch_kernel(kv_attention_kernel<kD, kNT>, dim3(static_cast<unsigned>(sms * P::kCtas)), dim3(kKvThreads),
                                  P::smem(a.B), s, a);
    return e == cudaSuccess ? GGUF_OK : set_cuda_error("KvCacheAttention launch", e);
  }
};
// The tile kernel.
template <int kD>
struct Tile {
  using P = KvTilePlan<kD>;
  template <int kGroups>
  static cudaError_t join(const KvAttnArgs& a, int sms, cudaStream_t s) {
    using J = KvJoinPlan<kD, kGroups>;
    const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(a.R) * a.group + J::kRows - 1) / J::kRows), static_cast<unsigned>(a.c.kv_heads), static_cast<unsigned>(a.B));
    return launch_kernel(kv_attention_join_kernel<kD, kGroups>, grid, dim3(kJoinThreads), (a.B + 1) * sizeof(int), s, a, sms);
  }
  static int64_t part_bytes(int sms) { return 4ll * sms * kTileRows * kD * 4; }
  static int64_t ml_bytes(int sms) { return 4ll * sms * kTileRows * 8; }
  static int run(const KvAttnArgs& a, int sms, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    static std::atomic<int> regs{0};
    if (!regs.load()) {  // the kernel's warp groups share out what it is launched with
      cudaFuncAttributes f;
      cudaError_t e = cudaFuncGetAttributes(&f, kv_attention_tile_kernel<kD>);
      if (e != cudaSuccess) return set_cuda_error("KvCacheAttention", e);
      if (f.numRegs < kTileLaunchRegs) return set_error(GGUF_ERR_CUDA, "KvCacheAttention: built with too few registers");
      regs.store(f.numRegs);
    }
    if (int rc = raise_smem(kv_attention_tile_kernel<kD>, P::smem(kTileMaxBatch), done)) return rc;
    cudaError_t e = launch_kernel(kv_attention_tile_kernel<kD>, dim3(static_cast<unsigned>(sms)), dim3(kTileThreads), P::smem(a.B), s, a);
    if (e != cudaSuccess) return set_cuda_error("KvCacheAttention launch", e);
    // The join's blocks: few rows each while that leaves them in one wave (eight an SM), four times as many after that.
    const int64_t few = (static_cast<int64_t>(a.R) * a.group + KvJoinPlan<kD, 1>::kRows - 1) / KvJoinPlan<kD, 1>::kRows * a.c.kv_heads * a.B;
    e = few <= 8ll * sms ? join<1>(a, sms, s) : join<4>(a, sms, s);
    return e == cudaSuccess ? GGUF_OK : set_cuda_error("KvCacheAttention launch", e);
  }
};

// Calls f with the kernel of a plan.
template <typename F>
auto attention_dispatch(const AttentionPlan& p, int64_t D, F&& f) {
  if (p.tile) return D == 64 ? f(Tile<64>{}) : f(Tile<128>{});
  const bool one = p.rows == 8;
  switch (D) {
    case 64: return one ? f(Stream<64, 1>{}) : f(Stream<64, 2>{});
    case 96: return one ? f(Stream<96, 1>{}) : f(Stream<96, 2>{});
    case 128: return one ? f(Stream<128, 1>{}) : f(Stream<128, 2>{});
    case 192: return one ? f(Stream<192, 1>{}) : f(Stream<192, 2>{});
    default: return one ? f(Stream<256, 1>{}) : f(Stream<256, 2>{});
  }
}

int attention_shape(const char* op, int64_t B, int64_t R, int64_t heads, int64_t kv_heads) {
  if (B < 0 || B > kKvMaxBatch) return invalid(op, "batch must be in [0, 4096]");
  if (R < 0 || R > (1 << 24)) return invalid(op, "bad number of rows");
  if (kv_heads < 1 || heads < 1 || heads > (1 << 16) || heads % kv_heads != 0) return invalid(op, "heads must be a multiple of kv heads");
  return GGUF_OK;
}

}  // namespace
}  // namespace gguf_b200

using namespace gguf_b200;

extern "C" {

int gguf_qk_norm_rope(const void* x, const float* gamma_q, const float* gamma_k, const float* cos_table,
                      const float* sin_table, const int32_t* positions, void* q, void* k, int64_t T, int64_t row_stride,
                      int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rot, int64_t max_pos, float eps,
                      int interleaved, void* stream) {
  clear_error();
  const char* op = "QkNormRope";
  if (head_dim < 8 || head_dim > 256 || head_dim % 8 != 0) return invalid(op, "head_dim must be a multiple of 8 in [8, 256]");
  if (rot < 0 || rot > head_dim || rot % 8 != 0) return invalid(op, "the rotated width must be a multiple of 8 in [0, head_dim]");
  if (heads < 1 || kv_heads < 1 || heads > (1 << 16) || kv_heads > (1 << 16)) return invalid(op, "bad number of heads");
  if (T < 0 || T > (1ll << 31) / (heads + kv_heads)) return invalid(op, "bad number of tokens");
  if (row_stride < 0 || row_stride % 4 != 0) return invalid(op, "rows must start at multiples of 4 values");
  if (T == 0) return GGUF_OK;
  if (!x || !q || !k || (rot > 0 && (!cos_table || !sin_table || !positions))) return invalid(op, "null tensor pointer");
  if (rot > 0 && (max_pos < 1 || max_pos >= (1ll << 31))) return invalid(op, "bad number of table rows");
  if (!is_aligned(x, 8) || !is_aligned(q, 16) || !is_aligned(k, 16)) return invalid(op, "x must be 8-byte aligned, outputs 16-byte");
  for (const float* f : {gamma_q, gamma_k, cos_table, sin_table})
    if (f && !is_aligned(f, 16)) return invalid(op, "gamma and the tables must be 16-byte aligned");
  int sms = 0, rc;
  if ((rc = device_sms(&sms))) return rc;
  const RopeArgs a{static_cast<const bf16*>(x), gamma_q, gamma_k, cos_table, sin_table, positions, static_cast<bf16*>(q),
                   static_cast<bf16*>(k), row_stride, T, static_cast<int>(heads), static_cast<int>(kv_heads),
                   static_cast<int>(head_dim), static_cast<int>(rot), static_cast<int>(max_pos), eps};
  auto* s = static_cast<cudaStream_t>(stream);
  // One head per lane group while the call does not fill the GPU, four after that (their loads overlap, and cos, sin and
  // gamma are read once for the four).  40 heads of 128, one / four, in us: 1 token 1.8 / 2.4, 128 tokens 2.4 / 2.6, 256 tokens
  // 3.2 / 2.9, 8191 tokens 43 / 33.
  const int lanes = head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32;
  const bool few = T * (heads + kv_heads) * lanes <= static_cast<int64_t>(sms) * 1024;
  const bool in = interleaved != 0;
  cudaError_t e;
  if (lanes == 8) e = few ? run_rope<8, 1>(a, in, s) : run_rope<8, 4>(a, in, s);
  else if (lanes == 16) e = few ? run_rope<16, 1>(a, in, s) : run_rope<16, 4>(a, in, s);
  else e = few ? run_rope<32, 1>(a, in, s) : run_rope<32, 4>(a, in, s);
  return e == cudaSuccess ? GGUF_OK : set_cuda_error("QkNormRope launch", e);
}

int gguf_kv_cache_write(const GgufKvCache* cache, const void* k, const void* v, const int32_t* table,
                        const int32_t* lens, const int32_t* new_lens, int64_t B, int64_t R, int64_t table_cols,
                        int64_t k_stride_b, int64_t k_stride_r, int64_t v_stride_b, int64_t v_stride_r, void* stream) {
  clear_error();
  const char* op = "KvCacheWrite";
  KvWriteArgs a{};
  if (int rc = check_cache(op, cache, table, lens, B, table_cols, &a.c)) return rc;
  if (R < 0 || R >= (1ll << 30)) return invalid(op, "bad number of rows");
  if (B == 0 || R == 0) return GGUF_OK;
  if (!k || !v) return invalid(op, "null tensor pointer");
  if (!is_aligned(k, 16) || !is_aligned(v, 16) || k_stride_b % 8 || k_stride_r % 8 || v_stride_b % 8 || v_stride_r % 8)
    return invalid(op, "k and v must be 16-byte aligned with strides in multiples of 8 values");
  a.x[0] = static_cast<const bf16*>(k), a.x[1] = static_cast<const bf16*>(v);
  a.codes[0] = static_cast<int8_t*>(cache->k), a.codes[1] = static_cast<int8_t*>(cache->v);
  a.scales[0] = cache->k_scale, a.scales[1] = cache->v_scale;
  a.lens = lens, a.news = new_lens;
  a.stride_b[0] = k_stride_b, a.stride_b[1] = v_stride_b, a.stride_r[0] = k_stride_r, a.stride_r[1] = v_stride_r;
  a.R = static_cast<int>(R);
  const int64_t touched = (R + cache->page - 2) / cache->page + 1;  // pages that R tokens can lie in
  cudaError_t e = by_dim(cache->head_dim, [&](auto d) {
    return launch_kernel(kv_write_kernel<d.value>,
                         dim3(static_cast<unsigned>(touched * 2), static_cast<unsigned>(cache->kv_heads), static_cast<unsigned>(B)),
                         dim3(kKvWriteThreads), 0, static_cast<cudaStream_t>(stream), a);
  });
  return e == cudaSuccess ? GGUF_OK : set_cuda_error("KvCacheWrite launch", e);
}

int gguf_kv_cache_read(const GgufKvCache* cache, const int32_t* table, const int32_t* lens, void* k, void* v, int64_t B,
                       int64_t rows, int64_t table_cols, void* stream) {
  clear_error();
  const char* op = "KvCacheRead";
  KvReadArgs a{};
  if (int rc = check_cache(op, cache, table, lens, B, table_cols, &a.c)) return rc;
  if (rows < 0 || rows >= (1ll << 31)) return invalid(op, "bad number of rows");
  if (B == 0 || rows == 0) return GGUF_OK;
  if (!k || !v) return invalid(op, "null tensor pointer");
  if (!is_aligned(k, 32) || !is_aligned(v, 32)) return invalid(op, "outputs must be 32-byte aligned");
  a.codes[0] = static_cast<const int8_t*>(cache->k), a.codes[1] = static_cast<const int8_t*>(cache->v);
  a.scales[0] = cache->k_scale, a.scales[1] = cache->v_scale;
  a.y[0] = static_cast<bf16*>(k), a.y[1] = static_cast<bf16*>(v);
  a.lens = lens, a.rows = static_cast<int>(rows);
  const int64_t pieces = rows * cache->kv_heads * (cache->head_dim / 16), per_block = kKvReadThreads * kKvReadPieces;
  if (pieces >= (1ll << 31)) return invalid(op, "too many rows");
  cudaError_t e = by_dim(cache->head_dim, [&](auto d) {
    return launch_kernel(kv_read_kernel<d.value>, dim3(static_cast<unsigned>((pieces + per_block - 1) / per_block), 2, static_cast<unsigned>(B)),
                         dim3(kKvReadThreads), 0, static_cast<cudaStream_t>(stream), a);
  });
  return e == cudaSuccess ? GGUF_OK : set_cuda_error("KvCacheRead launch", e);
}

int gguf_kv_cache_attention_workspace(int64_t B, int64_t R, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                      int64_t* bytes, int64_t* counters) {
  clear_error();
  const char* op = "KvCacheAttention";
  if (!bytes || !counters) return invalid(op, "null pointer");
  if (int rc = attention_shape(op, B, R, heads, kv_heads)) return rc;
  if (!known_dim(head_dim)) return invalid(op, "head_dim must be 64, 96, 128, 192 or 256");
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  auto bytes_of = [&](const AttentionPlan& p) {
    return attention_dispatch(p, head_dim, [&](auto k) { return k.part_bytes(sms) + k.ml_bytes(sms); });
  };
  const int64_t rows = R * (heads / kv_heads);
  const AttentionPlan p = stream_plan(rows);
  *bytes = bytes_of(p);
  *counters = B * kv_heads * p.row_tiles;  // one per unit
  if (tile_rows(B, rows, head_dim)) {  // either kernel, by the width of the page table; the tile kernel needs no counters
    *bytes = std::max(*bytes, bytes_of({true, kTileUnitRows, 1}));
    *counters = std::min(*counters, tile_work(head_dim, sms));
  }
  return GGUF_OK;
}

int gguf_kv_cache_attention(const GgufKvCache* cache, const void* q, const int32_t* table, const int32_t* lens,
                            const int32_t* new_lens, void* out, float* lse, void* workspace, int32_t* counters, int64_t B,
                            int64_t R, int64_t heads, int64_t table_cols, int64_t q_stride_b, int64_t q_stride_r,
                            float scale, int64_t window, void* stream) {
  clear_error();
  const char* op = "KvCacheAttention";
  KvAttnArgs a{};
  if (int rc = check_cache(op, cache, table, lens, B, table_cols, &a.c)) return rc;
  if (int rc = attention_shape(op, B, R, heads, cache->kv_heads)) return rc;
  if (window < 0) return invalid(op, "window must be >= 0 (0: none)");
  if (!(scale > -INFINITY && scale < INFINITY)) return invalid(op, "scale must be finite");
  if (B == 0 || R == 0) return GGUF_OK;
  if (!q || !out || !workspace || !counters) return invalid(op, "null tensor pointer");
  if (!is_aligned(q, 16) || !is_aligned(out, 16) || !is_aligned(workspace, 16) || q_stride_b % 8 || q_stride_r % 8)
    return invalid(op, "tensors must be 16-byte aligned with strides in multiples of 8 values");
  const int64_t group = heads / cache->kv_heads, rows = R * group;
  const int64_t width = table_cols << a.c.log2_page, positions = window > 0 ? std::min(width, window + R) : width;
  if (rows >= (1ll << 31)) return invalid(op, "too many rows");
  // The kernels sum the line's tiles of all sequences (the tile kernel: of all their row tiles) in 32 bits.
  const int64_t line = B * (positions / kKvTile + 2 + kKvUnitCost);
  const int64_t tile_line = B * ((rows + kTileUnitRows - 1) / kTileUnitRows) * (positions / kTileTokens + 2 + kTileUnitCost);
  if (line >= (1ll << 31) || (tile_rows(B, rows, cache->head_dim) && tile_line >= (1ll << 31)))
    return invalid(op, "too many positions in all (a narrower page table, or fewer sequences or rows a call)");
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  const AttentionPlan p = attention_plan(B, rows, cache->head_dim, cache->kv_heads, positions, sms);
  if (B * cache->kv_heads * p.row_tiles >= (1ll << 31)) return invalid(op, "too many rows");
  a.k = static_cast<const int8_t*>(cache->k), a.v = static_cast<const int8_t*>(cache->v);
  a.ks = cache->k_scale, a.vs = cache->v_scale;
  a.q = static_cast<const bf16*>(q), a.o = static_cast<bf16*>(out), a.lse = lse;
  a.lens = lens, a.news = new_lens;
  a.q_stride_b = q_stride_b, a.q_stride_r = q_stride_r;
  a.scale_log2 = scale * 1.44269504088896341f;
  a.B = static_cast<int>(B), a.R = static_cast<int>(R), a.heads = static_cast<int>(heads), a.group = static_cast<int>(group);
  a.window = static_cast<int>(std::min<int64_t>(window, 0x7fffffff));
  a.row_tiles = static_cast<int>(p.row_tiles);
  a.counters = counters;
  return attention_dispatch(p, cache->head_dim, [&](auto k) {
    a.part = static_cast<float4*>(workspace);
    a.ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + k.part_bytes(sms));
    return k.run(a, sms, static_cast<cudaStream_t>(stream));
  });
}

int gguf_draft_verify(const float* target, const float* draft_probs, const int32_t* draft, const float* u_accept,
                      const float* u_sample, const int32_t* drafts, int32_t* accepted, int32_t* tokens, int64_t B,
                      int64_t R, int64_t V, void* stream) {
  clear_error();
  const char* op = "DraftVerify";
  if (R < 1 || R > kDraftMax) return invalid(op, "drafted tokens must be in [1, 32]");
  if (V < 1 || V > (1 << 24)) return invalid(op, "vocabulary must be in [1, 2^24]");
  if (B < 0 || B > (1 << 20)) return invalid(op, "bad batch");
  if (B == 0) return GGUF_OK;
  if (!target || !draft || !u_accept || !u_sample || !accepted || !tokens) return invalid(op, "null tensor pointer");
  const DraftArgs a{target, draft_probs, draft, u_accept, u_sample, drafts, accepted, tokens, static_cast<int>(R), static_cast<int>(V)};
  const bool wide = V % 4 == 0 && is_aligned(target, 16) && (!draft_probs || is_aligned(draft_probs, 16));
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  // A sequence's row is shared by as many CTAs (8 at most) as keep the whole call in one wave of two an SM.  8 / 4 / 2 / 1 CTAs, in
  // us, rows from memory: 131072 tokens, 16 sequences 8.1 / 10.1 / 16.3 / 28.4, 64 sequences 21.1 / 17.9 / 22.6 / 35.5; 32000
  // tokens, 256 sequences 50.2 / 26.0 / 18.7 / 15.7.  (64 sequences whose rows the L2 still holds: 17.5 / 13.3 / 17.2 / 31.5.)
  int ctas = kDraftCtas;
  while (ctas > 1 && B * ctas > 2 * sms) ctas /= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B * ctas));
  cfg.blockDim = dim3(kDraftThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, wide ? draft_verify_kernel<4> : draft_verify_kernel<1>, a);
  return e == cudaSuccess ? GGUF_OK : set_cuda_error("DraftVerify launch", e);
}

}  // extern "C"
