// K9 — moves of cache pages (blocks) inside the pool.
//
// b2p_copy_blocks copies block src[i] to block dst[i] in every layer of K and V (with the
// scales of an 8-bit pool) in one launch: what a forked sequence needs for its last, partly
// filled block before it writes on (full blocks are shared by reference count).
//
// b2p_compact_blocks packs the live blocks (those that the used part of a block table names)
// into the pool's first num_live blocks. Only blocks that sit at or past num_live move: the
// j-th of them, in ascending order, goes to the j-th free block below num_live, so every
// source is live and every target free, no block is both, and all moves are independent.
//   1. mark: one bit per live block (atomic ORs: the result does not depend on their order);
//   2. plan: one CTA counts the bits, pairs sources with targets and writes new_ids;
//   3. move: all SMs copy the pairs over all layers, and rewrite the block tables.
// One CTA does 1 and 2 on bits in shared memory where the tables are small enough for it.
// Both are bound by HBM: each moved byte is read once and written once.
#include "common.cuh"

namespace {

using namespace b2p;

// One page is block_bytes contiguous bytes in each layer of K and of V.
struct Pages {
  uint8_t* cache[2];
  float* scales[2];  // null: no scales
  int64_t block_bytes;
  int64_t num_blocks, num_layers;
  int hkv;
};

constexpr int kCopyThreads = 128;
constexpr int kCopyUnroll = 4;

// One CTA: block src to block dst in one layer of K (kv 0) or V (kv 1).
template <typename V>
__device__ __forceinline__ void copy_page(const Pages& g, int64_t src, int64_t dst, int64_t layer,
                                          int kv) {
  const int64_t n = g.block_bytes / (int64_t)sizeof(V);
  const int64_t base = layer * g.num_blocks;
  const V* from = reinterpret_cast<const V*>(g.cache[kv] + (base + src) * g.block_bytes);
  V* to = reinterpret_cast<V*>(g.cache[kv] + (base + dst) * g.block_bytes);
  for (int64_t i = threadIdx.x; i < n; i += kCopyThreads * kCopyUnroll) {
    V x[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (i + u * kCopyThreads < n) x[u] = from[i + u * kCopyThreads];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (i + u * kCopyThreads < n) to[i + u * kCopyThreads] = x[u];
  }
  if (g.scales[kv] != nullptr)
    for (int h = threadIdx.x; h < g.hkv; h += kCopyThreads)
      g.scales[kv][(base + dst) * g.hkv + h] = g.scales[kv][(base + src) * g.hkv + h];
}

template <typename V>
__global__ void __launch_bounds__(kCopyThreads) copy_blocks(const Pages g, const int32_t* src,
                                                            const int32_t* dst, int64_t pairs,
                                                            int32_t* err) {
  const int64_t total = pairs * g.num_layers * 2;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int64_t i = w / (2 * g.num_layers), r = w - i * 2 * g.num_layers;
    const int64_t s = __ldg(src + i), d = __ldg(dst + i);
    if (s < 0 || d < 0) continue;  // padding: nothing to copy
    if (s >= g.num_blocks || d >= g.num_blocks) {
      if (threadIdx.x == 0 && r == 0) set_device_error(err, B2P_DEV_BLOCK_RANGE);
      continue;
    }
    if (s != d) copy_page<V>(g, s, d, r >> 1, (int)(r & 1));
  }
}

struct CompactPlan {
  uint32_t* bits;  // one per block, zero at the start
  int32_t* src;    // moves (at most num_blocks / 2 of them)
  int32_t* dst;
  int32_t* moves;  // their number
};

struct Tables {
  const int32_t* tables;
  int64_t stride;
  const int32_t* ctx;
  int num_seqs, width, block_size;
};

// Entries i, i + step, .. of the tables (row by row): the bits of the blocks that they name.
__device__ __forceinline__ void mark_entries(const Tables& t, int64_t i, int64_t step, int64_t num_blocks,
                                             uint32_t* bits, int32_t* err) {
  const int64_t total = (int64_t)t.num_seqs * t.width;
  for (; i < total; i += step) {
    const int seq = (int)(i / t.width), col = (int)(i - (int64_t)seq * t.width);
    const int c = __ldg(t.ctx + seq);
    const int64_t used = c > 0 ? ((int64_t)c + t.block_size - 1) / t.block_size : 0;
    if (col == 0 && used > t.width) set_device_error(err, B2P_DEV_LENGTH);
    if (col >= used) continue;
    const int32_t b = t.tables[seq * t.stride + col];
    if (b < 0 || b >= num_blocks) {
      set_device_error(err, B2P_DEV_BLOCK_RANGE);
      continue;
    }
    atomicOr(bits + (b >> 5), 1u << (b & 31));
  }
}

__global__ void __launch_bounds__(256) mark_live(const Tables t, int64_t num_blocks, uint32_t* bits, int32_t* err) {
  mark_entries(t, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll, num_blocks, bits, err);
}

constexpr int kPlanThreads = 1024;

// Exclusive scan over the CTA's threads; returns this thread's offset and the total.
__device__ int scan_cta(int x, int* shared, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();  // shared is free (a scan before this one)
  if (lane == 31) shared[warp] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += shared[w];
    total += shared[w];
  }
  return before + incl - x;
}

// Words of 32 blocks, a contiguous run per thread.
__device__ __forceinline__ void plan(const uint32_t* bits, const CompactPlan& pl, int64_t num_blocks,
                                     int32_t* new_ids, int32_t* num_live) {
  __shared__ int shared[kPlanThreads / 32];
  const int words = (int)((num_blocks + 31) / 32);
  const int per = (words + kPlanThreads - 1) / kPlanThreads;
  const int w0 = min(words, (int)threadIdx.x * per), w1 = min(words, w0 + per);
  int mine = 0, live = 0, moves = 0;
  for (int w = w0; w < w1; ++w) mine += __popc(bits[w]);
  scan_cta(mine, shared, live);
  // holes: free blocks below `live`; movers: live blocks from there on
  auto below = [&](int w) {
    const int64_t n = (int64_t)live - 32ll * w;
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
  };
  int holes = 0, movers = 0;
  for (int w = w0; w < w1; ++w) {
    holes += __popc(~bits[w] & below(w));
    movers += __popc(bits[w] & ~below(w));
  }
  int h = scan_cta(holes, shared, moves);
  int m = scan_cta(movers, shared, moves);
  for (int w = w0; w < w1; ++w) {
    for (uint32_t x = ~bits[w] & below(w); x != 0; x &= x - 1) pl.dst[h++] = 32 * w + __ffs(x) - 1;
    for (uint32_t x = bits[w] & ~below(w); x != 0; x &= x - 1) pl.src[m++] = 32 * w + __ffs(x) - 1;
  }
  for (int64_t b = threadIdx.x; b < num_blocks; b += kPlanThreads)
    new_ids[b] = b < live && (bits[b >> 5] >> (b & 31) & 1u) ? (int32_t)b : -1;
  __syncthreads();  // the lists and the ids of the blocks that stay are written
  for (int k = threadIdx.x; k < moves; k += kPlanThreads) new_ids[pl.src[k]] = pl.dst[k];
  if (threadIdx.x == 0) {
    *pl.moves = moves;
    *num_live = live;
  }
}

__global__ void __launch_bounds__(kPlanThreads) plan_moves(const CompactPlan pl, int64_t num_blocks,
                                                           int32_t* new_ids, int32_t* num_live) {
  plan(pl.bits, pl, num_blocks, new_ids, num_live);
}

__global__ void __launch_bounds__(kPlanThreads) mark_and_plan(const Tables t, const CompactPlan pl,
                                                              int64_t num_blocks, int32_t* new_ids,
                                                              int32_t* num_live, int32_t* err) {
  extern __shared__ uint32_t marks[];
  const int words = (int)((num_blocks + 31) / 32);
  for (int i = threadIdx.x; i < words; i += kPlanThreads) marks[i] = 0;
  __syncthreads();
  mark_entries(t, threadIdx.x, kPlanThreads, num_blocks, marks, err);
  __syncthreads();
  plan(marks, pl, num_blocks, new_ids, num_live);
}

template <typename V>
__global__ void __launch_bounds__(kCopyThreads) move_blocks(const Pages g, const CompactPlan pl,
                                                            const int32_t* new_ids, int32_t* tables,
                                                            int64_t stride, int width,
                                                            const int32_t* ctx, int num_seqs,
                                                            int block_size) {
  const int64_t total = (int64_t)__ldg(pl.moves) * g.num_layers * 2;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int64_t i = w / (2 * g.num_layers), r = w - i * 2 * g.num_layers;
    copy_page<V>(g, __ldg(pl.src + i), __ldg(pl.dst + i), r >> 1, (int)(r & 1));
  }
  const int64_t entries = (int64_t)num_seqs * width;
  for (int64_t i = blockIdx.x * (int64_t)kCopyThreads + threadIdx.x; i < entries;
       i += (int64_t)gridDim.x * kCopyThreads) {
    const int seq = (int)(i / width), col = (int)(i - (int64_t)seq * width);
    const int c = __ldg(ctx + seq);
    if (c <= 0 || col >= ((int64_t)c + block_size - 1) / block_size) continue;
    int32_t* e = tables + seq * stride + col;
    if (*e >= 0 && *e < g.num_blocks) *e = __ldg(new_ids + *e);
  }
}

int pages_of(Pages& g, void* key_cache, void* value_cache, float* key_scales, float* value_scales,
             int64_t num_layers, int64_t num_slots, int num_kv_heads, int head_dim,
             int element_bytes, int block_size) {
  if (num_layers <= 0 || num_slots <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      num_slots % block_size != 0 || (key_scales == nullptr) != (value_scales == nullptr))
    return B2P_EINVAL;
  if ((element_bytes != 1 && element_bytes != 2 && element_bytes != 4) || num_slots > 0x7fffffffLL)
    return B2P_EUNSUPPORTED;
  g.cache[0] = static_cast<uint8_t*>(key_cache);
  g.cache[1] = static_cast<uint8_t*>(value_cache);
  g.scales[0] = key_scales;
  g.scales[1] = value_scales;
  g.block_bytes = (int64_t)block_size * num_kv_heads * head_dim * element_bytes;
  g.num_blocks = num_slots / block_size;
  g.num_layers = num_layers;
  g.hkv = num_kv_heads;
  return B2P_OK;
}

bool vector16(const Pages& g) {
  return g.block_bytes % 16 == 0 &&
         ((reinterpret_cast<uintptr_t>(g.cache[0]) | reinterpret_cast<uintptr_t>(g.cache[1])) & 15u) == 0;
}

// Tables and pools that one CTA marks and plans for, without a memset and a second launch: 1792
// entries 10.3 us with nothing to move against 13.7, 4096: 12.8 against 14.7, 8192: 16.6 both (and
// 4 us less on the host), 32768: 35 against 27.
constexpr int64_t kOneCtaEntries = 8192;
constexpr int64_t kOneCtaBlocks = 8 * 32 * 1024;  // their bits fit 32 KB of shared memory

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace

extern "C" int b2p_copy_blocks(void* key_cache, void* value_cache, float* key_scales,
                               float* value_scales, const int32_t* src_blocks,
                               const int32_t* dst_blocks, int64_t num_pairs, int64_t num_layers,
                               int64_t num_slots, int num_kv_heads, int head_dim,
                               int element_bytes, int block_size, int32_t* err_flag, void* stream) {
  Pages g;
  const int rc = pages_of(g, key_cache, value_cache, key_scales, value_scales, num_layers, num_slots,
                          num_kv_heads, head_dim, element_bytes, block_size);
  if (rc != B2P_OK) return rc;
  if (num_pairs < 0) return B2P_EINVAL;
  if (num_pairs == 0) return B2P_OK;
  if (!key_cache || !value_cache || !src_blocks || !dst_blocks) return B2P_EINVAL;
  const int64_t work = num_pairs * num_layers * 2;
  const int64_t most = (int64_t)b2p_host::sm_count() * 16;
  const unsigned grid = (unsigned)(work < most ? work : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (vector16(g))
    copy_blocks<uint4><<<grid, kCopyThreads, 0, s>>>(g, src_blocks, dst_blocks, num_pairs, err_flag);
  else
    copy_blocks<uint8_t><<<grid, kCopyThreads, 0, s>>>(g, src_blocks, dst_blocks, num_pairs, err_flag);
  return b2p_host::check_launch();
}

extern "C" size_t b2p_compact_blocks_workspace_size(int64_t num_blocks) {
  if (num_blocks <= 0) return 0;
  return align256((size_t)(num_blocks + 31) / 32 * 4) + 2 * align256((size_t)(num_blocks / 2 + 1) * 4) + 256;
}

extern "C" int b2p_compact_blocks(void* key_cache, void* value_cache, float* key_scales,
                                  float* value_scales, int32_t* block_tables,
                                  int64_t block_table_stride, int table_width,
                                  const int32_t* context_lens, int num_seqs, int64_t num_layers,
                                  int64_t num_slots, int num_kv_heads, int head_dim,
                                  int element_bytes, int block_size, int32_t* new_ids,
                                  int32_t* num_live, void* workspace, size_t workspace_size,
                                  int32_t* err_flag, void* stream) {
  Pages g;
  const int rc = pages_of(g, key_cache, value_cache, key_scales, value_scales, num_layers, num_slots,
                          num_kv_heads, head_dim, element_bytes, block_size);
  if (rc != B2P_OK) return rc;
  if (num_seqs < 0 || table_width < 0 || block_table_stride < table_width) return B2P_EINVAL;
  if (!key_cache || !value_cache || !new_ids || !num_live ||
      (num_seqs > 0 && table_width > 0 && (!block_tables || !context_lens)))
    return B2P_EINVAL;
  if (reinterpret_cast<uintptr_t>(workspace) & 15u) return B2P_EINVAL;
  if (!workspace || workspace_size < b2p_compact_blocks_workspace_size(g.num_blocks))
    return B2P_EWORKSPACE;
  const size_t bits_bytes = align256((size_t)(g.num_blocks + 31) / 32 * 4);
  const size_t list_bytes = align256((size_t)(g.num_blocks / 2 + 1) * 4);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  CompactPlan pl;
  pl.bits = reinterpret_cast<uint32_t*>(ws);
  pl.src = reinterpret_cast<int32_t*>(ws + bits_bytes);
  pl.dst = reinterpret_cast<int32_t*>(ws + bits_bytes + list_bytes);
  pl.moves = reinterpret_cast<int32_t*>(ws + bits_bytes + 2 * list_bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Tables t{block_tables, block_table_stride, context_lens, num_seqs, table_width, block_size};
  const int64_t entries = (int64_t)num_seqs * table_width;
  if (entries <= kOneCtaEntries && g.num_blocks <= kOneCtaBlocks) {
    mark_and_plan<<<1, kPlanThreads, (size_t)(g.num_blocks + 31) / 32 * 4, s>>>(t, pl, g.num_blocks, new_ids,
                                                                               num_live, err_flag);
    const int lrc = b2p_host::check_launch();
    if (lrc != B2P_OK) return lrc;
  } else {
    const cudaError_t e = cudaMemsetAsync(pl.bits, 0, bits_bytes, s);
    if (e != cudaSuccess) return b2p_host::record_error(e);
    const int64_t want = (entries + 255) / 256, most = (int64_t)b2p_host::sm_count() * 4;
    if (entries > 0)
      mark_live<<<(unsigned)(want < most ? want : most), 256, 0, s>>>(t, g.num_blocks, pl.bits, err_flag);
    const int lrc = b2p_host::check_launch();
    if (lrc != B2P_OK) return lrc;
    plan_moves<<<1, kPlanThreads, 0, s>>>(pl, g.num_blocks, new_ids, num_live);
    const int prc = b2p_host::check_launch();
    if (prc != B2P_OK) return prc;
  }
  const unsigned grid = (unsigned)b2p_host::sm_count() * 16;
  if (vector16(g))
    move_blocks<uint4><<<grid, kCopyThreads, 0, s>>>(g, pl, new_ids, block_tables,
                                                     block_table_stride, table_width, context_lens,
                                                     num_seqs, block_size);
  else
    move_blocks<uint8_t><<<grid, kCopyThreads, 0, s>>>(g, pl, new_ids, block_tables,
                                                       block_table_stride, table_width,
                                                       context_lens, num_seqs, block_size);
  return b2p_host::check_launch();
}
