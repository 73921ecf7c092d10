// Entry points of attention over the 8-bit KV cache: b2p_paged_decode_fp8 (one query row per
// sequence) and b2p_paged_prefill_fp8 (q_len_i rows, causal: the rows of drafted tokens, of
// prompt slices and of whole prompts).
//
// Few rows stream the codes (decode_fp8.cu). Many rows are bound by the tensor cores and read
// every key tile once per 128-row query tile and head pair; there the histories are widened once
// per call into a 16-bit scratch pool (23 us of the 777 below) and the 16-bit tile kernel
// (prefill_tc.cu) runs on that. Widening inside the tile kernel instead, by two more warps that
// fill its shared-memory tiles from the codes, repeats the conversion for every query tile and
// head pair: 2351 us against 777 on 32 prompts of 64 to 8192 tokens.
#include <type_traits>

#include "fp8.cuh"

int b2p_attn_fp8_simt(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                      const void* key_cache, const void* value_cache, const float* key_scales,
                      const float* value_scales, int64_t layer_index, int64_t num_slots,
                      const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_q,
                      const int32_t* context_lens, int num_seqs, int64_t num_rows, int num_q_heads,
                      int num_kv_heads, int head_dim, int block_size, float scale, void* out,
                      int64_t out_tok_stride, int64_t out_head_stride, int dtype,
                      int32_t* err_flag, void* stream);

bool b2p_rows_fp8_takes(int group, int head_dim, int block_size, int dtype, int max_q_len);
size_t b2p_rows_fp8_workspace(int num_seqs, int num_kv_heads);
int b2p_rows_fp8(const void* q, int64_t q_tok_stride, int64_t q_head_stride, const void* key_cache,
                 const void* value_cache, const float* key_scales, const float* value_scales,
                 int64_t layer_index, int64_t num_layers, int64_t num_slots,
                 const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_q,
                 const int32_t* context_lens, int num_seqs, int64_t num_rows, int max_q_len,
                 int num_q_heads, int num_kv_heads, int head_dim, int block_size, float scale,
                 void* out, int64_t out_tok_stride, int64_t out_head_stride, void* workspace,
                 size_t workspace_size, int dtype, int32_t* err_flag, void* stream);

float b2p_prefill_no_weight();
int b2p_prefill_tc_runs(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                        const void* key_cache, const void* value_cache, int64_t num_slots,
                        const int32_t* block_tables, int64_t block_table_stride,
                        const int32_t* cu_seqlens_q, const int32_t* context_lens, int num_seqs,
                        int64_t total_q, int num_q_heads, int num_kv_heads, int head_dim,
                        int block_size, float scale, void* out, int64_t out_tok_stride,
                        int64_t out_head_stride, int dtype, int32_t* err_flag, void* stream,
                        int32_t* claims, int splits, float* part, float* lse);

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// What prefill_tc.cu asks of the query and output rows.
bool tile_rows_fit(const void* q, int64_t q_tok, int64_t q_head, const void* out, int64_t o_tok, int64_t o_head) {
  return aligned(q, 16) && aligned(out, 16) && q_tok % 8 == 0 && q_head % 8 == 0 && o_tok % 8 == 0 && o_head % 8 == 0;
}

// Pool rows fit TMA boxes, query rows 8-byte loads, output rows 4-byte stores.
bool rows_fit(const void* q, int64_t q_tok, int64_t q_head, const void* kc, const void* vc,
              const void* out, int64_t o_tok, int64_t o_head) {
  return aligned(q, 8) && q_tok % 4 == 0 && q_head % 4 == 0 && aligned(kc, 16) && aligned(vc, 16) &&
         aligned(out, 4) && o_tok % 2 == 0 && o_head % 2 == 0;
}

using namespace b2p;

constexpr int kWidenThreads = 256;
constexpr int kWidenLoads = 2;  // loads that a thread has in flight

struct WidenParams {
  const uint8_t* codes[2];  // layer bases of K and V
  const float* scales[2];
  uint8_t* wide[2];         // scratch pools
  int32_t* tables;          // scratch block tables [num_seqs, width]; null: blocks keep their ids
  const int32_t* block_tables;
  int64_t bt_stride;
  int width;
  int parts, share;  // pieces of a block, rounds of the CTA's loads in each
  const int32_t* cu;
  const int32_t* ctx;
  int32_t* safe_cu;   // [num_seqs + 1] and [num_seqs]: the same within q's rows and the tables'
  int32_t* safe_ctx;  // reach, for the tile kernel, which trusts them
  int32_t* claims;    // the tile kernel's two claim counters, to zero
  uint8_t* out;
  int64_t o_tok, o_head, num_rows;
  int num_seqs, hq, hkv, d, block_size;
  int64_t num_blocks;
  float* lse;  // split calls: weights to clear, num_lse of them (null: none)
  int64_t num_lse;
  float no_weight;
  int32_t* err;
};

constexpr float kF16Scale = 146.f;  // 448 times a larger one may pass 65,536, the largest value of f16 rows

// f16 keeps 65,472 where a product passes it (the next stored value is 65,536): 2^-11 below f16's largest
// finite value, which is what the rounding of the weights in P V may add to a mean.
template <typename T>
__device__ __forceinline__ float bounded(float x) {
  return std::is_same<T, __half>::value ? (x > 65472.f ? 65472.f : x < -65472.f ? -65472.f : x) : x;
}

__device__ __forceinline__ int row_within(const WidenParams& p, int row) {
  return (int)min(max((int64_t)row, (int64_t)0), p.num_rows);
}

// A CTA takes pieces of the used blocks of all histories in turn (found by a scan of the lengths,
// 32 sequences at a time: with one CTA per table entry, most of a ragged batch's are empty, 35 us
// against 22 on 32 prompts) and writes their codes as 16-bit rows: into a scratch block of the entry's
// own, which the scratch table names, or into a scratch pool with the blocks' own ids, whichever pool
// is smaller. (With their own ids, sequences that share a block write the same bytes to it.) A piece is
// a whole block where there are many, else down to what the CTA's threads have in flight at once
// (one sequence of 210 rows and 4 heads in blocks of 64: the call takes 17.9 us, 22.5 with whole
// blocks). Memory-bound: 1 byte read and 2 written per element.
template <typename T>
__global__ void __launch_bounds__(kWidenThreads, 8) widen_histories(const WidenParams p) {
  __shared__ int found[2];  // sequence (-1: no block left) and block number
  // the tile kernel may set itself up meanwhile; it reads nothing before this grid has ended
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x < 2) p.claims[threadIdx.x] = 0;
  for (int64_t i = blockIdx.x * (int64_t)kWidenThreads + threadIdx.x; i < p.num_lse;
       i += (int64_t)gridDim.x * kWidenThreads)
    p.lse[i] = p.no_weight;
  // rows before a sequence's first position see nothing: zeros (the tile kernel may skip them)
  for (int seq = blockIdx.x; seq < p.num_seqs; seq += gridDim.x) {
    const int first = __ldg(p.cu + seq), last = __ldg(p.cu + seq + 1), ctx = __ldg(p.ctx + seq);
    const int q0 = row_within(p, first), rows = row_within(p, last) - q0;
    const int blind = min(rows, rows - max(ctx, 0));
    if (threadIdx.x == 0) {
      if (q0 != first || q0 + rows != last || (rows > 0 && blind > 0)) set_device_error(p.err, B2P_DEV_LENGTH);
      if (rows > 0 && ctx > (int64_t)p.width * p.block_size) set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
      p.safe_cu[seq] = q0;
      if (seq == p.num_seqs - 1) p.safe_cu[seq + 1] = q0 + rows;
      p.safe_ctx[seq] = (int)min((int64_t)ctx, (int64_t)p.width * p.block_size);
    }
    for (int64_t e = threadIdx.x; e < (int64_t)max(blind, 0) * p.hq * p.d; e += kWidenThreads) {
      const int64_t row = q0 + e / (p.hq * p.d);
      const int r = (int)(e % (p.hq * p.d));
      reinterpret_cast<T*>(p.out)[row * p.o_tok + (int64_t)(r / p.d) * p.o_head + r % p.d] = from_f32<T>(0.f);
    }
  }
  const int per_row = p.hkv * p.d / 16, per_head = p.d / 16;  // 16-code loads
  for (int64_t unit = blockIdx.x;; unit += gridDim.x) {
    __syncthreads();  // the previous round has read `found`
    if (threadIdx.x < 32) {
      int64_t want = unit / p.parts;
      int seq = -1, col = 0;
      for (int base = 0; base < p.num_seqs && seq < 0; base += 32) {
        const int s = base + lane;
        int n = 0;
        if (s < p.num_seqs && __ldg(p.cu + s + 1) > __ldg(p.cu + s))
          n = (int)min((int64_t)p.width,
                       ((int64_t)max(__ldg(p.ctx + s), 0) + p.block_size - 1) / p.block_size);
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, incl > want);
        if (hit) {
          const int src = __ffs(hit) - 1;
          seq = base + src;
          col = (int)(want - __shfl_sync(0xffffffffu, incl - n, src));
        } else {
          want -= __shfl_sync(0xffffffffu, incl, 31);
        }
      }
      if (lane == 0) {
        found[0] = seq;
        found[1] = col;
      }
    }
    __syncthreads();
    const int seq = found[0], col = found[1], part = (int)(unit % p.parts);
    if (seq < 0) return;
    const int64_t entry = (int64_t)seq * p.width + col;
    const int tokens = min(p.block_size, __ldg(p.ctx + seq) - col * p.block_size);
    const int32_t blk = __ldg(p.block_tables + (int64_t)seq * p.bt_stride + col);
    const bool have = blk >= 0 && blk < p.num_blocks;
    if (threadIdx.x == 0 && part == 0) {
      if (p.tables != nullptr) p.tables[entry] = (int32_t)entry;
      if (!have) set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
    }
    if (p.tables == nullptr && !have) continue;  // the tile kernel finds the bad id itself
    const int64_t w = p.tables != nullptr ? entry : blk;
    const int loads = tokens * per_row;  // of K, and as many of V
    const int share = p.share * kWidenLoads * kWidenThreads;
    const int end = min(2 * loads, (part + 1) * share);
    for (int i0 = part * share + threadIdx.x; i0 < end; i0 += kWidenLoads * kWidenThreads) {
      uint4 raw[kWidenLoads];
      float sk[kWidenLoads], sv[kWidenLoads];
#pragma unroll
      for (int k = 0; k < kWidenLoads; ++k) {
        const int i = i0 + k * kWidenThreads;
        raw[k] = make_uint4(0, 0, 0, 0);
        sk[k] = sv[k] = 0.f;
        if (have && i < end) {
          const bool is_v = i >= loads;
          const int at = is_v ? i - loads : i;
          raw[k] = __ldg(reinterpret_cast<const uint4*>(p.codes[is_v]) + (int64_t)blk * p.block_size * per_row + at);
          const int64_t sc = (int64_t)blk * p.hkv + at % per_row / per_head;
          sk[k] = __ldg(p.scales[0] + sc);
          sv[k] = __ldg(p.scales[1] + sc);
        }
      }
#pragma unroll
      for (int k = 0; k < kWidenLoads; ++k) {
        const int i = i0 + k * kWidenThreads;
        if (i >= end) break;
        const bool is_v = i >= loads;
        const int at = is_v ? i - loads : i;
        // A NaN value block shows through the scores alone: rows that do not see it would
        // otherwise meet it as 0 * NaN in P V.
        const float s = is_v ? (sv[k] == sv[k] ? sv[k] : 0.f) : (sv[k] == sv[k] ? sk[k] : sv[k]);
        uint32_t words[8];
        const uint32_t in[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        if (std::is_same<T, __half>::value && fabsf(s) > kF16Scale) {  // not from f16 rows, as a rule
          bool past = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t two = fp8x2_to_f16x2((uint16_t)(in[e >> 1] >> (16 * (e & 1))));
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&two));
            past |= fabsf(x.x * s) > 65536.f || fabsf(x.y * s) > 65536.f;
          }
          if (past) set_device_error(p.err, B2P_DEV_VALUE_RANGE);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t two = fp8x2_to_f16x2((uint16_t)(in[e >> 1] >> (16 * (e & 1))));
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&two));
          words[e] = pack2<T>(bounded<T>(x.x * s), bounded<T>(x.y * s));
        }
        uint4* to = reinterpret_cast<uint4*>(p.wide[is_v]) + (w * p.block_size * per_row + at) * 2;
        to[0] = make_uint4(words[0], words[1], words[2], words[3]);
        to[1] = make_uint4(words[4], words[5], words[6], words[7]);
      }
    }
  }
}

constexpr int kMostSplits = 8;
constexpr int kRunTiles = 8;

// Scratch of the widened form: the checked offsets and lengths, the claim counters and (blocks by table
// entry) the block tables, then K, then V, then (split calls) the runs' results and weights. The
// 16-bit copies take as many blocks as the tables have entries or as the pool has blocks, whichever is
// less: tables are as wide as their longest sequence, and a batch of unlike lengths would
// otherwise ask for many times what it holds (32 prompts of which one has 131,072 tokens, 8 heads of
// 128: 17 GB).
size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

struct Scratch {
  int64_t blocks;  // of the 16-bit copies
  bool own_ids;    // they are the pool's own
  size_t tables, pool, part, lse;  // bytes
  size_t total() const { return tables + 2 * pool + part + lse; }
};

Scratch scratch_of(int num_seqs, int64_t width, int64_t pool_blocks, int num_kv_heads, int head_dim, int block_size,
                   int splits, int64_t total_q, int num_q_heads) {
  Scratch c;
  const int64_t entries = (int64_t)num_seqs * width;
  c.own_ids = pool_blocks < entries;
  c.blocks = c.own_ids ? pool_blocks : entries;
  c.tables = align256(((c.own_ids ? 0 : (size_t)entries) + 2 * (size_t)num_seqs + 1 + 2) * 4);
  c.pool = align256((size_t)c.blocks * block_size * num_kv_heads * head_dim * 2);
  const size_t rows = splits > 1 ? (size_t)splits * total_q * num_q_heads : 0;
  c.part = align256(rows * head_dim * 4);
  c.lse = align256(rows * 4);
  return c;
}

// Runs that every (query tile, pair of heads) item's keys are cut into, where a call has too few
// items for the SMs: one wave of them where they are fewer than half the SMs, else about three
// per SM, so that a long history next to short ones does not set the time. A run is at least
// kRunTiles KV tiles of the longest history that table_width allows (for the lengths are on the device). Four 512-token
// slices over 100 to 7777 tokens (14/2 heads): 103 us whole, 88 in two runs, 78 in three, 89 in
// six; one such slice over 8000 tokens (12/2 heads): 63 in five runs, 83 in eight (a second
// wave); four whole 512-token prompts: 47 whole, 60 in four runs.
int key_splits(int num_seqs, int64_t total_q, int64_t table_width, int num_q_heads, int num_kv_heads, int block_size) {
  const int pairs = (num_q_heads / num_kv_heads + 1) / 2;
  const int64_t items = ((total_q + 127) / 128 + num_seqs - 1) * num_kv_heads * pairs;
  const int64_t sms = b2p_host::sm_count();
  const int64_t most = table_width * block_size / 128 / kRunTiles;
  int64_t n = items >= 3 * sms ? 1 : items <= sms / 2 ? sms / items : (3 * sms + items - 1) / items;
  n = n < most ? n : most;
  n = n < kMostSplits ? n : kMostSplits;
  return (int)(n > 1 ? n : 1);
}

bool tile_shape(int head_dim, int block_size, int dtype) {
  return (head_dim == 64 || head_dim == 128) && block_size % 16 == 0 &&
         (dtype == B2P_BF16 || dtype == B2P_F16);
}

int check_args(const void* key_cache, const void* value_cache, const void* workspace, float scale,
               int64_t layer_index, int64_t num_layers, int64_t num_slots, int num_seqs,
               int64_t num_rows, int max_q_len, int num_q_heads, int num_kv_heads, int head_dim,
               int block_size, int64_t block_table_stride, int dtype) {
  if (num_seqs < 0 || num_rows < 0 || max_q_len < 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      head_dim <= 0 || block_size <= 0 || num_slots <= 0 || num_layers <= 0 ||
      block_table_stride < 0)
    return B2P_EINVAL;
  if (num_q_heads % num_kv_heads != 0 || num_slots % block_size != 0) return B2P_EINVAL;
  if (dtype < B2P_BF16 || dtype > B2P_F32) return B2P_EINVAL;
  if (layer_index < 0 || layer_index >= num_layers) return B2P_ERANGE;
  if (!aligned(key_cache, 8) || !aligned(value_cache, 8) || !aligned(workspace, 16)) return B2P_EINVAL;
  if (!(scale >= 0.f)) return B2P_EINVAL;  // the running maxima take a larger product for a larger score
  if (head_dim % 8 != 0 || head_dim > 256 || num_slots > 0x7fffffffLL || num_rows > 0x7fffffffLL)
    return B2P_EUNSUPPORTED;
  return B2P_OK;
}

}  // namespace

extern "C" size_t b2p_paged_fp8_workspace_size(int num_seqs, int num_q_heads, int num_kv_heads,
                                               int head_dim, int max_q_len) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || head_dim <= 0 || max_q_len < 0) return 0;
  if (num_q_heads % num_kv_heads != 0) return 0;
  // shapes that only the CUDA-core kernel takes need none
  if (!b2p_rows_fp8_takes(num_q_heads / num_kv_heads, head_dim, 16, B2P_BF16, 1)) return 16;
  return b2p_rows_fp8_workspace(num_seqs, num_kv_heads);
}

extern "C" int b2p_paged_decode_fp8(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                    const void* key_cache, const void* value_cache,
                                    const float* key_scales, const float* value_scales,
                                    int64_t layer_index, int64_t num_layers, int64_t num_slots,
                                    const int32_t* block_tables, int64_t block_table_stride,
                                    const int32_t* context_lens, int num_seqs, int num_q_heads,
                                    int num_kv_heads, int head_dim, int block_size, float scale,
                                    void* out, int64_t out_tok_stride, int64_t out_head_stride,
                                    void* workspace, size_t workspace_size, int dtype,
                                    int32_t* err_flag, void* stream) {
  const int rc = check_args(key_cache, value_cache, workspace, scale, layer_index, num_layers, num_slots, num_seqs, num_seqs, 1, num_q_heads,
                            num_kv_heads, head_dim, block_size, block_table_stride, dtype);
  if (rc != B2P_OK || num_seqs == 0) return rc;
  if (!q || !key_cache || !value_cache || !key_scales || !value_scales || !block_tables ||
      !context_lens || !out)
    return B2P_EINVAL;
  if (b2p_rows_fp8_takes(num_q_heads / num_kv_heads, head_dim, block_size, dtype, 1) &&
      rows_fit(q, q_tok_stride, q_head_stride, key_cache, value_cache, out, out_tok_stride, out_head_stride))
    return b2p_rows_fp8(q, q_tok_stride, q_head_stride, key_cache, value_cache, key_scales,
                        value_scales, layer_index, num_layers, num_slots, block_tables,
                        block_table_stride, nullptr, context_lens, num_seqs, num_seqs, 1,
                        num_q_heads, num_kv_heads, head_dim, block_size, scale, out,
                        out_tok_stride, out_head_stride, workspace, workspace_size, dtype,
                        err_flag, stream);
  if (dtype != B2P_F32) b2p_host::note_fallback(2);
  return b2p_attn_fp8_simt(q, q_tok_stride, q_head_stride, key_cache, value_cache, key_scales,
                           value_scales, layer_index, num_slots, block_tables, block_table_stride,
                           nullptr, context_lens, num_seqs, num_seqs, num_q_heads, num_kv_heads,
                           head_dim, block_size, scale, out, out_tok_stride, out_head_stride,
                           dtype, err_flag, stream);
}

extern "C" size_t b2p_paged_prefill_fp8_pool_scratch_size(int num_seqs, int64_t total_q, int64_t table_width,
                                                          int64_t num_slots, int num_q_heads, int num_kv_heads,
                                                          int head_dim, int block_size, int max_q_len, int dtype) {
  if (num_seqs <= 0 || total_q <= 0 || table_width <= 0 || num_slots <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      head_dim <= 0 || block_size <= 0 || max_q_len < 0 || num_q_heads % num_kv_heads != 0 ||
      !tile_shape(head_dim, block_size, dtype))
    return 0;
  if (b2p_rows_fp8_takes(num_q_heads / num_kv_heads, head_dim, block_size, dtype, max_q_len)) return 0;
  const int splits = key_splits(num_seqs, total_q, table_width, num_q_heads, num_kv_heads, block_size);
  return scratch_of(num_seqs, table_width, num_slots / block_size, num_kv_heads, head_dim, block_size, splits, total_q,
                    num_q_heads)
      .total();
}

// The same for any pool: one with more blocks than the tables have entries asks for the most.
extern "C" size_t b2p_paged_prefill_fp8_scratch_size(int num_seqs, int64_t total_q, int64_t table_width, int num_q_heads,
                                                     int num_kv_heads, int head_dim, int block_size,
                                                     int max_q_len, int dtype) {
  return b2p_paged_prefill_fp8_pool_scratch_size(num_seqs, total_q, table_width, INT64_MAX, num_q_heads, num_kv_heads,
                                                 head_dim, block_size, max_q_len, dtype);
}

extern "C" int b2p_paged_prefill_fp8_reach(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                           const void* key_cache, const void* value_cache,
                                           const float* key_scales, const float* value_scales,
                                           int64_t layer_index, int64_t num_layers, int64_t num_slots,
                                           const int32_t* block_tables, int64_t block_table_stride,
                                           int64_t table_width,
                                           const int32_t* cu_seqlens_q, const int32_t* context_lens,
                                           int num_seqs, int64_t total_q, int max_q_len, int num_q_heads,
                                           int num_kv_heads, int head_dim, int block_size, float scale,
                                           void* out, int64_t out_tok_stride, int64_t out_head_stride,
                                           void* workspace, size_t workspace_size, void* scratch,
                                           size_t scratch_size, int dtype,
                                           int32_t* err_flag, void* stream) {
  const int rc = check_args(key_cache, value_cache, workspace, scale, layer_index, num_layers, num_slots, num_seqs, total_q, max_q_len,
                            num_q_heads, num_kv_heads, head_dim, block_size, block_table_stride,
                            dtype);
  if (rc == B2P_OK && (table_width < 0 || table_width > block_table_stride)) return B2P_EINVAL;
  if (rc != B2P_OK || num_seqs == 0 || total_q == 0 || max_q_len == 0) return rc;
  if (!q || !key_cache || !value_cache || !key_scales || !value_scales || !block_tables ||
      !cu_seqlens_q || !context_lens || !out)
    return B2P_EINVAL;
  if (b2p_rows_fp8_takes(num_q_heads / num_kv_heads, head_dim, block_size, dtype, max_q_len) &&
      rows_fit(q, q_tok_stride, q_head_stride, key_cache, value_cache, out, out_tok_stride, out_head_stride))
    return b2p_rows_fp8(q, q_tok_stride, q_head_stride, key_cache, value_cache, key_scales,
                        value_scales, layer_index, num_layers, num_slots, block_tables,
                        block_table_stride, cu_seqlens_q, context_lens, num_seqs, total_q,
                        max_q_len, num_q_heads, num_kv_heads, head_dim, block_size, scale, out,
                        out_tok_stride, out_head_stride, workspace, workspace_size, dtype,
                        err_flag, stream);
  const int64_t width = table_width;
  if (tile_shape(head_dim, block_size, dtype) && aligned(key_cache, 16) && aligned(value_cache, 16) && width > 0 &&
      tile_rows_fit(q, q_tok_stride, q_head_stride, out, out_tok_stride, out_head_stride)) {
    const int splits = key_splits(num_seqs, total_q, width, num_q_heads, num_kv_heads, block_size);
    const Scratch need = scratch_of(num_seqs, width, num_slots / block_size, num_kv_heads, head_dim, block_size, splits,
                                    total_q, num_q_heads);
    if (!scratch || scratch_size < need.total() || !aligned(scratch, 16)) return B2P_EWORKSPACE;
    WidenParams w;
    const int64_t layer_codes = num_slots * num_kv_heads * head_dim;
    const int64_t layer_scales = num_slots / block_size * num_kv_heads;
    w.codes[0] = static_cast<const uint8_t*>(key_cache) + layer_index * layer_codes;
    w.codes[1] = static_cast<const uint8_t*>(value_cache) + layer_index * layer_codes;
    w.scales[0] = key_scales + layer_index * layer_scales;
    w.scales[1] = value_scales + layer_index * layer_scales;
    uint8_t* base = static_cast<uint8_t*>(scratch);
    w.safe_cu = reinterpret_cast<int32_t*>(base);
    w.safe_ctx = w.safe_cu + num_seqs + 1;
    w.claims = w.safe_ctx + num_seqs;
    w.tables = need.own_ids ? nullptr : w.claims + 2;
    w.wide[0] = base + need.tables;
    w.wide[1] = base + need.tables + need.pool;
    w.block_tables = block_tables;
    w.bt_stride = block_table_stride;
    w.width = (int)width;
    const int64_t most = (int64_t)b2p_host::sm_count() * 8;
    const int64_t blocks = (int64_t)num_seqs * width;
    // rounds that a block takes; it is cut into pieces where the call's own rows do not fill the CTAs
    const int rounds = (int)(((int64_t)2 * block_size * num_kv_heads * head_dim / 16 + kWidenLoads * kWidenThreads - 1) /
                             (kWidenLoads * kWidenThreads));
    const int64_t wanted = most * block_size / total_q + 1;
    w.parts = (int)(wanted < rounds ? wanted : rounds);
    w.share = (rounds + w.parts - 1) / w.parts;
    w.parts = (rounds + w.share - 1) / w.share;
    w.cu = cu_seqlens_q;
    w.ctx = context_lens;
    w.out = static_cast<uint8_t*>(out);
    w.o_tok = out_tok_stride;
    w.o_head = out_head_stride;
    w.num_rows = total_q;
    w.num_seqs = num_seqs;
    w.hq = num_q_heads;
    w.hkv = num_kv_heads;
    w.d = head_dim;
    w.block_size = block_size;
    w.num_blocks = num_slots / block_size;
    w.err = err_flag;
    float* part = reinterpret_cast<float*>(base + need.tables + 2 * need.pool);
    w.lse = reinterpret_cast<float*>(base + need.tables + 2 * need.pool + need.part);
    w.num_lse = splits > 1 ? (int64_t)splits * total_q * num_q_heads : 0;
    w.no_weight = b2p_prefill_no_weight();
    const unsigned grid = (unsigned)(blocks * w.parts < most ? blocks * w.parts : most);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == B2P_BF16)
      widen_histories<__nv_bfloat16><<<grid, kWidenThreads, 0, s>>>(w);
    else
      widen_histories<__half><<<grid, kWidenThreads, 0, s>>>(w);
    const int wrc = b2p_host::check_launch();
    if (wrc != B2P_OK) return wrc;
    const int trc = b2p_prefill_tc_runs(
        q, q_tok_stride, q_head_stride, w.wide[0], w.wide[1], need.blocks * block_size,
        need.own_ids ? block_tables : w.tables, need.own_ids ? block_table_stride : width, w.safe_cu, w.safe_ctx,
        num_seqs, total_q, num_q_heads, num_kv_heads, head_dim, block_size, scale, out, out_tok_stride,
        out_head_stride, dtype, err_flag, stream, w.claims, splits, part, w.lse);
    if (trc != B2P_EUNSUPPORTED) return trc;  // a device that the tile kernel does not fit: as b2p_paged_prefill does
  }
  if (dtype != B2P_F32) b2p_host::note_fallback(3);
  return b2p_attn_fp8_simt(q, q_tok_stride, q_head_stride, key_cache, value_cache, key_scales,
                           value_scales, layer_index, num_slots, block_tables, block_table_stride,
                           cu_seqlens_q, context_lens, num_seqs, total_q, num_q_heads,
                           num_kv_heads, head_dim, block_size, scale, out, out_tok_stride,
                           out_head_stride, dtype, err_flag, stream);
}

// The same over tables whose whole width counts.
extern "C" int b2p_paged_prefill_fp8(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                     const void* key_cache, const void* value_cache,
                                     const float* key_scales, const float* value_scales,
                                     int64_t layer_index, int64_t num_layers, int64_t num_slots,
                                     const int32_t* block_tables, int64_t block_table_stride,
                                     const int32_t* cu_seqlens_q, const int32_t* context_lens,
                                     int num_seqs, int64_t total_q, int max_q_len, int num_q_heads,
                                     int num_kv_heads, int head_dim, int block_size, float scale,
                                     void* out, int64_t out_tok_stride, int64_t out_head_stride,
                                     void* workspace, size_t workspace_size, void* scratch,
                                     size_t scratch_size, int dtype,
                                     int32_t* err_flag, void* stream) {
  return b2p_paged_prefill_fp8_reach(
      q, q_tok_stride, q_head_stride, key_cache, value_cache, key_scales, value_scales, layer_index, num_layers,
      num_slots, block_tables, block_table_stride, block_table_stride, cu_seqlens_q, context_lens, num_seqs, total_q,
      max_q_len, num_q_heads, num_kv_heads, head_dim, block_size, scale, out, out_tok_stride, out_head_stride,
      workspace, workspace_size, scratch, scratch_size, dtype, err_flag, stream);
}
