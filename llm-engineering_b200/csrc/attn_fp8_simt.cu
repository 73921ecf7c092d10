// CUDA-core attention over the 8-bit KV cache: fp32 queries and what the tensor-core kernels do
// not take (head dims other than 64 and 128, block sizes that are not a multiple of 16, decode
// steps of GQA groups above 160, unaligned rows).
//
// One warp owns one (query row, query head). Keys go 32 at a time: lane j computes the dot
// product of key (base + j) with the query (in shared memory, read as a broadcast) and
// multiplies it by the block's key scale; the warp updates its online softmax; then each lane
// accumulates P.V, P already multiplied by the block's value scale, for the head dims it owns.
// A query row j of a sequence with q_len rows and ctx keys sits at position ctx - q_len + j
// and sees keys 0 .. that position. Everything is fp32 from the codes on. Every (row, head) reads
// its keys anew and converts them one by one, which bounds it, not bytes: a decode step of 256
// sequences over 512 to 4096 tokens (12/2 heads, d 128) takes 3.3 ms in fp32, 59 us in bf16.
#include "fp8.cuh"

namespace {

using namespace b2p;

constexpr int kWarps = 4;
constexpr int kMaxD = 256;

struct SimtFp8Params {
  const uint8_t* q;
  int64_t q_tok, q_head;
  const uint8_t* k_cache;  // layer bases
  const uint8_t* v_cache;
  const float* k_scales;
  const float* v_scales;
  int64_t row_elems;  // num_kv_heads * head_dim
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* cu_q;  // null: row i is sequence i with q_len 1
  const int32_t* context_lens;
  int num_seqs, num_q_heads, num_kv_heads, group, head_dim, block_size;
  int64_t num_blocks, num_rows;
  float scale;
  uint8_t* out;
  int64_t o_tok, o_head;
  int32_t* err;
};

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_attn_fp8_simt(const SimtFp8Params p) {
  __shared__ float qs[kWarps][kMaxD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x + (p.cu_q == nullptr ? 0 : __ldg(p.cu_q));
  const int qh = blockIdx.y * kWarps + warp;
  if (qh >= p.num_q_heads || row < 0 || row >= p.num_rows) return;
  int seq = (int)row, q_len = 1, q_idx = 0;
  if (p.cu_q != nullptr) {
    int lo = 0, hi = p.num_seqs - 1;  // last sequence with cu_q[seq] <= row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(p.cu_q + mid) <= row) lo = mid; else hi = mid - 1;
    }
    seq = lo;
    if (row >= __ldg(p.cu_q + p.num_seqs)) return;  // the grid covers all rows of q
    q_len = __ldg(p.cu_q + seq + 1) - __ldg(p.cu_q + seq);
    q_idx = (int)(row - __ldg(p.cu_q + seq));
  }
  const int ctx = __ldg(p.context_lens + seq);
  const int pos = ctx - q_len + q_idx;  // position of this query
  const int kvh = qh / p.group, D = p.head_dim;
  const T* qrow = reinterpret_cast<const T*>(p.q) + row * p.q_tok + (int64_t)qh * p.q_head;
  for (int d = lane; d < D; d += 32) qs[warp][d] = to_f32<T>(qrow[d]);
  __syncwarp();
  T* orow = reinterpret_cast<T*>(p.out) + row * p.o_tok + (int64_t)qh * p.o_head;
  if (pos < 0 || q_len <= 0 || ctx <= 0) {  // nothing to attend: zeros, and the flag
    if (lane == 0) set_device_error(p.err, B2P_DEV_LENGTH);
    for (int d = lane; d < D; d += 32) orow[d] = from_f32<T>(0.f);
    return;
  }
  float m = -INFINITY, l = 0.f;
  float acc[kMaxD / 32];
#pragma unroll
  for (int k = 0; k < kMaxD / 32; ++k) acc[k] = 0.f;
  const int32_t* bt = p.block_tables + (int64_t)seq * p.bt_stride;
  const int64_t reach = p.bt_stride * p.block_size;  // what the table's row names
  const int nkeys = (int)min((int64_t)pos + 1, reach);
  if (pos >= reach && lane == 0) set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
  for (int base = 0; base < nkeys; base += 32) {
    const int t = base + lane;
    float s = -INFINITY, vs = 0.f;
    int64_t slot = -1;
    if (t < nkeys) {
      const int64_t col = t / p.block_size;
      const int32_t blk = col < p.bt_stride ? __ldg(bt + col) : -1;
      if (blk < 0 || blk >= p.num_blocks) {
        set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
      } else {
        slot = (int64_t)blk * p.block_size + t % p.block_size;
        const uint8_t* krow = p.k_cache + slot * p.row_elems + (int64_t)kvh * D;
        float dot = 0.f;
        for (int d = 0; d < D; d += 8) {
          const uint2 raw = __ldg(reinterpret_cast<const uint2*>(krow + d));
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dot = fmaf(qs[warp][d + e], fp8_value((uint8_t)((e < 4 ? raw.x : raw.y) >> (8 * (e & 3)))), dot);
        }
        s = dot * __ldg(p.k_scales + (int64_t)blk * p.num_kv_heads + kvh) * p.scale;
        vs = __ldg(p.v_scales + (int64_t)blk * p.num_kv_heads + kvh);
      }
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.f : mn;  // no valid key so far
    const float alpha = __expf(m - ref);
    const float pr = slot < 0 ? 0.f : __expf(s - ref);
    float ps = pr;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
    l = l * alpha + ps;
    m = mn;
#pragma unroll
    for (int k = 0; k < kMaxD / 32; ++k) acc[k] *= alpha;
    const int cnt = min(32, nkeys - base);
    const float pv = pr * vs;
    for (int j = 0; j < cnt; ++j) {
      const float pj = __shfl_sync(0xffffffffu, pv, j);
      const int64_t sj = __shfl_sync(0xffffffffu, slot, j);
      if (sj < 0) continue;
      const uint8_t* vrow = p.v_cache + sj * p.row_elems + (int64_t)kvh * D;
#pragma unroll
      for (int k = 0; k < kMaxD / 32; ++k) {
        const int d = lane + 32 * k;
        if (d < D) acc[k] = fmaf(pj, fp8_value(__ldg(vrow + d)), acc[k]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int k = 0; k < kMaxD / 32; ++k) {
    const int d = lane + 32 * k;
    if (d < D) orow[d] = value_as<T>(acc[k] * inv);
  }
}

}  // namespace

// num_rows: rows of q (and out); cu_q null means one row per sequence.
int b2p_attn_fp8_simt(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                      const void* key_cache, const void* value_cache, const float* key_scales,
                      const float* value_scales, int64_t layer_index, int64_t num_slots,
                      const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_q,
                      const int32_t* context_lens, int num_seqs, int64_t num_rows, int num_q_heads,
                      int num_kv_heads, int head_dim, int block_size, float scale, void* out,
                      int64_t out_tok_stride, int64_t out_head_stride, int dtype,
                      int32_t* err_flag, void* stream) {
  if (head_dim > kMaxD || head_dim % 8 != 0 || num_rows > 0x7fffffffLL) return B2P_EUNSUPPORTED;
  SimtFp8Params p;
  p.q = static_cast<const uint8_t*>(q);
  p.q_tok = q_tok_stride;
  p.q_head = q_head_stride;
  p.row_elems = (int64_t)num_kv_heads * head_dim;
  p.num_blocks = num_slots / block_size;
  p.k_cache = static_cast<const uint8_t*>(key_cache) + layer_index * num_slots * p.row_elems;
  p.v_cache = static_cast<const uint8_t*>(value_cache) + layer_index * num_slots * p.row_elems;
  p.k_scales = key_scales + layer_index * p.num_blocks * num_kv_heads;
  p.v_scales = value_scales + layer_index * p.num_blocks * num_kv_heads;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.cu_q = cu_q;
  p.context_lens = context_lens;
  p.num_seqs = num_seqs;
  p.num_rows = num_rows;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.scale = scale;
  p.out = static_cast<uint8_t*>(out);
  p.o_tok = out_tok_stride;
  p.o_head = out_head_stride;
  p.err = err_flag;
  const dim3 grid((unsigned)num_rows, (unsigned)((num_q_heads + kWarps - 1) / kWarps));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B2P_BF16)
    paged_attn_fp8_simt<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(p);
  else if (dtype == B2P_F16)
    paged_attn_fp8_simt<__half><<<grid, kWarps * 32, 0, s>>>(p);
  else
    paged_attn_fp8_simt<float><<<grid, kWarps * 32, 0, s>>>(p);
  return b2p_host::check_launch();
}
