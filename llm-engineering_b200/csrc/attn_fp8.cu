// Entry points of attention over the 8-bit KV cache: b2p_paged_decode_fp8 (one query row per
// sequence) and b2p_paged_prefill_fp8 (q_len_i rows, causal: the rows of drafted tokens, of
// prompt slices and of whole prompts).
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

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Pool rows fit TMA boxes, query rows 8-byte loads, output rows 4-byte stores.
bool rows_fit(const void* q, int64_t q_tok, int64_t q_head, const void* kc, const void* vc,
              const void* out, int64_t o_tok, int64_t o_head) {
  return aligned(q, 8) && q_tok % 4 == 0 && q_head % 4 == 0 && aligned(kc, 16) && aligned(vc, 16) &&
         aligned(out, 4) && o_tok % 2 == 0 && o_head % 2 == 0;
}

int check_args(const void* key_cache, const void* value_cache, int64_t layer_index, int64_t num_layers, int64_t num_slots, int num_seqs,
               int64_t num_rows, int max_q_len, int num_q_heads, int num_kv_heads, int head_dim,
               int block_size, int64_t block_table_stride, int dtype) {
  if (num_seqs < 0 || num_rows < 0 || max_q_len < 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      head_dim <= 0 || block_size <= 0 || num_slots <= 0 || num_layers <= 0 ||
      block_table_stride < 0)
    return B2P_EINVAL;
  if (num_q_heads % num_kv_heads != 0 || num_slots % block_size != 0) return B2P_EINVAL;
  if (dtype < B2P_BF16 || dtype > B2P_F32) return B2P_EINVAL;
  if (layer_index < 0 || layer_index >= num_layers) return B2P_ERANGE;
  if ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) & 7u)
    return B2P_EINVAL;
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
  const int rc = check_args(key_cache, value_cache, layer_index, num_layers, num_slots, num_seqs, num_seqs, 1, num_q_heads,
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

extern "C" int b2p_paged_prefill_fp8(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                     const void* key_cache, const void* value_cache,
                                     const float* key_scales, const float* value_scales,
                                     int64_t layer_index, int64_t num_layers, int64_t num_slots,
                                     const int32_t* block_tables, int64_t block_table_stride,
                                     const int32_t* cu_seqlens_q, const int32_t* context_lens,
                                     int num_seqs, int64_t total_q, int max_q_len, int num_q_heads,
                                     int num_kv_heads, int head_dim, int block_size, float scale,
                                     void* out, int64_t out_tok_stride, int64_t out_head_stride,
                                     void* workspace, size_t workspace_size, int dtype,
                                     int32_t* err_flag, void* stream) {
  const int rc = check_args(key_cache, value_cache, layer_index, num_layers, num_slots, num_seqs, total_q, max_q_len,
                            num_q_heads, num_kv_heads, head_dim, block_size, block_table_stride,
                            dtype);
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
  if (dtype != B2P_F32) b2p_host::note_fallback(3);
  return b2p_attn_fp8_simt(q, q_tok_stride, q_head_stride, key_cache, value_cache, key_scales,
                           value_scales, layer_index, num_slots, block_tables, block_table_stride,
                           cu_seqlens_q, context_lens, num_seqs, total_q, num_q_heads,
                           num_kv_heads, head_dim, block_size, scale, out, out_tok_stride,
                           out_head_stride, dtype, err_flag, stream);
}
