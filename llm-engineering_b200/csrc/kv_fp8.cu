// K7 — rows into and out of the 8-bit KV cache (the format is described in fp8.cuh).
//
// b2p_kv_write_fp8: sequence i of a packed batch appends its q_len_i rows at positions
// ctx_i - q_len_i .. ctx_i - 1, found through its block table. One scale covers a block's
// rows of one head, so the unit of work is not a row but a (sequence, touched block, head):
// with every row of the block in one warp's hands, the largest magnitude, the scale and the
// codes come from one pass over the new rows and need no atomics. Of the blocks that a
// sequence touches only the first can hold older rows; where the new rows need a larger
// scale there, the older codes are rounded to it in the same pass.
//   e_new = max(e_old if the write leaves the block's first slot alone, e(amax of the new rows))
// The work is pure streaming: every new row is read once, its codes are written once.
#include "fp8.cuh"

namespace {

using namespace b2p;

struct WriteFp8Params {
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_tok, k_head, v_tok, v_head;  // element strides
  uint8_t* k_cache;                      // base of the selected layer
  uint8_t* v_cache;
  float* k_scales;  // base of the selected layer, [num_blocks, num_kv_heads]
  float* v_scales;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* cu;
  const int32_t* ctx;
  int64_t num_rows, num_blocks;
  int num_seqs, max_q_len, touched, hkv, d, block_size;
  int32_t* err;
};

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// One warp: the rows [row0, row0 + n) of one head into slots off0 .. off0 + n - 1 of a block.
template <typename T>
__device__ void write_block_head(const T* src, int64_t tok, uint8_t* dst, int64_t row_bytes,
                                 float* scale, int d, int off0, int n, int lane) {
  float amax = 0.f;
  bool bad = false;
  for (int i = lane; i < n * d; i += 32) {
    const float x = to_f32<T>(src[(int64_t)(i / d) * tok + i % d]);
    bad |= fp8_bad(x);
    amax = fmaxf(amax, fabsf(x));
  }
  amax = warp_max(amax);
  bad = __any_sync(0xffffffffu, bad);
  float old = 0.f;
  if (off0 > 0) old = *scale;  // one address: every lane sees the same value
  __syncwarp();
  bad |= off0 > 0 && !(old <= 3.402823466e38f);
  const float s = bad ? 1.f : fmaxf(exp2_int(fp8_block_exp(fminf(amax, kFp8Saturate))), old);
  if (off0 > 0 && !bad && s != old) {
    const float shift = old / s;  // a power of two, at most 1/2
    for (int i = lane; i < off0 * d; i += 32) {
      uint8_t* c = dst + (int64_t)(i / d) * row_bytes + i % d;
      *c = fp8_code(fp8_value(*c), shift);
    }
  }
  const float inv = 1.f / s;
  for (int i = lane; i < n * d; i += 32) {
    const float x = to_f32<T>(src[(int64_t)(i / d) * tok + i % d]);
    dst[(int64_t)(off0 + i / d) * row_bytes + i % d] = bad ? 0 : fp8_code(x, inv);
  }
  if (lane == 0) *scale = bad ? __int_as_float(0x7fffffff) : s;
}

template <typename T>
__global__ void __launch_bounds__(128) kv_write_fp8_rows(const WriteFp8Params p) {
  const int lane = threadIdx.x & 31;
  const int64_t per_seq = (int64_t)p.touched * p.hkv * 2;
  const int64_t total = per_seq * p.num_seqs;
  for (int64_t w = blockIdx.x * 4ll + (threadIdx.x >> 5); w < total; w += gridDim.x * 4ll) {
    const int seq = (int)(w / per_seq);
    const int r = (int)(w - seq * per_seq);
    const int j = r / (2 * p.hkv), h = (r >> 1) % p.hkv;
    const bool is_v = r & 1;
    const int q0 = __ldg(p.cu + seq), q1 = __ldg(p.cu + seq + 1), ctx = __ldg(p.ctx + seq);
    const int qlen = q1 - q0;
    if (qlen <= 0) continue;
    if (qlen > p.max_q_len || ctx < qlen || q0 < 0 || q1 > p.num_rows) {
      if (lane == 0) set_device_error(p.err, B2P_DEV_LENGTH);
      continue;
    }
    const int start = ctx - qlen;  // position of the first new row
    const int b = start / p.block_size + j;
    const int lo = max(start, b * p.block_size);
    const int hi = (int)min((int64_t)ctx, (int64_t)(b + 1) * p.block_size);
    if (lo >= hi) continue;
    const int32_t blk = b < p.bt_stride ? __ldg(p.block_tables + (int64_t)seq * p.bt_stride + b) : -1;
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane == 0) set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
      continue;
    }
    const int64_t row_bytes = (int64_t)p.hkv * p.d;
    uint8_t* dst = (is_v ? p.v_cache : p.k_cache) + (int64_t)blk * p.block_size * row_bytes + (int64_t)h * p.d;
    float* scale = (is_v ? p.v_scales : p.k_scales) + (int64_t)blk * p.hkv + h;
    const int64_t row = q0 + (lo - start);
    const T* src = reinterpret_cast<const T*>(is_v ? p.v : p.k) +
                   (is_v ? row * p.v_tok + h * p.v_head : row * p.k_tok + h * p.k_head);
    write_block_head<T>(src, is_v ? p.v_tok : p.k_tok, dst, row_bytes, scale, p.d,
                        lo - b * p.block_size, hi - lo, lane);
  }
}

struct ReadFp8Params {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scales;
  const float* v_scales;
  const int32_t* slots;
  uint8_t* k;
  uint8_t* v;
  int64_t num_rows, num_slots;
  int hkv, d, block_size;
  int32_t* err;
};

// One thread per 8 codes of a row (head_dim is a multiple of 8).
template <typename T>
__global__ void __launch_bounds__(256) kv_read_fp8(const ReadFp8Params p) {
  const int64_t per_row = (int64_t)p.hkv * p.d / 8;
  const int64_t total = p.num_rows * per_row * 2;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / (per_row * 2);
    const int64_t rem = i - row * per_row * 2;
    const bool is_v = rem >= per_row;
    const int c = (int)(is_v ? rem - per_row : rem);
    const int32_t slot = __ldg(p.slots + row);
    T* out = reinterpret_cast<T*>(is_v ? p.v : p.k) + row * per_row * 8 + c * 8;
    if (slot >= p.num_slots && c == 0 && !is_v) set_device_error(p.err, B2P_DEV_SLOT_RANGE);
    const bool have = slot >= 0 && slot < p.num_slots;
    uint2 raw = make_uint2(0u, 0u);
    float s = 0.f;
    if (have) {
      raw = __ldg(reinterpret_cast<const uint2*>((is_v ? p.v_cache : p.k_cache) + slot * per_row * 8) + c);
      s = __ldg((is_v ? p.v_scales : p.k_scales) + (int64_t)(slot / p.block_size) * p.hkv + c * 8 / p.d);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t code = (uint8_t)((e < 4 ? raw.x : raw.y) >> (8 * (e & 3)));
      out[e] = from_f32<T>(fp8_value(code) * s);
    }
  }
}

int element_size(int dtype) {
  return dtype == B2P_F32 ? 4 : dtype == B2P_BF16 || dtype == B2P_F16 ? 2 : 0;
}

}  // namespace

extern "C" int b2p_kv_write_fp8(const void* keys, int64_t k_tok_stride, int64_t k_head_stride,
                                const void* values, int64_t v_tok_stride, int64_t v_head_stride,
                                void* key_cache, void* value_cache, float* key_scales,
                                float* value_scales, const int32_t* block_tables,
                                int64_t block_table_stride, const int32_t* cu_seqlens_q,
                                const int32_t* context_lens, int num_seqs, int64_t num_rows,
                                int max_q_len, int64_t layer_index, int64_t num_layers,
                                int64_t num_slots, int num_kv_heads, int head_dim, int block_size,
                                int dtype, int32_t* err_flag, void* stream) {
  if (num_seqs < 0 || num_rows < 0 || max_q_len < 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      block_size <= 0 || num_slots <= 0 || num_layers <= 0 || num_slots % block_size != 0 ||
      block_table_stride < 0)
    return B2P_EINVAL;
  if (layer_index < 0 || layer_index >= num_layers) return B2P_ERANGE;
  if (element_size(dtype) == 0 || head_dim % 8 != 0 || num_slots > 0x7fffffffLL)
    return B2P_EUNSUPPORTED;
  if (num_seqs == 0 || num_rows == 0 || max_q_len == 0) return B2P_OK;
  if (!keys || !values || !key_cache || !value_cache || !key_scales || !value_scales ||
      !block_tables || !cu_seqlens_q || !context_lens)
    return B2P_EINVAL;
  WriteFp8Params p;
  p.k = static_cast<const uint8_t*>(keys);
  p.v = static_cast<const uint8_t*>(values);
  p.k_tok = k_tok_stride;
  p.k_head = k_head_stride;
  p.v_tok = v_tok_stride;
  p.v_head = v_head_stride;
  const int64_t layer_bytes = num_slots * num_kv_heads * head_dim;
  p.num_blocks = num_slots / block_size;
  p.k_cache = static_cast<uint8_t*>(key_cache) + layer_index * layer_bytes;
  p.v_cache = static_cast<uint8_t*>(value_cache) + layer_index * layer_bytes;
  p.k_scales = key_scales + layer_index * p.num_blocks * num_kv_heads;
  p.v_scales = value_scales + layer_index * p.num_blocks * num_kv_heads;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.cu = cu_seqlens_q;
  p.ctx = context_lens;
  p.num_seqs = num_seqs;
  p.num_rows = num_rows;
  p.max_q_len = max_q_len;
  p.touched = (int)(((int64_t)max_q_len + block_size - 2) / block_size + 1);
  p.hkv = num_kv_heads;
  p.d = head_dim;
  p.block_size = block_size;
  p.err = err_flag;
  const int64_t warps = (int64_t)num_seqs * p.touched * num_kv_heads * 2;
  const int64_t most = (int64_t)b2p_host::sm_count() * 16;
  const unsigned grid = (unsigned)((warps + 3) / 4 < most ? (warps + 3) / 4 : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B2P_BF16)
    kv_write_fp8_rows<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  else if (dtype == B2P_F16)
    kv_write_fp8_rows<__half><<<grid, 128, 0, s>>>(p);
  else
    kv_write_fp8_rows<float><<<grid, 128, 0, s>>>(p);
  return b2p_host::check_launch();
}

extern "C" int b2p_kv_read_fp8(const void* key_cache, const void* value_cache,
                               const float* key_scales, const float* value_scales,
                               const int32_t* slot_mapping, int64_t num_rows, void* keys,
                               void* values, int64_t layer_index, int64_t num_layers,
                               int64_t num_slots, int num_kv_heads, int head_dim, int block_size,
                               int dtype, int32_t* err_flag, void* stream) {
  if (num_rows < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_slots <= 0 ||
      num_layers <= 0 || num_slots % block_size != 0)
    return B2P_EINVAL;
  if (layer_index < 0 || layer_index >= num_layers) return B2P_ERANGE;
  if (element_size(dtype) == 0 || head_dim % 8 != 0 || num_slots > 0x7fffffffLL)
    return B2P_EUNSUPPORTED;
  if (num_rows == 0) return B2P_OK;
  if (!key_cache || !value_cache || !key_scales || !value_scales || !slot_mapping || !keys || !values)
    return B2P_EINVAL;
  if ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) & 7u)
    return B2P_EINVAL;
  ReadFp8Params p;
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  const int64_t num_blocks = num_slots / block_size;
  p.k_cache = static_cast<const uint8_t*>(key_cache) + layer_index * num_slots * row;
  p.v_cache = static_cast<const uint8_t*>(value_cache) + layer_index * num_slots * row;
  p.k_scales = key_scales + layer_index * num_blocks * num_kv_heads;
  p.v_scales = value_scales + layer_index * num_blocks * num_kv_heads;
  p.slots = slot_mapping;
  p.k = static_cast<uint8_t*>(keys);
  p.v = static_cast<uint8_t*>(values);
  p.num_rows = num_rows;
  p.num_slots = num_slots;
  p.hkv = num_kv_heads;
  p.d = head_dim;
  p.block_size = block_size;
  p.err = err_flag;
  const int64_t items = num_rows * (row / 8) * 2;
  const int64_t most = (int64_t)b2p_host::sm_count() * 16;
  const unsigned grid = (unsigned)((items + 255) / 256 < most ? (items + 255) / 256 : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B2P_BF16)
    kv_read_fp8<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
  else if (dtype == B2P_F16)
    kv_read_fp8<__half><<<grid, 256, 0, s>>>(p);
  else
    kv_read_fp8<float><<<grid, 256, 0, s>>>(p);
  return b2p_host::check_launch();
}
