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
// The work is pure streaming: every new row is read once, its codes are written once. A warp holds
// its rows in registers between the two (16 rows of 128 take 8 16-byte pieces a lane); where they
// do not fit it reads them again, from L2.
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
  bool vec;   // every row of keys and values starts on a 16-byte boundary
  bool seek;  // units are the touched blocks alone, found by a scan of the lengths
  int32_t* err;
};

// Eight elements of a row: values, and the running maximum of their magnitudes as bits (magnitudes
// of floats are ordered as their bits are; infinities and NaN come out on top).
template <typename T>
struct Piece {  // bf16, f16
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void max_bits(uint32_t& m) const {
    m = __vmaxu2(m, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
  }
  __device__ static __forceinline__ float magnitude(uint32_t m) {
    const uint16_t b = (uint16_t)max(m & 0xffffu, m >> 16);
    return to_f32<T>(*reinterpret_cast<const T*>(&b));
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t b = (uint16_t)(in[i >> 1] >> (16 * (i & 1)));
      x[i] = to_f32<T>(*reinterpret_cast<const T*>(&b));
    }
  }
};

template <>
struct Piece<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void max_bits(uint32_t& m) const {
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  }
  __device__ static __forceinline__ float magnitude(uint32_t m) { return __uint_as_float(m); }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};

// Four codes of x * inv, ties to even.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
  const uint16_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
  const uint16_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inv, d * inv), __NV_SATFINITE, __NV_E4M3);
  return lo | (uint32_t)hi << 16;
}

template <typename T>
__device__ __forceinline__ uint2 codes8(const Piece<T>& p, float inv, bool clamp) {
  float x[8];
  p.values(x);
  if (clamp) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -kFp8Saturate), kFp8Saturate);
  }
  return make_uint2(codes4(x[0], x[1], x[2], x[3], inv), codes4(x[4], x[5], x[6], x[7], inv));
}

// The block's scale from the largest magnitude of its new rows; NaN where a row is not finite or
// the scale it keeps already is. `old` counts where the write leaves the block's first slot alone.
__device__ __forceinline__ float new_scale(float amax, float old, bool keep) {
  const bool bad = !(amax <= 3.402823466e38f) || (keep && !(old <= 3.402823466e38f));
  if (bad) return __int_as_float(0x7fffffff);
  const float s = exp2_int(fp8_block_exp(fminf(amax, kFp8Saturate)));
  return keep ? fmaxf(s, old) : s;
}

// The codes of the block's older rows, rounded to the larger scale.
__device__ __forceinline__ void rescale(uint8_t* dst, int64_t row_bytes, int d, int rows, float shift, int lane) {
  const int per_row = d / 8;
  for (int i = lane; i < rows * per_row; i += 32) {
    uint2* at = reinterpret_cast<uint2*>(dst + (int64_t)(i / per_row) * row_bytes) + i % per_row;
    const uint2 w = *at;
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = fp8_value((uint8_t)((k < 4 ? w.x : w.y) >> (8 * (k & 3))));
    *at = make_uint2(codes4(x[0], x[1], x[2], x[3], shift), codes4(x[4], x[5], x[6], x[7], shift));
  }
}

constexpr int kHold = 8;  // pieces of eight elements that a lane keeps

// One warp: n rows of one head into slots off0 .. off0 + n - 1 of a block, by 16-byte pieces. kD:
// the head dim where it is known, which spares the divisions by a row's pieces (32 prompts written
// and read back: 40.7 us against 45.5), 0 otherwise.
template <typename T, int kD>
__device__ void write_block_vec(const T* src, int64_t tok, uint8_t* dst, int64_t row_bytes,
                                float* scale, int head_dim, int off0, int n, int lane) {
  const int d = kD != 0 ? kD : head_dim;
  const int per_row = d / 8, total = n * per_row;
  const bool keep = off0 > 0;
  const float old = keep ? *scale : 0.f;  // one address for the warp
  uint32_t m = 0;
  Piece<T> held[kHold];
  const bool fits = total <= 32 * kHold;
  auto at = [&](int i) { return src + (int64_t)(i / per_row) * tok + (i % per_row) * 8; };
  if (fits) {
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (lane + 32 * k < total) held[k].load(at(lane + 32 * k));
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (lane + 32 * k < total) held[k].max_bits(m);
  } else {
    for (int i = lane; i < total; i += 32) {
      held[0].load(at(i));
      held[0].max_bits(m);
    }
  }
  const float amax = Piece<T>::magnitude(m);
  // bits again: __reduce_max_sync orders NaN and infinities above every number
  const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
  const float s = new_scale(top, old, keep);
  const bool bad = s != s;
  if (keep && !bad && s != old) rescale(dst, row_bytes, d, off0, old / s, lane);
  const float inv = bad ? 0.f : 1.f / s;
  const bool clamp = top > kFp8Saturate;
  auto put = [&](int i, const Piece<T>& p) {
    const uint2 c = bad ? make_uint2(0u, 0u) : codes8<T>(p, inv, clamp);
    reinterpret_cast<uint2*>(dst + (int64_t)(off0 + i / per_row) * row_bytes)[i % per_row] = c;
  };
  if (fits) {
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (lane + 32 * k < total) put(lane + 32 * k, held[k]);
  } else {
    for (int i = lane; i < total; i += 32) {
      held[0].load(at(i));
      put(i, held[0]);
    }
  }
  if (lane == 0) *scale = s;
}

// The same by single elements, for rows that are not 16-byte aligned.
template <typename T>
__device__ void write_block_elem(const T* src, int64_t tok, uint8_t* dst, int64_t row_bytes,
                                 float* scale, int d, int off0, int n, int lane) {
  const bool keep = off0 > 0;
  const float old = keep ? *scale : 0.f;
  uint32_t m = 0;
  for (int i = lane; i < n * d; i += 32)
    m = max(m, __float_as_uint(to_f32<T>(src[(int64_t)(i / d) * tok + i % d])) & 0x7fffffffu);
  const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, m));
  const float s = new_scale(top, old, keep);
  const bool bad = s != s;
  if (keep && !bad && s != old) rescale(dst, row_bytes, d, off0, old / s, lane);
  const float inv = bad ? 0.f : 1.f / s;
  for (int i = lane; i < n * d; i += 32) {
    const float x = to_f32<T>(src[(int64_t)(i / d) * tok + i % d]);
    dst[(int64_t)(off0 + i / d) * row_bytes + i % d] = bad ? 0 : fp8_code(x, inv);
  }
  if (lane == 0) *scale = s;
}

// What a sequence appends: rows q0 .. q0 + qlen - 1 at positions start ..; qlen 0: nothing, or
// refused.
struct Append {
  int q0, qlen, start;
};

__device__ __forceinline__ Append append_of(const WriteFp8Params& p, int seq) {
  const int q0 = __ldg(p.cu + seq), q1 = __ldg(p.cu + seq + 1), ctx = __ldg(p.ctx + seq);
  Append a{q0, q1 - q0, ctx - (q1 - q0)};
  if (a.qlen < 0 || a.qlen > p.max_q_len || a.start < 0 || q0 < 0 || q1 > p.num_rows) {
    set_device_error(p.err, B2P_DEV_LENGTH);
    a.qlen = 0;
  }
  return a;
}

__device__ __forceinline__ int touched_blocks(const Append& a, int block_size) {
  return a.qlen <= 0 ? 0 : (a.start + a.qlen - 1) / block_size - a.start / block_size + 1;
}

// A unit is (sequence, touched block, head, K or V), one per warp and round.
template <typename T, int kD>
__global__ void __launch_bounds__(128) kv_write_fp8_rows(const WriteFp8Params p) {
  // The attention that follows may start its look at lengths and tables, which this kernel does
  // not write, while it runs; it waits for this grid's end before it touches the pool.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int per_block = 2 * p.hkv;
  const int64_t per_seq = (int64_t)p.touched * per_block;
  for (int64_t u = blockIdx.x * 4ll + (threadIdx.x >> 5);; u += gridDim.x * 4ll) {
    int seq, j;
    const int r = (int)(u % per_block), h = r >> 1;
    if (p.seek) {
      // the sequence that holds touched block u / per_block, 32 sequences at a time
      int64_t want = u / per_block;
      seq = -1;
      j = 0;
      for (int base = 0; base < p.num_seqs && seq < 0; base += 32) {
        const int n = base + lane < p.num_seqs ? touched_blocks(append_of(p, base + lane), p.block_size) : 0;
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
          j = (int)(want - __shfl_sync(0xffffffffu, incl - n, src));
        } else {
          want -= __shfl_sync(0xffffffffu, incl, 31);
        }
      }
      if (seq < 0) return;  // past the last touched block
    } else {
      if (u >= per_seq * p.num_seqs) return;
      seq = (int)(u / per_seq);
      j = (int)(u - seq * per_seq) / per_block;
    }
    const Append a = append_of(p, seq);
    if (a.qlen <= 0) continue;
    const bool is_v = r & 1;
    const int ctx = a.start + a.qlen;
    const int b = a.start / p.block_size + j;
    const int lo = max(a.start, b * p.block_size);
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
    const int64_t row = a.q0 + (lo - a.start);
    const T* src = reinterpret_cast<const T*>(is_v ? p.v : p.k) +
                   (is_v ? row * p.v_tok + h * p.v_head : row * p.k_tok + h * p.k_head);
    const int off0 = lo - b * p.block_size;
    if (p.vec)
      write_block_vec<T, kD>(src, is_v ? p.v_tok : p.k_tok, dst, row_bytes, scale, p.d, off0, hi - lo, lane);
    else
      write_block_elem<T>(src, is_v ? p.v_tok : p.k_tok, dst, row_bytes, scale, p.d, off0, hi - lo, lane);
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

// A warp takes kReadRows rows at a time, a lane 8 codes of each of them (head_dim is a multiple of
// 8): the rows' slots come in one load, then all their codes and scales are in flight together.
constexpr int kReadRows = 4;

template <typename T>
__global__ void __launch_bounds__(256) kv_read_fp8_rows(const ReadFp8Params p) {
  const int per_row = p.hkv * p.d / 8, per_head = p.d / 8;
  const int lane = threadIdx.x & 31;
  for (int64_t row0 = (blockIdx.x * 8ll + (threadIdx.x >> 5)) * kReadRows; row0 < p.num_rows;
       row0 += gridDim.x * 8ll * kReadRows) {
    int32_t mine = -1;
    if (lane < kReadRows && row0 + lane < p.num_rows) {
      mine = __ldg(p.slots + row0 + lane);
      if (mine >= p.num_slots) {
        set_device_error(p.err, B2P_DEV_SLOT_RANGE);
        mine = -1;
      }
    }
    const int my_block = mine < 0 ? 0 : mine / p.block_size;
    int32_t slot[kReadRows], block[kReadRows];
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
      slot[k] = __shfl_sync(0xffffffffu, mine, k);
      block[k] = __shfl_sync(0xffffffffu, my_block, k);
    }
    for (int i = lane; i < 2 * per_row; i += 32) {
      const bool is_v = i >= per_row;
      const int c = is_v ? i - per_row : i, h = c / per_head;
      const uint2* codes = reinterpret_cast<const uint2*>(is_v ? p.v_cache : p.k_cache) + c;
      const float* scales = (is_v ? p.v_scales : p.k_scales) + h;
      uint2 raw[kReadRows];
      float s[kReadRows];
#pragma unroll
      for (int k = 0; k < kReadRows; ++k) {
        raw[k] = make_uint2(0u, 0u);
        s[k] = 0.f;
        if (slot[k] >= 0) {
          raw[k] = __ldg(codes + (int64_t)slot[k] * per_row);
          s[k] = __ldg(scales + (int64_t)block[k] * p.hkv);
        }
      }
#pragma unroll
      for (int k = 0; k < kReadRows; ++k) {
        if (row0 + k >= p.num_rows) break;
        T* out = reinterpret_cast<T*>(is_v ? p.v : p.k) + ((row0 + k) * per_row + c) * 8;
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t two = fp8x2_to_f16x2((uint16_t)((e < 2 ? raw[k].x : raw[k].y) >> (16 * (e & 1))));
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&two));
          x[2 * e] = v.x * s[k];
          x[2 * e + 1] = v.y * s[k];
        }
        if constexpr (sizeof(T) == 4) {
          reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
          reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
          *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]),
                                                      pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
        }
      }
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
  if ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) & 7u)
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
  const int es = element_size(dtype);
  p.vec = ((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values) | (uintptr_t)(k_tok_stride * es) |
            (uintptr_t)(k_head_stride * es) | (uintptr_t)(v_tok_stride * es) | (uintptr_t)(v_head_stride * es)) & 15u) == 0;
  // Units by (sequence, block number) where every sequence touches about as many blocks as the
  // longest may; in a batch of unlike lengths most of those are empty (32 prompts of 64 to 8192
  // tokens: 4 of 5, 46 us), and the touched ones are found by a scan instead.
  const int64_t direct = (int64_t)num_seqs * p.touched;
  const int64_t bound = num_rows / block_size + 2ll * num_seqs;
  p.seek = direct > 2 * bound;
  const int64_t warps = (p.seek ? bound : direct) * num_kv_heads * 2;
  const int64_t most = (int64_t)b2p_host::sm_count() * 16;
  const unsigned grid = (unsigned)((warps + 3) / 4 < most ? (warps + 3) / 4 : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int kind = head_dim == 128 ? 2 : head_dim == 64 ? 1 : 0;
  void (*const fns[3][3])(WriteFp8Params) = {
      {kv_write_fp8_rows<__nv_bfloat16, 0>, kv_write_fp8_rows<__nv_bfloat16, 64>, kv_write_fp8_rows<__nv_bfloat16, 128>},
      {kv_write_fp8_rows<__half, 0>, kv_write_fp8_rows<__half, 64>, kv_write_fp8_rows<__half, 128>},
      {kv_write_fp8_rows<float, 0>, kv_write_fp8_rows<float, 64>, kv_write_fp8_rows<float, 128>}};
  fns[dtype][kind]<<<grid, 128, 0, s>>>(p);
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
  if (((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) & 7u) ||
      ((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) & 15u))
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
  const int64_t want = (num_rows + 8 * kReadRows - 1) / (8 * kReadRows);
  const int64_t most = (int64_t)b2p_host::sm_count() * 16;
  const unsigned grid = (unsigned)(want < most ? want : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B2P_BF16)
    kv_read_fp8_rows<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
  else if (dtype == B2P_F16)
    kv_read_fp8_rows<__half><<<grid, 256, 0, s>>>(p);
  else
    kv_read_fp8_rows<float><<<grid, 256, 0, s>>>(p);
  return b2p_host::check_launch();
}
