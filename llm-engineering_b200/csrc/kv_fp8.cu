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
// Every new row is read once, its codes are written once. A warp holds its rows in registers
// between the two (16 rows of 128 take 8 16-byte pieces a lane); where they do not fit it reads them
// again, from L2, piece by piece: 53,400 rows of 2 x 128 in bf16 take 22.6 us with blocks of 16 tokens,
// 36.9 with 32 and 39.5 with 64 (d 64: 14.4 with 32, 20.6 with 64); in fp32 29.2 with 16, 53.7 with 32.
#include <type_traits>

#include "fp8.cuh"

namespace {

using namespace b2p;

constexpr int kWriteThreads = 128;
template <typename T>
constexpr int kWriteCtas = sizeof(T) == 4 ? 4 : 6;  // CTAs of the write per SM

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
  int num_seqs, max_q_len, hkv, d, block_size;
  unsigned touched;  // blocks that a sequence may touch
  int block_warps;
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

// What turns a block's values into codes: inv = 2^-e. Where `packed`, 16-bit values are multiplied in
// pairs in their own type: a power of two leaves their bits alone except below the normal range
// (f16: 2^-14), where the code is zero either way (e4m3 rounds to zero up to 2^-10).
struct Coder {
  float inv;
  bool clamp;     // some value is above kFp8Saturate
  bool packed;
  uint32_t inv2;  // a pair of inv in the values' type
};

template <typename T>
__device__ __forceinline__ Coder coder_of(float s, float top) {
  Coder c;
  c.inv = 1.f / s;
  c.clamp = top > kFp8Saturate;
  c.inv2 = pack2<T>(c.inv, c.inv);
  // f16 holds 2^-24 to 2^15; a scale kept from rows that another program wrote may be no power of two
  c.packed = !c.clamp && (__float_as_uint(c.inv) & 0x7fffffu) == 0 &&
             (std::is_same<T, __nv_bfloat16>::value || (c.inv <= 0x1p15f && c.inv >= 0x1p-24f));
  return c;
}
template <>
__device__ __forceinline__ Coder coder_of<float>(float s, float top) {
  return Coder{1.f / s, top > kFp8Saturate, false, 0u};
}

__device__ __forceinline__ uint16_t codes2_packed(uint32_t w, uint32_t inv2, __half) {
  const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&inv2));
  return __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(y), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint16_t codes2_packed(uint32_t w, uint32_t inv2, __nv_bfloat16) {
  const __nv_bfloat162 y =
      __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&inv2));
  const uint32_t b = *reinterpret_cast<const uint32_t*>(&y);
  return __nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)),
                                  __NV_SATFINITE, __NV_E4M3);
}

template <typename T>
__device__ __forceinline__ uint2 codes8(const Piece<T>& p, const Coder& c) {
  if constexpr (sizeof(T) == 2) {
    if (c.packed) {
      const uint32_t in[4] = {p.w.x, p.w.y, p.w.z, p.w.w};
      uint32_t two[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) two[i] = codes2_packed(in[i], c.inv2, T());
      return make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
    }
  }
  float x[8];
  p.values(x);
  if (c.clamp) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -kFp8Saturate), kFp8Saturate);
  }
  return make_uint2(codes4(x[0], x[1], x[2], x[3], c.inv), codes4(x[4], x[5], x[6], x[7], c.inv));
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

// n rows of one head for slots off0 .. off0 + n - 1 of a block.
template <typename T>
struct Target {
  const T* src;
  uint8_t* dst;  // slot 0 of the block
  float* scale;
  int64_t tok;
  int off0, n;
};

// One warp writes a target, by 16-byte pieces: load() sends for the rows, finish() does the rest.
// kD: the head dim where it is known and a row's pieces divide the warp's lanes, 0 otherwise. Then
// a lane's pieces are one column of every 256 / kD-th row, and neither divisions nor bounds on
// pieces are left.
template <typename T, int kD>
struct BlockWriter {
  static constexpr int kStep = kD != 0 ? 256 / kD : 1;  // rows from one of a lane's pieces to its next
  int lane, per_row, row0, col;
  int64_t row_bytes;
  Piece<T> held[kHold];
  float old;

  __device__ __forceinline__ BlockWriter(int head_dim, int64_t row_bytes)
      : lane(threadIdx.x & 31), per_row((kD != 0 ? kD : head_dim) / 8), row0(kD != 0 ? lane / per_row : 0),
        col(kD != 0 ? lane % per_row : 0), row_bytes(row_bytes) {}
  __device__ __forceinline__ bool fits(const Target<T>& t) const { return t.n * per_row <= 32 * kHold; }
  __device__ __forceinline__ bool have(const Target<T>& t, int k) const {
    return kD != 0 ? row0 + k * kStep < t.n : lane + 32 * k < t.n * per_row;
  }
  __device__ __forceinline__ const T* from(const Target<T>& t, int k) const {
    if (kD != 0) return t.src + (row0 + k * kStep) * t.tok + col * 8;
    const int i = lane + 32 * k;
    return t.src + (i / per_row) * t.tok + (i % per_row) * 8;
  }
  __device__ __forceinline__ uint2* to(const Target<T>& t, int k) const {
    if (kD != 0) return reinterpret_cast<uint2*>(t.dst + (t.off0 + row0 + k * kStep) * row_bytes) + col;
    const int i = lane + 32 * k;
    return reinterpret_cast<uint2*>(t.dst + (t.off0 + i / per_row) * row_bytes) + i % per_row;
  }
  __device__ __forceinline__ void load(const Target<T>& t) {
    old = t.off0 > 0 ? *t.scale : 0.f;  // one address for the warp
    if (!fits(t)) return;
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (have(t, k)) held[k].load(from(t, k));
  }
  __device__ __forceinline__ void finish(const Target<T>& t) {
    const bool keep = t.off0 > 0, whole = fits(t);
    uint32_t m = 0;
    if (whole) {
#pragma unroll
      for (int k = 0; k < kHold; ++k)
        if (have(t, k)) held[k].max_bits(m);
    } else {
      for (int k = 0; have(t, k); ++k) {
        held[0].load(from(t, k));
        held[0].max_bits(m);
      }
    }
    const float amax = Piece<T>::magnitude(m);
    // bits again: __reduce_max_sync orders NaN and infinities above every number
    const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    const float s = new_scale(top, old, keep);
    const bool bad = s != s;
    if (keep && !bad && s != old) rescale(t.dst, row_bytes, per_row * 8, t.off0, old / s, lane);
    const Coder coder = coder_of<T>(s, top);
    auto put = [&](int k, const Piece<T>& x) { *to(t, k) = bad ? make_uint2(0u, 0u) : codes8<T>(x, coder); };
    if (whole) {
#pragma unroll
      for (int k = 0; k < kHold; ++k)
        if (have(t, k)) put(k, held[k]);
    } else {
      for (int k = 0; have(t, k); ++k) {
        held[0].load(from(t, k));
        put(k, held[0]);
      }
    }
    if (lane == 0) *t.scale = s;
  }
};

// The same by single elements, for rows that are not 16-byte aligned.
template <typename T>
__device__ __noinline__ void write_block_elem(const Target<T>& t, int64_t row_bytes, int d, int lane) {
  const T* src = t.src;
  uint8_t* dst = t.dst;
  float* scale = t.scale;
  const int64_t tok = t.tok;
  const int off0 = t.off0, n = t.n;
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

// Where a sequence's new rows meet a block: rows row .. row + n - 1 go to its slots off0 ...
struct Touched {
  int64_t row;
  int32_t block;
  int off0, n;  // n 0: nothing to do here
};

// Touched block u of the batch; false past the last one.
__device__ __forceinline__ bool find_touched(const WriteFp8Params& p, unsigned u, Touched& t) {
  const int lane = threadIdx.x & 31;
  int seq, j;
  if (p.seek) {  // the sequence that holds it, 32 sequences at a time
    int64_t want = u;
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
    if (seq < 0) return false;
  } else {
    if (u >= (unsigned)p.num_seqs * p.touched) return false;
    seq = u / p.touched;
    j = u - seq * p.touched;
  }
  t.n = 0;
  const Append a = append_of(p, seq);
  if (a.qlen <= 0) return true;
  const int ctx = a.start + a.qlen;
  const int b = a.start / p.block_size + j;
  const int lo = max(a.start, b * p.block_size);
  const int hi = (int)min((int64_t)ctx, (int64_t)(b + 1) * p.block_size);
  if (lo >= hi) return true;
  t.block = b < p.bt_stride ? __ldg(p.block_tables + (int64_t)seq * p.bt_stride + b) : -1;
  if (t.block < 0 || t.block >= p.num_blocks) {
    if (lane == 0) set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
    return true;
  }
  t.row = a.q0 + (lo - a.start);
  t.off0 = lo - b * p.block_size;
  t.n = hi - lo;
  return true;
}

// p.block_warps warps of a CTA share a touched block; a warp takes every so many of its (head, K or
// V) targets, then those of a later block. While a target's rows are on their way the warp looks
// for the next one: 53,400 f16 rows of 2 x 128 in 19.6 us against 22.5 with a search per target
// and nothing in flight meanwhile (bytes alone: 12.5 us). Six CTAs per SM; with eight the rows no
// longer fit the registers (24.6 us), with four that hold two targets each 22.0.
template <typename T, int kD>
__global__ void __launch_bounds__(kWriteThreads, kWriteCtas<T>) kv_write_fp8_rows(const WriteFp8Params p) {
  // The attention that follows may start its look at lengths and tables, which this kernel does
  // not write, while it runs; it waits for this grid's end before it touches the pool.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row_bytes = (int64_t)p.hkv * p.d;
  const unsigned per_cta = kWriteThreads / 32 / p.block_warps;
  const unsigned stride = gridDim.x * per_cta;
  unsigned u = blockIdx.x * per_cta + warp / p.block_warps;
  const int first = warp % p.block_warps;
  int c = first;
  Touched at;
  bool more = find_touched(p, u, at);
  auto settle = [&]() {  // on to a block with something to do
    while (more && at.n == 0) {
      u += stride;
      more = find_touched(p, u, at);
    }
  };
  settle();
  auto target = [&]() {
    Target<T> t;
    const int h = c >> 1;
    const bool is_v = c & 1;
    t.tok = is_v ? p.v_tok : p.k_tok;
    t.src = reinterpret_cast<const T*>(is_v ? p.v : p.k) + at.row * t.tok + h * (is_v ? p.v_head : p.k_head);
    t.dst = (is_v ? p.v_cache : p.k_cache) + (int64_t)at.block * p.block_size * row_bytes + (int64_t)h * p.d;
    t.scale = (is_v ? p.v_scales : p.k_scales) + (int64_t)at.block * p.hkv + h;
    t.off0 = at.off0;
    t.n = at.n;
    return t;
  };
  auto advance = [&]() {
    c += p.block_warps;
    if (c < 2 * p.hkv) return;
    c = first;
    u += stride;
    more = find_touched(p, u, at);
    settle();
  };
  if (p.vec) {
    BlockWriter<T, kD> writer(p.d, row_bytes);
    while (more) {
      const Target<T> t = target();
      writer.load(t);
      advance();
      writer.finish(t);
    }
  } else {
    while (more) {
      write_block_elem<T>(target(), row_bytes, p.d, lane);
      advance();
    }
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
          *reinterpret_cast<uint4*>(out) = make_uint4(pack_values<T>(x[0], x[1]), pack_values<T>(x[2], x[3]),
                                                      pack_values<T>(x[4], x[5]), pack_values<T>(x[6], x[7]));
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
  p.touched = (unsigned)(((int64_t)max_q_len + block_size - 2) / block_size + 1);
  p.hkv = num_kv_heads;
  p.d = head_dim;
  p.block_size = block_size;
  p.err = err_flag;
  const int es = element_size(dtype);
  p.vec = ((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values) | (uintptr_t)(k_tok_stride * es) |
            (uintptr_t)(k_head_stride * es) | (uintptr_t)(v_tok_stride * es) | (uintptr_t)(v_head_stride * es)) & 15u) == 0;
  // Units by (sequence, block number) where every sequence touches about as many blocks as the
  // longest may; in a batch of unlike lengths most of those are empty (32 prompts of 64 to 8192
  // tokens: 4 of 5), and the touched ones are found by a scan instead.
  const int64_t direct = (int64_t)num_seqs * p.touched;
  const int64_t bound = num_rows / block_size + 2ll * num_seqs;
  p.seek = direct > 2 * bound;
  const int64_t units = p.seek ? bound : direct;
  if (units > 0x3fffffffLL) return B2P_EUNSUPPORTED;
  p.block_warps = num_kv_heads == 1 ? 2 : 4;
  const int per_cta = kWriteThreads / 32 / p.block_warps;
  const int64_t ctas = (units + per_cta - 1) / per_cta;
  const int64_t most = (int64_t)b2p_host::sm_count() * (dtype == B2P_F32 ? kWriteCtas<float> : kWriteCtas<__half>);
  const unsigned grid = (unsigned)(ctas < most ? ctas : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int kind = head_dim == 128 ? 2 : head_dim == 64 ? 1 : 0;
  void (*const fns[3][3])(WriteFp8Params) = {
      {kv_write_fp8_rows<__nv_bfloat16, 0>, kv_write_fp8_rows<__nv_bfloat16, 64>, kv_write_fp8_rows<__nv_bfloat16, 128>},
      {kv_write_fp8_rows<__half, 0>, kv_write_fp8_rows<__half, 64>, kv_write_fp8_rows<__half, 128>},
      {kv_write_fp8_rows<float, 0>, kv_write_fp8_rows<float, 64>, kv_write_fp8_rows<float, 128>}};
  fns[dtype][kind]<<<grid, kWriteThreads, 0, s>>>(p);
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
