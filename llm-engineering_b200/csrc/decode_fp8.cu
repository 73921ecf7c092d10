// Attention of a few query rows per sequence over the 8-bit paged cache (bf16 / f16 queries):
// the decode step (one row), the rows of drafted tokens, short prompt slices.
//
//   out[r, h, :] = softmax_t(q[r, h, :] . kc[t] * ks[blk t] * scale, t <= pos(r)) @ (vc[t] * vs[blk t])
// with e4m3 codes kc, vc and one scale per (block of tokens, KV head). HBM-bound: 2 * head_dim
// bytes of codes per token and KV head, half of what the 16-bit cache reads, for the same
// arithmetic, so the instructions per byte are what the design saves on.
//
//  * A sequence's columns are its (row, query head of the GQA group) pairs, q_len * G of them;
//    up to 8 * NT go through one pass over its keys ("virtual sequence"), more in further ones,
//    which mostly find the codes in L2. NT is 2 at most: with 4 (one pass of 32 columns) O alone
//    takes 128 registers and the loop spills; 128 sequences of 1 to 6 rows took 119 us against 71.
//  * Work = per KV head the flattened list of 32-token tiles of all virtual sequences, cut into
//    equal ranges, one per warp (stream-K at warp granularity). A warp owns a ring of S stages
//    that its lane 0 fills by TMA (two 16-token boxes of K and of V per stage) and resolves the
//    next 32 tiles' slots and scales one chunk ahead.
//  * S^T = K Q^T and O^T += V^T P^T on mma.sync m16n8k16 in f16: codes become f16 exactly, two
//    per cvt.rn.f16x2.e4m3x2 (measured at 1.3 a clock and SM against 0.8 for the same by shifts
//    and masks). The contraction order over head_dim is free, so the four bytes that an
//    8x8 ldmatrix hands a lane (four consecutive dims of one token) become the A fragment with
//    no byte permutation, and Q's fragment is one 8-byte load; V^T needs one PRMT per word
//    (two tokens x two dims), with even dims in the fragment's upper rows and odd ones below.
//    bf16 query rows are scaled by a power of two into f16's range (exact: 8-bit mantissas; only
//    values 2^-28 below a row's largest lose bits).
//  * ks goes into the scores' fp32 factor. vs goes into P before P is rounded to f16 (11 bits),
//    against a reference of its own: m_y tracks the largest score + log2(vs), as m_x does the
//    scores. References only move when a score passes them by 2^4 (one warp vote per tile
//    instead of shuffles and a rescale of O), and P vs is kept times 2^10, so that the largest
//    lies in [2^10, 2^15) of f16's [2^-14, 2^16): weights down to 2^-24 of the largest keep their
//    11 bits, smaller ones are rounded by 2^-35 of it. That matters where one key outweighs the
//    others and its value is small (an attention sink): the output is then made of small
//    weights, which l, a sum in fp32, counts in full. (With a slack of 2^8 and P as it is, weights
//    of 2^-20.5 lost 4 % and those of 2^-25 were zero.)
//  * Sequences cut by range boundaries leave partial records (O scaled into [-1, 1], then m_x, the
//    sum and the scale in fp32) in shared memory. When a CTA's warps are through, they merge
//    their records together, a 16-dim chunk per warp: sequences that lie inside the CTA's range
//    are finished there, the (at most two) others leave one record per CTA in the workspace, and
//    the last CTA to count in merges those. With every warp's records in the workspace and one
//    merging warp per sequence, 8 sequences of 4000 tokens took 48 us, most of it one warp
//    reading 74 records.
#include <mutex>
#include <type_traits>

#include "fp8.cuh"

namespace {

using namespace b2p;

constexpr int kSub = 16;   // tokens per TMA box (any block size that is a multiple of 16)
constexpr int kTile = 32;  // tokens per stage
constexpr float kNoMax = -1e30f;     // log2 weight of a record that saw nothing
constexpr float kSlack = 4.0f;       // log2 units a score may pass its reference by
constexpr float kLift = 10.0f;       // log2 of what P vs is multiplied by: 2^(kSlack + kLift + 1) fits f16
constexpr int kL2Prefetch = 4;       // tiles per warp prefetched into L2 before the launch wait

struct Fp8Params {
  const uint8_t* q;
  int64_t q_tok, q_head;  // element strides
  uint8_t* out;
  int64_t o_tok, o_head;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* ctx;
  const int32_t* cu;  // null: one row per sequence
  int64_t num_rows;
  int num_seqs, max_q_len;
  int groups_per_seq;  // column groups (virtual sequences) per sequence
  int group, group_inv;  // G and ceil(2^16 / G)
  int layer, block_size, hkv;
  int most_keys;         // what a row of the block table reaches
  int64_t num_blocks;
  const float* k_scales;  // layer bases [num_blocks, hkv]
  const float* v_scales;
  float scale_log2;
  float* joined;      // [hkv][CTAs][2][record]: the CTAs' open sequences
  int32_t* counters;  // [hkv][virtual sequences], zero between launches
  int32_t* err;
};

// A virtual sequence: columns col0 .. col0 + cols - 1 of sequence i, keys 0 .. keys - 1.
struct Virtual {
  int seq, row0, qlen, ctx, col0, cols, keys;
};

// Row of a column: col / G, exact for the columns that occur (col * G < 2^16).
__device__ __forceinline__ int row_of(const Fp8Params& p, int col) {
  return (int)((unsigned)(col * p.group_inv) >> 16);
}

template <int NC>
__device__ __forceinline__ Virtual virtual_of(const Fp8Params& p, int v) {
  Virtual t;
  t.seq = p.groups_per_seq == 1 ? v : v / p.groups_per_seq;
  t.col0 = (v - t.seq * p.groups_per_seq) * NC;
  t.ctx = min(__ldg(p.ctx + t.seq), p.most_keys);
  if (p.cu == nullptr) {  // one row per sequence
    t.row0 = t.seq;
    t.qlen = 1;
    t.cols = min(NC, p.group - t.col0);
    t.keys = max(0, t.ctx);
    return t;
  }
  t.row0 = __ldg(p.cu + t.seq);
  const int end = __ldg(p.cu + t.seq + 1);
  t.qlen = end - t.row0;
  if (t.qlen <= 0 || t.qlen > p.max_q_len || t.row0 < 0 || end > p.num_rows) t.qlen = 0;
  t.cols = min(NC, t.qlen * p.group - t.col0);
  if (t.cols <= 0) {
    t.cols = t.keys = 0;
    return t;
  }
  const int last = row_of(p, t.col0 + t.cols - 1);  // the group's last row sees the most
  t.keys = max(0, t.ctx - t.qlen + last + 1);
  return t;
}

template <int NC>
__device__ __forceinline__ int tiles_of(const Fp8Params& p, int v, int nv) {
  return v < nv ? (virtual_of<NC>(p, v).keys + kTile - 1) / kTile : 0;
}

// A partial result: O^T / (l s) in MMA fragment order, then per column the logarithm of its
// weight, m_x + log2(l) (kNoMax: it saw nothing), and the scale s = max_d |O / l|. For bf16
// output O is kept in f16 (2^-11 of the column's largest value, against an output step of 2^-8);
// for f16 output it is kept in fp32 (in f16 it would round once more as coarsely as the output).
// CTAs' records are fp32.
template <int D, int NT, bool kWide>
struct Fp8Record {
  static constexpr int kStats = (D / 16) * NT * 32 * (kWide ? 16 : 8) / 4;  // float index
  static constexpr int kFloats = kStats + NT * 8 * 2;

  __device__ static void put(float* rec, int item, int lane, float a, float b, float c, float d) {
    if constexpr (kWide)
      reinterpret_cast<float4*>(rec)[item * 32 + lane] = make_float4(a, b, c, d);
    else
      reinterpret_cast<uint2*>(rec)[item * 32 + lane] = make_uint2(pack2<__half>(a, b), pack2<__half>(c, d));
  }
  __device__ static void put_stats(float* rec, int c, float weight, float scale) {
    *reinterpret_cast<float2*>(rec + kStats + 2 * c) = make_float2(weight, scale);
  }
  template <bool kGlobal>  // another CTA's record (L2), or this CTA's in shared memory
  __device__ static float4 get(const float* rec, int item, int lane) {
    if constexpr (kWide) {
      const float4* at = reinterpret_cast<const float4*>(rec) + item * 32 + lane;
      return kGlobal ? __ldcg(at) : *at;
    } else {
      const uint2* at = reinterpret_cast<const uint2*>(rec) + item * 32 + lane;
      const uint2 v = kGlobal ? __ldcg(at) : *at;
      const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
      const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
      return make_float4(lo.x, lo.y, hi.x, hi.y);
    }
  }
  template <bool kGlobal>  // (weight, scale) of columns c and c + 1
  __device__ static float4 stats(const float* rec, int c) {
    const float4* at = reinterpret_cast<const float4*>(rec + kStats + 2 * c);
    return kGlobal ? __ldcg(at) : *at;
  }
};

__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2 weight of a column whose sum is l against m.
__device__ __forceinline__ float weight_of(float m, float l) { return l == 0.f ? kNoMax : m + log2_fast(l); }

// One fragment (item = chunk * NT + nn; a lane's four values of two columns) of records merged:
// o = sum_k 2^(w_k - top) s_k O_k, l = sum_k 2^(w_k - top). A CTA runs two warps per scheduler at
// this point, so instructions count: some twenty per record.
template <typename Rec, int NT, bool kGlobal>
struct Merge {
  float top[2] = {kNoMax, kNoMax}, l[2] = {0.f, 0.f};
  float o[4] = {0.f, 0.f, 0.f, 0.f};

  template <int kBatch, typename At>  // kBatch records' loads go out together
  __device__ void run(int count, int item, int lane, const At& at) {
    const int c = (item % NT) * 8 + 2 * (lane & 3);
    for (int k0 = 0; k0 < count; k0 += kBatch) {
      float4 v[kBatch], st[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        st[b] = make_float4(kNoMax, 0.f, kNoMax, 0.f);
        v[b] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k0 + b < count) {
          const float* rec = at(k0 + b);
          st[b] = Rec::template stats<kGlobal>(rec, c);
          v[b] = Rec::template get<kGlobal>(rec, item, lane);
        }
      }
      float t0 = top[0], t1 = top[1];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        t0 = fmaxf(t0, st[b].x);
        t1 = fmaxf(t1, st[b].z);
      }
      if (k0 > 0) {
        const float a0 = fast_exp2(top[0] - t0), a1 = fast_exp2(top[1] - t1);
        l[0] *= a0;
        l[1] *= a1;
        o[0] *= a0;
        o[1] *= a1;
        o[2] *= a0;
        o[3] *= a1;
      }
      top[0] = t0;
      top[1] = t1;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (k0 + b < count) {
          float w0 = fast_exp2(st[b].x - t0), w1 = fast_exp2(st[b].z - t1);
          if (st[b].x == kNoMax) w0 = 0.f;  // also where every record of the column saw nothing
          if (st[b].z == kNoMax) w1 = 0.f;
          l[0] += w0;
          l[1] += w1;
          w0 *= st[b].y;
          w1 *= st[b].w;
          o[0] = fmaf(v[b].x, w0, o[0]);
          o[1] = fmaf(v[b].y, w1, o[1]);
          o[2] = fmaf(v[b].z, w0, o[2]);
          o[3] = fmaf(v[b].w, w1, o[3]);
        }
      }
    }
  }
};

// The tiles of all virtual sequences in equal ranges: the first `extra` units take base + 1 of
// them, the others base. (The host bounds the tile count to 31 bits.)
struct Fp8Range {
  int begin, end;            // tiles of this unit
  int total, parts;          // tiles, units that have any
  int base, extra;
  int seq0, cb0;             // virtual sequence of `begin` and its first tile
  bool odd;                  // some virtual sequence has no tile (nothing to see, or refused)

  __device__ __forceinline__ int start(int c) const { return c * base + min(c, extra); }
  __device__ __forceinline__ int unit_of(int b) const {
    const int cut = extra * (base + 1);
    return b < cut ? b / (base + 1) : extra + (b - cut) / base;
  }
};

// One warp: all tiles counted, then the virtual sequence that holds unit c's first one. A lane
// owns kPer consecutive ones of a 32 * kPer chunk and loads them before any arithmetic.
template <int NC>
__device__ void find_unit(const Fp8Params& p, int nv, int units, int c, Fp8Range& r) {
  constexpr int kPer = 8, kChunk = 32 * kPer;
  const int lane = threadIdx.x & 31;
  int nt[kPer];
  int total = 0;
  bool odd = false;
  for (int base = 0; base < nv; base += kChunk) {
    int sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) nt[j] = tiles_of<NC>(p, base + lane * kPer + j, nv);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      sum += nt[j];
      odd |= nt[j] == 0 && base + lane * kPer + j < nv;
    }
    total += (int)__reduce_add_sync(0xffffffffu, (unsigned)sum);
  }
  r.odd = __any_sync(0xffffffffu, odd);
  r.total = total;
  r.parts = min(units, total);  // every range holds a tile
  r.seq0 = nv;
  r.cb0 = total;
  r.begin = r.end = r.base = r.extra = 0;
  if (total == 0) return;
  r.base = total / r.parts;
  r.extra = total - r.base * r.parts;
  if (c >= r.parts) return;
  r.begin = r.start(c);
  r.end = r.start(c + 1);
  int run = 0;
  for (int base = 0; base < nv; base += kChunk) {
    if (nv > kChunk) {  // the registers hold the last chunk only
#pragma unroll
      for (int j = 0; j < kPer; ++j) nt[j] = tiles_of<NC>(p, base + lane * kPer + j, nv);
    }
    int sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += nt[j];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run + incl > r.begin);
    if (hit) {
      const int src = __ffs(hit) - 1;
      int k = 0, cb = run + incl - sum;
      bool found = false;
#pragma unroll
      for (int j = 0; j < kPer - 1; ++j) {
        found |= cb + nt[j] > r.begin;
        if (!found) {
          cb += nt[j];
          k = j + 1;
        }
      }
      r.seq0 = __shfl_sync(0xffffffffu, base + lane * kPer + k, src);
      r.cb0 = __shfl_sync(0xffffffffu, cb, src);
      return;
    }
    run += __shfl_sync(0xffffffffu, incl, 31);
  }
}

// Pool coordinates of 32 consecutive tiles of a unit, one per lane: the slot of each 16-token
// half (num_slots: out of range, the TMA unit fills it with zeros) and its block.
struct Slots {
  int32_t slot[2];
  int32_t block[2];  // -1: none
};

template <int NC>
struct TileResolver {
  int win;     // first virtual sequence that can hold the next chunk
  int win_cb;  // its first tile
  int begin, n;

  __device__ Slots operator()(const Fp8Params& p, int nv, int chunk0, int lane, int32_t num_slots) {
    const unsigned all = 0xffffffffu;
    const int g = begin + chunk0 + lane;
    const bool valid = chunk0 + lane < n;
    int my = -1, my_cb = 0;
    while (true) {  // windows of 32 virtual sequences
      const int nt = tiles_of<NC>(p, win + lane, nv);
      int incl = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(all, incl, o);
        if (lane >= o) incl += y;
      }
      const int end = win_cb + incl;
      int lo = 0, hi = 32;  // smallest j whose end passes g
#pragma unroll
      for (int step = 0; step < 6; ++step) {
        const int mid = (lo + hi) >> 1;
        const int e = __shfl_sync(all, end, mid < 32 ? mid : 31);
        if (lo < hi) {
          if (e > g) hi = mid; else lo = mid + 1;
        }
      }
      const int first = __shfl_sync(all, end - nt, lo < 32 ? lo : 31);
      if (valid && my < 0 && lo < 32) {
        my = win + lo;
        my_cb = first;
      }
      if (!__any_sync(all, valid && my < 0)) break;
      win_cb = __shfl_sync(all, end, 31);
      win += 32;
      if (win >= nv) break;
    }
    const unsigned have = __ballot_sync(all, valid && my >= 0);
    if (have) {  // the next chunk starts where this one ends
      const int last = 31 - __clz(have);
      win = __shfl_sync(all, my, last);
      win_cb = __shfl_sync(all, my_cb, last);
    }
    Slots s{{num_slots, num_slots}, {-1, -1}};
    if (!valid) return s;
    if (my < 0) {
      set_device_error(p.err, B2P_DEV_LENGTH);
      return s;
    }
    const Virtual v = virtual_of<NC>(p, my);
    const int tok = (g - my_cb) * kTile;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = tok + h * kSub;
      if (t >= v.keys) continue;
      const int col = t / p.block_size;  // < the table's width: keys end at most_keys
      const int32_t blk = __ldg(p.block_tables + (int64_t)v.seq * p.bt_stride + col);
      if (blk < 0 || blk >= p.num_blocks) {
        set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
      } else {
        s.block[h] = blk;
        s.slot[h] = blk * p.block_size + t - col * p.block_size;
      }
    }
    return s;
  }
};

// Byte offset of 16-byte chunk `chunk` of token row `tok` in a box of D-byte rows, as the TMA
// unit swizzles it (128-byte rows: chunk ^ row mod 8; 64-byte rows: chunk ^ row / 2 mod 4): the
// eight rows of an ldmatrix phase then lie in eight different 16-byte bank groups. For a fixed
// row and an even c, the offset of chunk c + dc is that of chunk dc with bits 5.. flipped by c.
template <int D>
__device__ __forceinline__ uint32_t box_off(int tok, int chunk) {
  return D == 128 ? (uint32_t)(tok * 128 + ((chunk ^ (tok & 7)) << 4))
                  : (uint32_t)(tok * 64 + ((chunk ^ ((tok >> 1) & 3)) << 4));
}

__device__ __forceinline__ uint32_t cvt_lo(uint32_t w) { return fp8x2_to_f16x2((uint16_t)w); }
__device__ __forceinline__ uint32_t cvt_hi(uint32_t w) { return fp8x2_to_f16x2((uint16_t)(w >> 16)); }

// ldmatrix and mma without `volatile`, so that the compiler may overlap one step's loads with
// another's products. What keeps them in place: their address comes from hold() after the stage's
// wait, and the products are held before the stage is refilled.
__device__ __forceinline__ void load_frag(uint32_t addr, uint32_t (&r)[4]) {
  asm("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void load_frag_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t hold(uint32_t x) {
  asm volatile("" : "+r"(x) : : "memory");
  return x;
}
__device__ __forceinline__ void hold4(float (&c)[4]) {
  asm volatile("" : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : : "memory");
}

__device__ __forceinline__ float scale_exp(float s) {  // floor(log2 s), bounded
  return (float)min(127, max(kFp8MinExp, (int)((__float_as_uint(s) >> 23) & 255) - 127));
}

template <typename T, int D, int NT, int S, int W>
__global__ void __launch_bounds__(W * 32, 1) paged_rows_fp8(const __grid_constant__ CUtensorMap kmap,
                                                            const __grid_constant__ CUtensorMap vmap,
                                                            const Fp8Params p) {
  constexpr int NC = NT * 8;
  constexpr int kChunks = D / 16;           // 16-byte chunks of a token row = k-steps of Q K^T
  constexpr int kBox = kSub * D;            // bytes of one box
  constexpr int kStage = 4 * kBox;          // K lo, K hi, V lo, V hi
  using Rec = Fp8Record<D, NT, std::is_same<T, __half>::value>;  // a warp's
  using Joined = Fp8Record<D, NT, true>;                        // a CTA's
  struct Cut {  // a segment that a warp left as a record, in shared memory
    int v, nt;
    int in_ring;  // the stream's last segment: in the warp's ring, done with by then
    int head;     // the first of its sequence's cuts in this CTA
    int cb;       // first tile of v
    int row0, col0, cols;
  };
  __shared__ Cut cuts[W][2];
  __shared__ int num_cuts[W];
  __shared__ int last_of[2];  // per open group: this CTA was the last to count in
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // Programmatic dependent launch: before the wait only lengths, offsets and block tables are
  // read. Of the kernels that let this one start early (itself, the 16-bit decode kernel, the
  // cache write) none writes those, and the kernels that do write them (table builds, compaction,
  // host copies) have completed before any of these started.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.y;
  uint8_t* ring = smem + (size_t)warp * S * kStage;
  uint8_t* firsts = smem + (size_t)W * S * kStage;  // [W][record]: cuts in mid-stream
  uint64_t* full = reinterpret_cast<uint64_t*>(firsts + (size_t)W * Rec::kFloats * 4) + warp * S;
  static_assert(Rec::kFloats * 4 <= S * kStage && Rec::kFloats % 4 == 0, "a ring holds a record");
  auto record_of = [&](int w, bool in_ring) {
    return reinterpret_cast<float*>(in_ring ? smem + (size_t)w * S * kStage : firsts + (size_t)w * Rec::kFloats * 4);
  };
  const int nv = p.num_seqs * p.groups_per_seq;
  const int32_t num_slots = (int32_t)(p.num_blocks * p.block_size);
  const int g8 = lane >> 2, t4 = lane & 3;

  // Rows without a key to see, and lengths that do not fit: zeros and the flag, by one warp per
  // KV head (no unit's range holds a virtual sequence without tiles).
  auto write_empties = [&]() {
    for (int base = 0; base < nv; base += 32) {
      const int v = base + lane;
      bool empty = false, bad = false;
      if (v < nv) {
        const Virtual t = virtual_of<NC>(p, v);
        empty = t.cols > 0 && t.keys <= 0;
        bad = empty;
        if (p.cu != nullptr && t.qlen == 0) {  // refused offsets, or simply no rows
          const int n = __ldg(p.cu + t.seq + 1) - t.row0;
          bad |= n > p.max_q_len || n < 0 || t.row0 < 0 || (int64_t)t.row0 + n > p.num_rows;
        }
      }
      if (bad) set_device_error(p.err, B2P_DEV_LENGTH);
      unsigned m = __ballot_sync(0xffffffffu, empty);
      while (m) {
        const Virtual t = virtual_of<NC>(p, base + __ffs(m) - 1);
        m &= m - 1;
        for (int e = lane; e < t.cols * D; e += 32) {
          const int c = t.col0 + e / D;
          reinterpret_cast<T*>(p.out)[(int64_t)(t.row0 + c / p.group) * p.o_tok +
                                      (int64_t)(head * p.group + c % p.group) * p.o_head + e % D] =
              from_f32<T>(0.f);
        }
      }
    }
  };
  const bool empties_warp = blockIdx.x == 0 && warp == W - 1;

  Fp8Range r;
  const int unit = blockIdx.x * W + warp;
  find_unit<NC>(p, nv, gridDim.x * W, unit, r);
  if ((int)blockIdx.x * W >= r.parts) {  // no tile for this CTA
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (empties_warp) write_empties();
    return;
  }
  const int n = r.end - r.begin;  // 0 for a warp without tiles
  if (lane == 0) {
    for (int s = 0; s < S; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  __syncwarp();

  TileResolver<NC> res{r.seq0, r.cb0, r.begin, n};
  Slots cur = res(p, nv, 0, lane, num_slots), nxt{{num_slots, num_slots}, {-1, -1}};
  if (lane < kL2Prefetch && lane < n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (cur.slot[h] < num_slots) {
        tma_prefetch_l2_5d(&kmap, 0, 0, head, cur.slot[h], p.layer);
        tma_prefetch_l2_5d(&vmap, 0, 0, head, cur.slot[h], p.layer);
      }
    }
  }
  // From here on what the previous kernel wrote is read from L2 (TMA, ld.cg): this grid may have
  // started before those writes, so nothing may come from an L1 line or the read-only path.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // Scales of this lane's tile, by half: loaded with the slots, a chunk ahead of their use. A NaN
  // value scale moves to the key scale: the scores then carry it to the rows that see the block,
  // and to no others.
  struct Scales {
    float k[2], v[2], e[2];  // e: floor(log2 v), bounded
  };
  auto load_scales = [&](const Slots& s, Scales& c) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool have = s.block[h] >= 0;
      const int64_t at = (int64_t)(have ? s.block[h] : 0) * p.hkv + head;
      c.k[h] = have ? __ldcg(p.k_scales + at) : 0.f;
      c.v[h] = have ? __ldcg(p.v_scales + at) : 0.f;
    }
  };
  auto settle_scales = [](Scales& c) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (c.v[h] != c.v[h]) {
        c.k[h] = c.v[h];
        c.v[h] = 0.f;
      }
      c.e[h] = scale_exp(c.v[h]);
    }
  };
  Scales sc_cur, sc_nxt{};
  load_scales(cur, sc_cur);
  int issue_base = 0;  // tiles [issue_base, issue_base + 32) are in the issue slots
  Slots isl = cur;     // slots that the issue side reads (may run a chunk ahead of the scales)
  int issued = 0, use_base = 0, issue_stage = 0;
  bool aborted = false;

  auto issue = [&]() {  // tile `issued` into the next stage
    if (issued >= issue_base + 32) {
      issue_base += 32;
      isl = nxt;
    }
    const int32_t s0 = __shfl_sync(0xffffffffu, isl.slot[0], issued - issue_base);
    const int32_t s1 = __shfl_sync(0xffffffffu, isl.slot[1], issued - issue_base);
    if (lane == 0) {
      uint8_t* dst = ring + issue_stage * kStage;
      uint64_t* bar = full + issue_stage;
      mbar_arrive_expect_tx(bar, kStage);
      tma_load_5d(dst, &kmap, bar, 0, 0, head, s0, p.layer);
      tma_load_5d(dst + kBox, &kmap, bar, 0, 0, head, s1, p.layer);
      tma_load_5d(dst + 2 * kBox, &vmap, bar, 0, 0, head, s0, p.layer);
      tma_load_5d(dst + 3 * kBox, &vmap, bar, 0, 0, head, s1, p.layer);
    }
    ++issued;
    issue_stage = issue_stage + 1 == S ? 0 : issue_stage + 1;
  };
#pragma unroll
  for (int k = 0; k < S; ++k)
    if (k < n) issue();
  if (empties_warp && r.odd) write_empties();  // while the first tiles are in flight

  int ncut = 0;  // records left (at most the unit's first and last segment)

  // Rows of one virtual sequence from O^T fragments: out = (O * f) * g. (Two factors: their product
  // may lie below the normal range where the output does not.)
  auto write_out = [&](const Virtual& t, float (&o)[kChunks][NT][4], float (&f)[NT][2], float (&g)[NT][2]) {
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const int c = nn * 8 + 2 * t4 + cc;
        if (c >= t.cols) continue;
        const int col = t.col0 + c;
        T* orow = reinterpret_cast<T*>(p.out) + (int64_t)(t.row0 + row_of(p, col)) * p.o_tok +
                  (int64_t)(head * p.group + col - row_of(p, col) * p.group) * p.o_head;
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
          *reinterpret_cast<uint32_t*>(orow + i * 16 + 2 * g8) =
              pack_values<T>(o[i][nn][cc] * f[nn][cc] * g[nn][cc], o[i][nn][2 + cc] * f[nn][cc] * g[nn][cc]);
      }
    }
  };

  int v = r.seq0;
  int cb = r.cb0, gidx = r.begin, k = 0, use_stage = 0;
  uint32_t phase = 0;
  while (gidx < r.end) {
    const Virtual t = virtual_of<NC>(p, v);
    const int ntl = (t.keys + kTile - 1) / kTile;
    if (ntl == 0) {  // written by the empties warp
      ++v;
      continue;
    }
    const int lb0 = gidx - cb;
    const int seg_end = min(r.end, cb + ntl);
    const int lb1 = seg_end - cb;
    if (lane == 0) {
      if (p.cu != nullptr && t.ctx < t.qlen) set_device_error(p.err, B2P_DEV_LENGTH);
      if (__ldg(p.ctx + t.seq) > p.most_keys) set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
    }

    // ---- Q fragments: column nn * 8 + g8, dims 16c + 4 t4 .. + 3 (8 bytes per lane and k-step)
    uint2 qf[kChunks][NT];
    float qfac[NT][2];  // scale_log2 / (power of two the query row was multiplied by)
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
      const int c = nn * 8 + g8;
      const bool ok = c < t.cols;
      const int col = t.col0 + (ok ? c : 0);
      const T* qrow = reinterpret_cast<const T*>(p.q) + (int64_t)(t.row0 + row_of(p, col)) * p.q_tok +
                      (int64_t)(head * p.group + col - row_of(p, col) * p.group) * p.q_head + 4 * t4;
      uint2 w[kChunks];
#pragma unroll
      for (int kk = 0; kk < kChunks; ++kk)
        w[kk] = ok ? __ldcg(reinterpret_cast<const uint2*>(qrow + kk * 16)) : make_uint2(0u, 0u);
      float inv = 1.f;
      if constexpr (!std::is_same<T, __half>::value) {
        float amax = 0.f;
#pragma unroll
        for (int kk = 0; kk < kChunks; ++kk) {
          amax = fmaxf(amax, fmaxf(fmaxf(fabsf(__uint_as_float(w[kk].x << 16)), fabsf(__uint_as_float(w[kk].x & 0xffff0000u))),
                                   fmaxf(fabsf(__uint_as_float(w[kk].y << 16)), fabsf(__uint_as_float(w[kk].y & 0xffff0000u)))));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // the row's largest value goes to [2^14, 2^15); rows of zeros, infinities and NaN stay
        const int ex = (int)(__float_as_uint(amax) >> 23) - 127;
        const int up = amax > 0.f && ex < 128 ? min(14 - ex, 120) : 0;
        const float mul = exp2_int(up);
        inv = exp2_int(-up);
#pragma unroll
        for (int kk = 0; kk < kChunks; ++kk) {
          w[kk].x = pack2<__half>(__uint_as_float(w[kk].x << 16) * mul, __uint_as_float(w[kk].x & 0xffff0000u) * mul);
          w[kk].y = pack2<__half>(__uint_as_float(w[kk].y << 16) * mul, __uint_as_float(w[kk].y & 0xffff0000u) * mul);
        }
      }
      // the factor of column 2 t4 + cc sits in the lanes whose g8 is that column
      qfac[nn][0] = __shfl_sync(0xffffffffu, inv, 8 * t4) * p.scale_log2;
      qfac[nn][1] = __shfl_sync(0xffffffffu, inv, 8 * t4 + 4) * p.scale_log2;
#pragma unroll
      for (int kk = 0; kk < kChunks; ++kk) qf[kk][nn] = w[kk];
    }
    // keys that each of this lane's columns sees (columns past the last: none)
    int lim[NT][2];
    int lim_min = t.keys;
#pragma unroll
    for (int nn = 0; nn < NT; ++nn)
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const int c = nn * 8 + 2 * t4 + cc;
        lim[nn][cc] = p.cu == nullptr ? t.keys : c < t.cols ? t.ctx - t.qlen + row_of(p, t.col0 + c) + 1 : t.keys;
      }
    if (p.cu != nullptr) lim_min = t.ctx - t.qlen + row_of(p, t.col0) + 1;

    float mx[NT][2], slack[NT][2], gy[NT][2], l[NT][2];
    float acc[kChunks][NT][4];
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
      mx[nn][0] = mx[nn][1] = 0.f;  // set by the segment's first tile
      slack[nn][0] = slack[nn][1] = kSlack;
      gy[nn][0] = gy[nn][1] = 1.f;
      l[nn][0] = l[nn][1] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int nn = 0; nn < NT; ++nn) acc[i][nn][0] = acc[i][nn][1] = acc[i][nn][2] = acc[i][nn][3] = 0.f;

    for (int lb = lb0; lb < lb1; ++lb, ++k) {
      if (k == use_base + 32) {  // rotate the scale buffers; the issue side has moved on already
        use_base += 32;
        sc_cur = sc_nxt;
      }
      if (k == use_base + 8 && use_base + 32 < n) {  // the next chunk, well before it is issued
        nxt = res(p, nv, use_base + 32, lane, num_slots);
        load_scales(nxt, sc_nxt);
      }
      if (k == use_base) settle_scales(sc_cur);
      const int src = k - use_base;
      float ks[2], vs[2], ev[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[h] = __shfl_sync(0xffffffffu, sc_cur.k[h], src);
        vs[h] = __shfl_sync(0xffffffffu, sc_cur.v[h], src);
        ev[h] = __shfl_sync(0xffffffffu, sc_cur.e[h], src);
      }
      if (!aborted && !mbar_wait_bounded(full + use_stage, phase, p.err)) aborted = true;
      aborted = __any_sync(0xffffffffu, aborted);
      if (aborted) continue;  // keep walking so every sequence still gets written
      uint8_t* stage = ring + use_stage * kStage;
      if (++use_stage == S) {
        use_stage = 0;
        phase ^= 1u;
      }
      const int tok0 = lb * kTile;
      const int valid = min(kTile, t.ctx - tok0);  // tokens that exist
      if (valid < kTile) {
        // Slots past the context may hold any code, NaN too, and 0 * NaN would poison O: zero
        // their V rows (a row is D contiguous bytes; the swizzle stays inside it or its pair,
        // so whole rows are zeroed through their swizzled chunks).
        for (int i = lane; i < (kTile - valid) * kChunks; i += 32) {
          const int tok = valid + i / kChunks;
          *reinterpret_cast<uint4*>(stage + (2 + tok / kSub) * kBox + box_off<D>(tok % kSub, i % kChunks)) =
              make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      const uint32_t base = hold(smem_u32(stage));

      // ---- S^T = K Q^T: 2 x 16 tokens, NC columns
      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nn = 0; nn < NT; ++nn) s[h][nn][0] = s[h][nn][1] = s[h][nn][2] = s[h][nn][3] = 0.f;
      {
        const uint32_t mine = base + box_off<D>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a[4];
            load_frag((mine + h * kBox) ^ (uint32_t)(c << 4), a);
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              mma_f16(s[h][nn], cvt_lo(a[0]), cvt_lo(a[1]), cvt_hi(a[0]), cvt_hi(a[1]), qf[c][nn].x, qf[c][nn].y);
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              mma_f16(s[h][nn], cvt_lo(a[2]), cvt_lo(a[3]), cvt_hi(a[2]), cvt_hi(a[3]), qf[c + 1][nn].x, qf[c + 1][nn].y);
          }
        }
      }

      // ---- scores in log2 units less m_x, masked where a column's rows end. A score may pass
      // its references by kSlack: thr is what is left of that for m_x and, with the half's
      // exponent, for m_y (slack = m_y - m_x + kSlack).
      const bool masked = tok0 + kTile > lim_min;
      const bool first = lb == lb0;
      bool over = first;
#pragma unroll
      for (int nn = 0; nn < NT; ++nn)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = ks[h] * qfac[nn][cc];
            float x0 = fmaf(s[h][nn][cc], f, -mx[nn][cc]), x1 = fmaf(s[h][nn][2 + cc], f, -mx[nn][cc]);
            if (masked) {
              const int left = lim[nn][cc] - tok0 - h * kSub;
              if (g8 >= left) x0 = -INFINITY;
              if (g8 + 8 >= left) x1 = -INFINITY;
            }
            s[h][nn][cc] = x0;
            s[h][nn][2 + cc] = x1;
            over |= fmaxf(x0, x1) > fminf(kSlack, slack[nn][cc] - ev[h]);
          }
      if (__any_sync(0xffffffffu, over)) {  // move the references (always on a segment's first tile)
#pragma unroll
        for (int nn = 0; nn < NT; ++nn)
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            float t0 = fmaxf(s[0][nn][cc], s[0][nn][2 + cc]), t1 = fmaxf(s[1][nn][cc], s[1][nn][2 + cc]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
              t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
              t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
            }
            // By how much m_x and m_y move (t0, t1 are relative to m_x): to the first tile's
            // largest, later only up. A column that sees nothing of the first tile sees nothing of
            // the later ones either (its keys end before them).
            const float gap = slack[nn][cc] - kSlack;  // m_y - m_x
            float dx = fmaxf(t0, t1), dy = fmaxf(t0 + ev[0], t1 + ev[1]) - gap;
            if (first) {
              dx = dx == -INFINITY ? 0.f : dx;
              dy = dy == -INFINITY ? 0.f : dy;
            } else {
              dx = fmaxf(dx, 0.f);
              dy = fmaxf(dy, 0.f);
              l[nn][cc] *= fast_exp2(-dx);
              const float al = fast_exp2(-dy);
#pragma unroll
              for (int i = 0; i < kChunks; ++i) {
                acc[i][nn][cc] *= al;
                acc[i][nn][2 + cc] *= al;
              }
            }
            mx[nn][cc] += dx;
            slack[nn][cc] += dy - dx;
            gy[nn][cc] = fast_exp2(kSlack + kLift - slack[nn][cc]);  // 2^(m_x - m_y + kLift)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s[h][nn][cc] -= dx;
              s[h][nn][2 + cc] -= dx;
            }
          }
      }
      // ---- P = 2^(x - m_x); its f16 copy carries vs and 2^kLift against m_y
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nn = 0; nn < NT; ++nn) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float pv[4];
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const float p0 = fast_exp2(s[h][nn][cc]), p1 = fast_exp2(s[h][nn][2 + cc]);
            l[nn][cc] += p0 + p1;
            // bounded: a block whose weights have all underflowed may have any factor
            const float f = fminf(vs[h] * gy[nn][cc], 0x1p126f);
            pv[cc] = p0 * f;
            pv[2 + cc] = p1 * f;
          }
          pb[h][nn][0] = movmatrix_trans(pack2<__half>(pv[0], pv[1]));
          pb[h][nn][1] = movmatrix_trans(pack2<__half>(pv[2], pv[3]));
        }
      }

      // ---- O^T += V^T P^T: 16 dims per fragment (even ones in rows 0..7, odd ones in 8..15)
      {
        const uint32_t mine = base + 2 * kBox + box_off<D>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a[4];
            load_frag_trans((mine + h * kBox) ^ (uint32_t)(c << 4), a);
#pragma unroll
            for (int k2 = 0; k2 < 4; ++k2) a[k2] = __byte_perm(a[k2], 0, 0x3120);
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              mma_f16(acc[c][nn], cvt_lo(a[0]), cvt_hi(a[0]), cvt_lo(a[1]), cvt_hi(a[1]), pb[h][nn][0], pb[h][nn][1]);
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              mma_f16(acc[c + 1][nn], cvt_lo(a[2]), cvt_hi(a[2]), cvt_lo(a[3]), cvt_hi(a[3]), pb[h][nn][0], pb[h][nn][1]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int nn = 0; nn < NT; ++nn) hold4(acc[i][nn]);
      // Refill the stage: its reads fed the MMAs above; generic writes need a proxy fence before
      // the TMA unit writes the same bytes.
      if (valid < kTile) fence_proxy_async_smem();
      __syncwarp();
      if (issued < n) issue();
    }

    // ---- finish the segment
#pragma unroll
    for (int nn = 0; nn < NT; ++nn)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[nn][0] += __shfl_xor_sync(0xffffffffu, l[nn][0], o);
        l[nn][1] += __shfl_xor_sync(0xffffffffu, l[nn][1], o);
      }
    if (lb0 == 0 && lb1 == ntl) {
      float f[NT][2], g[NT][2];
#pragma unroll
      for (int nn = 0; nn < NT; ++nn)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          f[nn][cc] = l[nn][cc] > 0.f ? 1.f / l[nn][cc] : 0.f;
          g[nn][cc] = fast_exp2(slack[nn][cc] - (kSlack + kLift));  // 2^(m_y - m_x - kLift)
        }
      write_out(t, acc, f, g);
    } else {
      const bool in_ring = seg_end == r.end;
      float* rec = record_of(warp, in_ring);
#pragma unroll
      for (int nn = 0; nn < NT; ++nn) {
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
          for (int cc = 0; cc < 2; ++cc)
            top[cc] = fmaxf(top[cc], fmaxf(fabsf(acc[i][nn][cc]), fabsf(acc[i][nn][2 + cc])));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
          top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
        }
        const float f0 = top[0] > 0.f ? 1.f / top[0] : 0.f, f1 = top[1] > 0.f ? 1.f / top[1] : 0.f;
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
          Rec::put(rec, i * NT + nn, lane, acc[i][nn][0] * f0, acc[i][nn][1] * f1, acc[i][nn][2] * f0, acc[i][nn][3] * f1);
        if (g8 == 0) {
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            Rec::put_stats(rec, nn * 8 + 2 * t4 + cc, weight_of(mx[nn][cc], l[nn][cc]),
                           l[nn][cc] > 0.f ? top[cc] / l[nn][cc] * fast_exp2(slack[nn][cc] - (kSlack + kLift)) : 0.f);
          }
        }
      }
      if (lane == 0 && ncut < 2) cuts[warp][ncut] = Cut{v, ntl, in_ring, lb0 == 0 || warp == 0, cb, t.row0, t.col0, t.cols};
      ++ncut;
    }
    gidx = seg_end;
    if (lb1 == ntl) {
      cb += ntl;
      ++v;
    }
  }
  // Never leave with TMA writes in flight (only after an abort: every issued tile is waited for).
  if (aborted && lane == 0)
    for (int st = 0; st < S; ++st) {  // a stage's last load has completed when its phase flips
      const int loads = (issued + S - 1 - st) / S;
      if (loads > 0) mbar_wait_bounded(full + st, (uint32_t)((loads - 1) & 1), nullptr);
    }

  // ---- merge what this CTA's warps left. The cuts, in tile order, fall into groups of one
  // virtual sequence each: a head cut and the first cut of each further warp up to the sequence's
  // end. Lane e looks at cut e % 2 of warp e / 2; a piece of work is one fragment (item) of a group.
  if (lane == 0) num_cuts[warp] = ncut;
  __syncthreads();
  constexpr int kItems = kChunks * NT;
  static_assert(2 * W <= 32, "a lane per cut");
  const int cta_unit = blockIdx.x * W;
  const int cta_begin = r.start(cta_unit), cta_end = r.start(min(cta_unit + W, r.parts));
  Cut mine{};
  int u_end = 0;       // unit that holds the end of the lane's sequence
  bool open = false, closed = false;
  if (lane < 2 * W && (lane & 1) < num_cuts[lane >> 1]) {
    mine = cuts[lane >> 1][lane & 1];
    u_end = r.unit_of(mine.cb + mine.nt - 1);
    const bool inside = mine.cb >= cta_begin && mine.cb + mine.nt <= cta_end;
    open = mine.head && !inside;  // other CTAs hold a part of the sequence
    closed = mine.head && inside;
  }
  const unsigned opens = __ballot_sync(0xffffffffu, open), closeds = __ballot_sync(0xffffffffu, closed);
  // rows of the output from one merged fragment
  auto write_item = [&](int row0, int col0, int cols, int item, const float (&o)[4], const float (&l)[2]) {
    const int i = item / NT, nn = item % NT;
#pragma unroll
    for (int cc = 0; cc < 2; ++cc) {
      const int c = nn * 8 + 2 * t4 + cc;
      if (c >= cols) continue;
      const int row = row_of(p, col0 + c);
      const float f = l[cc] > 0.f ? 1.f / l[cc] : 0.f;
      T* orow = reinterpret_cast<T*>(p.out) + (int64_t)(row0 + row) * p.o_tok +
                (int64_t)(head * p.group + col0 + c - row * p.group) * p.o_head;
      *reinterpret_cast<uint32_t*>(orow + i * 16 + 2 * g8) = pack_values<T>(o[cc] * f, o[2 + cc] * f);
    }
  };
  // The warp's share of the pieces of the groups in `heads`.
  auto merge_groups = [&](unsigned heads, bool inside) {
    const int pieces = __popc(heads) * kItems;
    const int per = (pieces + W - 1) / W;
    const int end = min(pieces, (warp + 1) * per);
    for (int piece = warp * per; piece < end; ++piece) {
      unsigned m = heads;
      for (int skip = piece / kItems; skip > 0; --skip) m &= m - 1;
      const int item = piece % kItems, e = __ffs(m) - 1, w0 = e >> 1;
      const int w1 = min(W - 1, __shfl_sync(0xffffffffu, u_end, e) - cta_unit);
      // a warp between the first and the last of a group has one segment, its stream's last
      const int ring0 = __shfl_sync(0xffffffffu, mine.in_ring, e);
      const int ring1 = __shfl_sync(0xffffffffu, mine.in_ring, 2 * w1);
      const int cb = __shfl_sync(0xffffffffu, mine.cb, e);
      const int row0 = __shfl_sync(0xffffffffu, mine.row0, e);
      const int col0 = __shfl_sync(0xffffffffu, mine.col0, e), cols = __shfl_sync(0xffffffffu, mine.cols, e);
      Merge<Rec, NT, false> mg;
      mg.template run<4>(w1 - w0 + 1, item, lane, [&](int k) -> const float* {
        return record_of(w0 + k, k == 0 ? ring0 : k == w1 - w0 ? ring1 : 1);
      });
      if (inside) {
        write_item(row0, col0, cols, item, mg.o, mg.l);
        continue;
      }
      float* joined = p.joined + (((size_t)head * gridDim.x + blockIdx.x) * 2 + (cb <= cta_begin ? 0 : 1)) * Joined::kFloats;
      const float i0 = mg.l[0] > 0.f ? 1.f / mg.l[0] : 0.f, i1 = mg.l[1] > 0.f ? 1.f / mg.l[1] : 0.f;
      Joined::put(joined, item, lane, mg.o[0] * i0, mg.o[1] * i1, mg.o[2] * i0, mg.o[3] * i1);
      if (item < NT && g8 == 0) {
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          Joined::put_stats(joined, item * 8 + 2 * t4 + cc, weight_of(mg.top[cc], mg.l[cc]), 1.f);
        }
      }
    }
  };
  // The open groups (at most two) first: their counts travel while the closed ones are written.
  if (opens != 0) {
    merge_groups(opens, false);
    __syncthreads();  // the CTA's joined records are written
    if (warp == 0 && open) {
      int seen;
      int32_t* counter = p.counters + (size_t)head * nv + mine.v;
      asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(seen) : "l"(counter) : "memory");
      const bool last = seen == u_end / W - r.unit_of(mine.cb) / W;
      if (last) *counter = 0;  // for the next launch
      last_of[mine.cb <= cta_begin ? 0 : 1] = last;
    }
  }
  if (closeds != 0) merge_groups(closeds, true);
  if (opens == 0) return;
  __syncthreads();
  for (unsigned m = opens; m != 0; m &= m - 1) {
    const int e = __ffs(m) - 1;
    const int cb = __shfl_sync(0xffffffffu, mine.cb, e);
    if (!last_of[cb <= cta_begin ? 0 : 1]) continue;
    const int c0 = r.unit_of(cb) / W, c1 = __shfl_sync(0xffffffffu, u_end, e) / W;
    const int row0 = __shfl_sync(0xffffffffu, mine.row0, e);
    const int col0 = __shfl_sync(0xffffffffu, mine.col0, e), cols = __shfl_sync(0xffffffffu, mine.cols, e);
    for (int item = warp; item < kItems; item += W) {
      Merge<Joined, NT, true> mg;
      mg.template run<8>(c1 - c0 + 1, item, lane, [&](int k) -> const float* {
        return p.joined + (((size_t)head * gridDim.x + c0 + k) * 2 + (cb <= r.start((c0 + k) * W) ? 0 : 1)) * Joined::kFloats;
      });
      write_item(row0, col0, cols, item, mg.o, mg.l);
    }
  }
}

// ====================================================================== host side
struct Fp8Plan {
  const void* fn = nullptr;
  int smem = 0, warps = 0, columns = 0;
};

template <typename T, int D, int NT, int S, int W>
Fp8Plan make_fp8_plan() {
  static_assert(NT <= 2 && D <= 128, "the workspace has room for these");
  Fp8Plan pl;
  pl.fn = reinterpret_cast<const void*>(&paged_rows_fp8<T, D, NT, S, W>);
  using Rec = Fp8Record<D, NT, std::is_same<T, __half>::value>;
  pl.smem = W * S * 4 * kSub * D + W * Rec::kFloats * 4 + W * S * 8 + 1024;
  static_assert(W * S * 4 * kSub * D + W * Rec::kFloats * 4 + W * S * 8 + 1024 + W * 100 + 64 <= 227 * 1024,
                "shared memory of an SM");
  pl.warps = W;
  pl.columns = NT * 8;
  return pl;
}

template <typename T>
bool select_fp8_plan(int head_dim, int columns, Fp8Plan& pl) {
  if (head_dim == 128)
    pl = columns <= 8 ? make_fp8_plan<T, 128, 1, 2, 8>() : make_fp8_plan<T, 128, 2, 2, 8>();
  else if (head_dim == 64)
    pl = columns <= 8 ? make_fp8_plan<T, 64, 1, 4, 8>() : make_fp8_plan<T, 64, 2, 4, 8>();
  else
    return false;
  return true;
}

// CTAs along x: one CTA per SM over the KV heads.
int64_t fp8_ctas(int num_kv_heads) {
  const int64_t c = b2p_host::sm_count() / num_kv_heads;
  return c < 1 ? 1 : c;
}

// Workspace: room for the records of the largest plan, then the counters, so that the counters
// sit at one place for every shape and call, in bytes that nothing else ever writes. (At a place
// that followed the call's own records, one buffer used for calls of one and of five rows in
// turn would find records where it looks for zeroed counters.)
constexpr int kMostColumns = 16;   // per virtual sequence
// Columns per sequence that calls here have at most; more belong to the tile kernel, which pays
// for 128 rows per query tile. 12/2 heads, histories of 512 to 4090 tokens, here against there:
// 128 sequences of 16 rows (96 columns) 179 us against 378, of 26 rows (156) 281 against 379; four
// sequences of 26 rows 28 against 47; short histories (20 to 300) of 26 rows 43 against 37.
constexpr int kRowColumns = 160;

size_t records_bytes(int num_kv_heads) {
  const int64_t ctas = num_kv_heads > b2p_host::sm_count() ? num_kv_heads : b2p_host::sm_count();
  return (size_t)ctas * 2 * Fp8Record<128, kMostColumns / 8, true>::kFloats * 4;
}

int column_groups(const Fp8Plan& pl, int group, int max_q_len) {
  return (int)(((int64_t)group * max_q_len + pl.columns - 1) / pl.columns);
}

}  // namespace

// Whether calls of this shape run here; rows beyond a few per sequence belong to the tile kernel.
bool b2p_rows_fp8_takes(int group, int head_dim, int block_size, int dtype, int max_q_len) {
  Fp8Plan pl;
  return (dtype == B2P_BF16 || dtype == B2P_F16) && block_size % kSub == 0 && max_q_len >= 1 &&
         (int64_t)group * max_q_len <= kRowColumns &&
         select_fp8_plan<__half>(head_dim, group * max_q_len, pl);
}

extern "C" int b2p_paged_fp8_row_columns(void) { return kRowColumns; }

size_t b2p_rows_fp8_workspace(int num_seqs, int num_kv_heads) {
  // a sequence has at most kRowColumns / 8 column groups (8 columns being the least a pass takes)
  const size_t counters = (size_t)num_kv_heads * num_seqs * (kRowColumns / 8) * 4;
  return records_bytes(num_kv_heads) + ((counters + 255) & ~size_t(255));
}

int b2p_rows_fp8(const void* q, int64_t q_tok_stride, int64_t q_head_stride, const void* key_cache,
                 const void* value_cache, const float* key_scales, const float* value_scales,
                 int64_t layer_index, int64_t num_layers, int64_t num_slots,
                 const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_q,
                 const int32_t* context_lens, int num_seqs, int64_t num_rows, int max_q_len,
                 int num_q_heads, int num_kv_heads, int head_dim, int block_size, float scale,
                 void* out, int64_t out_tok_stride, int64_t out_head_stride, void* workspace,
                 size_t workspace_size, int dtype, int32_t* err_flag, void* stream) {
  const int group = num_q_heads / num_kv_heads;
  Fp8Plan pl;
  const bool have = dtype == B2P_BF16 ? select_fp8_plan<__nv_bfloat16>(head_dim, group * max_q_len, pl)
                                      : select_fp8_plan<__half>(head_dim, group * max_q_len, pl);
  if (!have) return B2P_EUNSUPPORTED;
  if (!workspace || workspace_size < b2p_rows_fp8_workspace(num_seqs, num_kv_heads))
    return B2P_EWORKSPACE;
  static std::mutex mu;
  static const void* ready[64][32] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return b2p_host::record_error(e);
  if (dev < 0 || dev >= 64) return B2P_EUNSUPPORTED;
  {
    std::lock_guard<std::mutex> lock(mu);
    int i = 0;
    while (i < 32 && ready[dev][i] != nullptr && ready[dev][i] != pl.fn) ++i;
    if (i == 32 || ready[dev][i] == nullptr) {
      e = cudaFuncSetAttribute(pl.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, pl.smem);
      if (e != cudaSuccess) return b2p_host::record_error(e);
      if (i < 32) ready[dev][i] = pl.fn;
    }
  }
  // 31 bits count the tiles of a KV head
  const int64_t width_tiles = (block_table_stride * block_size + kTile - 1) / kTile;
  if (width_tiles * num_seqs * column_groups(pl, group, max_q_len) > 0x7fffffffLL) return B2P_EUNSUPPORTED;
  CUtensorMap kmap, vmap;
  int rc = b2p_host::fp8_pool_tensor_map(&kmap, key_cache, num_layers, num_slots, num_kv_heads, head_dim);
  if (rc != B2P_OK) return rc;
  rc = b2p_host::fp8_pool_tensor_map(&vmap, value_cache, num_layers, num_slots, num_kv_heads, head_dim);
  if (rc != B2P_OK) return rc;
  Fp8Params p;
  p.q = static_cast<const uint8_t*>(q);
  p.q_tok = q_tok_stride;
  p.q_head = q_head_stride;
  p.out = static_cast<uint8_t*>(out);
  p.o_tok = out_tok_stride;
  p.o_head = out_head_stride;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.ctx = context_lens;
  p.cu = cu_q;
  p.num_rows = num_rows;
  p.num_seqs = num_seqs;
  p.max_q_len = max_q_len;
  p.groups_per_seq = column_groups(pl, group, max_q_len);
  p.group = group;
  p.group_inv = (65536 + group - 1) / group;
  const int64_t reach = block_table_stride * block_size;
  p.most_keys = (int)(reach < 0x7fffff00LL ? reach : 0x7fffff00LL);
  p.layer = (int)layer_index;
  p.block_size = block_size;
  p.hkv = num_kv_heads;
  p.num_blocks = num_slots / block_size;
  p.k_scales = key_scales + layer_index * p.num_blocks * num_kv_heads;
  p.v_scales = value_scales + layer_index * p.num_blocks * num_kv_heads;
  p.scale_log2 = scale * kLog2e;
  p.joined = static_cast<float*>(workspace);
  p.counters = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + records_bytes(num_kv_heads));
  p.err = err_flag;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)fp8_ctas(num_kv_heads), (unsigned)num_kv_heads);
  cfg.blockDim = dim3(pl.warps * 32);
  cfg.dynamicSmemBytes = (size_t)pl.smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&kmap, &vmap, &p};
  e = cudaLaunchKernelExC(&cfg, pl.fn, args);
  if (e != cudaSuccess) return b2p_host::record_error(e);
  return b2p_host::check_launch();
}
