// Attention of a few query rows per sequence over the 8-bit paged cache (bf16 / f16 queries):
// the decode step (one row) and the rows of drafted tokens.
//
//   out[r, h, :] = softmax_t(q[r, h, :] . kc[t] * ks[blk t] * scale, t <= pos(r)) @ (vc[t] * vs[blk t])
// with e4m3 codes kc, vc and one scale per (block of tokens, KV head). HBM-bound: 2 * head_dim
// bytes of codes per token and KV head, half of what the 16-bit cache reads, for the same
// arithmetic, so the instructions per byte are what the design saves on.
//
//  * A sequence's columns are its (row, query head of the GQA group) pairs, q_len * G of them;
//    up to 8 * NT go through one pass over its keys ("virtual sequence"), more in further ones.
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
//    scores, so the weights that matter keep their 11 bits whatever the spread of the scales.
//    References only move when a score passes them by 2^8 (one warp vote per tile instead of
//    shuffles and a rescale of O).
//  * Sequences cut by range boundaries leave partial records (O scaled into [-1, 1] in f16,
//    then m_x, the sum and the scale in fp32); the last warp to count in merges them.
#include <mutex>
#include <type_traits>

#include "fp8.cuh"

namespace {

using namespace b2p;

constexpr int kSub = 16;   // tokens per TMA box (any block size that is a multiple of 16)
constexpr int kTile = 32;  // tokens per stage
constexpr float kNoMax = -1e30f;     // reference before the first key (finite: no inf - inf)
constexpr float kSlack = 8.0f;       // log2 units a score may pass its reference by
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
  int group, layer, block_size, hkv;
  int64_t num_blocks;
  const float* k_scales;  // layer bases [num_blocks, hkv]
  const float* v_scales;
  float scale_log2;
  float* partials;    // [hkv][units][2][record]
  int32_t* counters;  // [hkv][virtual sequences], zero between launches
  int32_t* err;
};

// A virtual sequence: columns col0 .. col0 + cols - 1 of sequence i, keys 0 .. keys - 1.
struct Virtual {
  int seq, row0, qlen, ctx, col0, cols, keys;
};

template <int NC>
__device__ __forceinline__ Virtual virtual_of(const Fp8Params& p, int v) {
  Virtual t;
  if (p.cu == nullptr) {
    t.seq = t.row0 = v;
    t.qlen = 1;
    t.ctx = t.keys = max(0, __ldg(p.ctx + v));
    t.col0 = 0;
    t.cols = p.group;
    return t;
  }
  t.seq = v / p.groups_per_seq;
  t.row0 = __ldg(p.cu + t.seq);
  const int end = __ldg(p.cu + t.seq + 1);
  t.ctx = __ldg(p.ctx + t.seq);
  t.qlen = end - t.row0;
  t.col0 = (v - t.seq * p.groups_per_seq) * NC;
  if (t.qlen <= 0 || t.qlen > p.max_q_len || t.row0 < 0 || end > p.num_rows) t.qlen = 0;
  t.cols = min(NC, t.qlen * p.group - t.col0);
  if (t.cols <= 0) {
    t.cols = t.keys = 0;
    return t;
  }
  const int last = (t.col0 + t.cols - 1) / p.group;  // the group's last row sees the most
  t.keys = max(0, t.ctx - t.qlen + last + 1);
  return t;
}

template <int NC>
__device__ __forceinline__ int tiles_of(const Fp8Params& p, int v, int nv) {
  return v < nv ? (virtual_of<NC>(p, v).keys + kTile - 1) / kTile : 0;
}

template <int D, int NT>
struct Fp8Record {
  static constexpr int kOBytes = (D / 16) * NT * 32 * 8;
  static constexpr int kM = kOBytes / 4;  // float index of the references
  static constexpr int kL = kM + NT * 8;  // ... of the sums
  static constexpr int kS = kL + NT * 8;  // ... of the scales
  static constexpr int kFloats = kS + NT * 8;
};

struct Fp8Range {
  int64_t begin, end, total, parts, cb0;  // tiles of this unit; first tile of seq0
  int seq0;
};

__device__ __forceinline__ int64_t unit_start(int64_t c, int64_t total, int64_t parts) {
  return (c * total) / parts;
}

__device__ __forceinline__ int64_t unit_of(int64_t b, int64_t total, int64_t parts) {
  return ((b + 1) * parts - 1) / total;
}

// One warp: all tiles counted, then the virtual sequence that holds unit c's first one. A lane
// owns kPer consecutive ones of a 32 * kPer chunk and loads them before any arithmetic.
template <int NC>
__device__ void find_unit(const Fp8Params& p, int nv, int64_t parts, int64_t c, Fp8Range& r) {
  constexpr int kPer = 8, kChunk = 32 * kPer;
  const int lane = threadIdx.x & 31;
  int nt[kPer];
  int64_t total = 0;
  for (int base = 0; base < nv; base += kChunk) {
    int sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) nt[j] = tiles_of<NC>(p, base + lane * kPer + j, nv);
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += nt[j];
    total += __reduce_add_sync(0xffffffffu, (unsigned)sum);
  }
  r.total = total;
  r.parts = parts < total ? parts : total;  // every range holds a tile
  r.seq0 = nv;
  r.cb0 = total;
  r.begin = r.end = 0;
  if (c >= r.parts) return;
  r.begin = unit_start(c, total, r.parts);
  r.end = unit_start(c + 1, total, r.parts);
  int64_t run = 0;
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
      int seq = 0;
      int64_t cb = run + incl - sum;
      if (lane == src) {
        int k = 0;
        bool found = false;
#pragma unroll
        for (int j = 0; j < kPer - 1; ++j) {
          if (!found && cb + nt[j] <= r.begin) {
            cb += nt[j];
            k = j + 1;
          } else {
            found = true;
          }
        }
        seq = base + lane * kPer + k;
      }
      r.seq0 = __shfl_sync(0xffffffffu, seq, src);
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
  int win;         // first virtual sequence that can hold the next chunk
  int64_t win_cb;  // its first tile
  int64_t begin, n;

  __device__ Slots operator()(const Fp8Params& p, int nv, int64_t chunk0, int lane, int32_t num_slots) {
    const unsigned all = 0xffffffffu;
    const int64_t g = begin + chunk0 + lane;
    const bool valid = chunk0 + lane < n;
    int my = -1;
    int64_t my_cb = 0;
    while (true) {  // windows of 32 virtual sequences
      const int nt = tiles_of<NC>(p, win + lane, nv);
      int incl = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(all, incl, o);
        if (lane >= o) incl += y;
      }
      const int64_t end = win_cb + incl;
      int lo = 0, hi = 32;  // smallest j whose end passes g
#pragma unroll
      for (int step = 0; step < 6; ++step) {
        const int mid = (lo + hi) >> 1;
        const int64_t e = __shfl_sync(all, end, mid < 32 ? mid : 31);
        if (lo < hi) {
          if (e > g) hi = mid; else lo = mid + 1;
        }
      }
      const int64_t first = __shfl_sync(all, end - nt, lo < 32 ? lo : 31);
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
    const int tok = (int)(g - my_cb) * kTile;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = tok + h * kSub;
      if (t >= v.keys) continue;
      const int64_t col = t / p.block_size;
      const int32_t blk = col < p.bt_stride ? __ldg(p.block_tables + (int64_t)v.seq * p.bt_stride + col) : -1;
      if (blk < 0 || blk >= p.num_blocks) {
        set_device_error(p.err, B2P_DEV_BLOCK_RANGE);
      } else {
        s.block[h] = blk;
        s.slot[h] = blk * p.block_size + t % p.block_size;
      }
    }
    return s;
  }
};

// Byte offset of 16-byte chunk `chunk` of token row `tok` in a box of D-byte rows, as the TMA
// unit swizzles it (128-byte rows: chunk ^ row mod 8; 64-byte rows: chunk ^ row / 2 mod 4): the
// eight rows of an ldmatrix phase then lie in eight different 16-byte bank groups.
template <int D>
__device__ __forceinline__ uint32_t box_off(int tok, int chunk) {
  return D == 128 ? (uint32_t)(tok * 128 + ((chunk ^ (tok & 7)) << 4))
                  : (uint32_t)(tok * 64 + ((chunk ^ ((tok >> 1) & 3)) << 4));
}

__device__ __forceinline__ uint32_t cvt_lo(uint32_t w) { return fp8x2_to_f16x2((uint16_t)w); }
__device__ __forceinline__ uint32_t cvt_hi(uint32_t w) { return fp8x2_to_f16x2((uint16_t)(w >> 16)); }

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
  constexpr bool kQShared = NT > 2;         // Q fragments in shared memory
  constexpr int kQBytes = kQShared ? kChunks * NT * 32 * 8 : 0;
  using Rec = Fp8Record<D, NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // Programmatic dependent launch, as in the 16-bit decode kernel: before the wait only
  // lengths, offsets and block tables are read, which no kernel that lets its successor start
  // early writes (the cache write and the table kernels do not).
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.y;
  uint8_t* ring = smem + (size_t)warp * S * kStage;
  uint2* qsm = reinterpret_cast<uint2*>(smem + (size_t)W * S * kStage + (size_t)warp * kQBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)W * (S * kStage + kQBytes)) + warp * S;
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
        bad = empty || (p.cu != nullptr && t.cols > 0 && t.ctx < t.qlen);
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
  const int64_t unit = (int64_t)blockIdx.x * W + warp;
  find_unit<NC>(p, nv, (int64_t)gridDim.x * W, unit, r);
  if (r.begin >= r.end) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (empties_warp) write_empties();
    return;
  }
  const int64_t n = r.end - r.begin;
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
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // scales of this lane's tile, by half: loaded with the slots, a chunk ahead of their use
  float ks_cur[2], vs_cur[2], ks_nxt[2], vs_nxt[2];
  auto load_scales = [&](const Slots& s, float (&ks)[2], float (&vs)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool have = s.block[h] >= 0;
      const int64_t at = (int64_t)(have ? s.block[h] : 0) * p.hkv + head;
      ks[h] = have ? __ldg(p.k_scales + at) : 0.f;
      vs[h] = have ? __ldg(p.v_scales + at) : 0.f;
    }
  };
  load_scales(cur, ks_cur, vs_cur);
  ks_nxt[0] = ks_nxt[1] = vs_nxt[0] = vs_nxt[1] = 0.f;
  int64_t issue_base = 0;  // tiles [issue_base, issue_base + 32) are in the issue slots
  Slots isl = cur;         // slots that the issue side reads (may run a chunk ahead of the scales)
  int64_t issued = 0, use_base = 0;
  bool aborted = false;

  auto issue = [&](int64_t k) {
    if (k >= issue_base + 32) {
      issue_base += 32;
      isl = nxt;
    }
    const int32_t s0 = __shfl_sync(0xffffffffu, isl.slot[0], (int)(k - issue_base));
    const int32_t s1 = __shfl_sync(0xffffffffu, isl.slot[1], (int)(k - issue_base));
    if (lane == 0) {
      const int st = (int)(k % S);
      uint8_t* dst = ring + st * kStage;
      mbar_arrive_expect_tx(&full[st], kStage);
      tma_load_5d(dst, &kmap, &full[st], 0, 0, head, s0, p.layer);
      tma_load_5d(dst + kBox, &kmap, &full[st], 0, 0, head, s1, p.layer);
      tma_load_5d(dst + 2 * kBox, &vmap, &full[st], 0, 0, head, s0, p.layer);
      tma_load_5d(dst + 3 * kBox, &vmap, &full[st], 0, 0, head, s1, p.layer);
    }
    issued = k + 1;
  };
  for (int64_t k = 0; k < S && k < n; ++k) issue(k);
  if (empties_warp) write_empties();  // while the first tiles are in flight
  if (n > 32) {
    nxt = res(p, nv, 32, lane, num_slots);
    load_scales(nxt, ks_nxt, vs_nxt);
  }

  int npend = 0;  // virtual sequences left as partials (at most the unit's first and last)
  int pend_v[2] = {0, 0};
  int64_t pend_cb[2] = {0, 0};
  int pend_nt[2] = {0, 0};

  // Rows of one virtual sequence from O^T fragments: out = O * factor.
  auto write_out = [&](const Virtual& t, float (&o)[kChunks][NT][4], float (&f)[NT][2]) {
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const int c = nn * 8 + 2 * t4 + cc;
        if (c >= t.cols) continue;
        const int col = t.col0 + c;
        T* orow = reinterpret_cast<T*>(p.out) + (int64_t)(t.row0 + col / p.group) * p.o_tok +
                  (int64_t)(head * p.group + col % p.group) * p.o_head;
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
          *reinterpret_cast<uint32_t*>(orow + i * 16 + 2 * g8) =
              pack2<T>(o[i][nn][cc] * f[nn][cc], o[i][nn][2 + cc] * f[nn][cc]);
      }
    }
  };

  int v = r.seq0;
  int64_t cb = r.cb0, gidx = r.begin, k = 0;
  while (gidx < r.end) {
    const Virtual t = virtual_of<NC>(p, v);
    const int ntl = (t.keys + kTile - 1) / kTile;
    if (ntl == 0) {  // written by the empties warp
      ++v;
      continue;
    }
    const int lb0 = (int)(gidx - cb);
    const int64_t seg_end = min(r.end, cb + ntl);
    const int lb1 = (int)(seg_end - cb);

    // ---- Q fragments: column nn * 8 + g8, dims 16c + 4 t4 .. + 3 (8 bytes per lane and k-step)
    uint2 qf[kQShared ? 1 : kChunks][kQShared ? 1 : NT];
    float qfac[NT][2];  // scale_log2 / (power of two the query row was multiplied by)
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
      const int c = nn * 8 + g8;
      const bool ok = c < t.cols;
      const int col = t.col0 + (ok ? c : 0);
      const T* qrow = reinterpret_cast<const T*>(p.q) + (int64_t)(t.row0 + col / p.group) * p.q_tok +
                      (int64_t)(head * p.group + col % p.group) * p.q_head + 4 * t4;
      uint2 w[kChunks];
#pragma unroll
      for (int kk = 0; kk < kChunks; ++kk)
        w[kk] = ok ? __ldg(reinterpret_cast<const uint2*>(qrow + kk * 16)) : make_uint2(0u, 0u);
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
      if constexpr (kQShared) {
        if (nn == 0) __syncwarp();  // the previous segment's reads are done
#pragma unroll
        for (int kk = 0; kk < kChunks; ++kk) qsm[(kk * NT + nn) * 32 + lane] = w[kk];
      } else {
#pragma unroll
        for (int kk = 0; kk < kChunks; ++kk) qf[kk][nn] = w[kk];
      }
    }
    // keys that each of this lane's columns sees (columns past the last: none)
    int lim[NT][2];
    int lim_min = t.keys;
#pragma unroll
    for (int nn = 0; nn < NT; ++nn)
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const int c = nn * 8 + 2 * t4 + cc;
        lim[nn][cc] = p.cu == nullptr ? t.keys : c < t.cols ? t.ctx - t.qlen + (t.col0 + c) / p.group + 1 : t.keys;
      }
    if (p.cu != nullptr) lim_min = t.ctx - t.qlen + t.col0 / p.group + 1;

    float mx[NT][2], my[NT][2], gy[NT][2], l[NT][2];
    float acc[kChunks][NT][4];
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
      mx[nn][0] = mx[nn][1] = my[nn][0] = my[nn][1] = kNoMax;
      gy[nn][0] = gy[nn][1] = 1.f;
      l[nn][0] = l[nn][1] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int nn = 0; nn < NT; ++nn) acc[i][nn][0] = acc[i][nn][1] = acc[i][nn][2] = acc[i][nn][3] = 0.f;

    for (int lb = lb0; lb < lb1; ++lb, ++k) {
      if (k >= use_base + 32) {  // rotate the scale buffers; the issue side has moved on already
        use_base += 32;
        ks_cur[0] = ks_nxt[0], ks_cur[1] = ks_nxt[1], vs_cur[0] = vs_nxt[0], vs_cur[1] = vs_nxt[1];
        if (use_base + 32 < n) {
          nxt = res(p, nv, use_base + 32, lane, num_slots);
          load_scales(nxt, ks_nxt, vs_nxt);
        }
      }
      const int src = (int)(k - use_base);
      float ks[2], vs[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[h] = __shfl_sync(0xffffffffu, ks_cur[h], src);
        vs[h] = __shfl_sync(0xffffffffu, vs_cur[h], src);
      }
      const int st = (int)(k % S);
      if (!aborted && !mbar_wait_bounded(&full[st], (uint32_t)((k / S) & 1), p.err)) aborted = true;
      aborted = __any_sync(0xffffffffu, aborted);
      if (aborted) continue;  // keep walking so every sequence still gets written
      uint8_t* stage = ring + st * kStage;
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
      const uint32_t base = smem_u32(stage);

      // ---- S^T = K Q^T: 2 x 16 tokens, NC columns
      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nn = 0; nn < NT; ++nn) s[h][nn][0] = s[h][nn][1] = s[h][nn][2] = s[h][nn][3] = 0.f;
      {
        const int tok = (lane & 7) + ((lane >> 3) & 1) * 8, dc = lane >> 4;
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint2 b[2][NT];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              b[j][nn] = kQShared ? qsm[((c + j) * NT + nn) * 32 + lane] : qf[kQShared ? 0 : c + j][kQShared ? 0 : nn];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a0, a1, a2, a3;
            ldmatrix_x4(base + h * kBox + box_off<D>(tok, c + dc), a0, a1, a2, a3);
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              MmaOp<__half>::run(s[h][nn], cvt_lo(a0), cvt_lo(a1), cvt_hi(a0), cvt_hi(a1), b[0][nn].x, b[0][nn].y);
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              MmaOp<__half>::run(s[h][nn], cvt_lo(a2), cvt_lo(a3), cvt_hi(a2), cvt_hi(a3), b[1][nn].x, b[1][nn].y);
          }
        }
      }

      // ---- scores in log2 units, masked where a column's rows end
      const bool masked = tok0 + kTile > lim_min;
      bool over = false;
      const float ev[2] = {scale_exp(vs[0]), scale_exp(vs[1])};
#pragma unroll
      for (int nn = 0; nn < NT; ++nn)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const float f = qfac[nn][cc];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x0 = s[h][nn][cc] * (ks[h] * f), x1 = s[h][nn][2 + cc] * (ks[h] * f);
            if (masked) {
              const int left = lim[nn][cc] - tok0 - h * kSub;
              if (g8 >= left) x0 = -INFINITY;
              if (g8 + 8 >= left) x1 = -INFINITY;
            }
            s[h][nn][cc] = x0;
            s[h][nn][2 + cc] = x1;
            const float top = fmaxf(x0, x1);
            over |= top - mx[nn][cc] > kSlack || top + ev[h] - my[nn][cc] > kSlack;
          }
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
            const float nx = fmaxf(mx[nn][cc], fmaxf(t0, t1));
            const float ny = fmaxf(my[nn][cc], fmaxf(t0 + ev[0], t1 + ev[1]));
            l[nn][cc] *= fast_exp2(mx[nn][cc] - nx);
            const float al = fast_exp2(my[nn][cc] - ny);
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
              acc[i][nn][cc] *= al;
              acc[i][nn][2 + cc] *= al;
            }
            mx[nn][cc] = nx;
            my[nn][cc] = ny;
            gy[nn][cc] = fast_exp2(nx - ny);
          }
      }
      // ---- P = 2^(x - m_x); its f16 copy carries vs against m_y
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nn = 0; nn < NT; ++nn) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float pv[4];
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const float p0 = fast_exp2(s[h][nn][cc] - mx[nn][cc]), p1 = fast_exp2(s[h][nn][2 + cc] - mx[nn][cc]);
            l[nn][cc] += p0 + p1;
            float f = vs[h] * gy[nn][cc];
            f = f > 0x1p126f ? 0x1p126f : f;  // a block whose weights have all underflowed; NaN stays
            pv[cc] = p0 * f;
            pv[2 + cc] = p1 * f;
            if (masked) {  // 0 * NaN of a poisoned block
              const int left = lim[nn][cc] - tok0 - h * kSub;
              if (g8 >= left) pv[cc] = 0.f;
              if (g8 + 8 >= left) pv[2 + cc] = 0.f;
            }
          }
          pb[h][nn][0] = movmatrix_trans(pack2<__half>(pv[0], pv[1]));
          pb[h][nn][1] = movmatrix_trans(pack2<__half>(pv[2], pv[3]));
        }
      }

      // ---- O^T += V^T P^T: 16 dims per fragment (even ones in rows 0..7, odd ones in 8..15)
      {
        const int tok = (lane & 7) + ((lane >> 3) & 1) * 8, dc = lane >> 4;
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a0, a1, a2, a3;
            ldmatrix_x4_trans(base + (2 + h) * kBox + box_off<D>(tok, c + dc), a0, a1, a2, a3);
            a0 = __byte_perm(a0, 0, 0x3120), a1 = __byte_perm(a1, 0, 0x3120);
            a2 = __byte_perm(a2, 0, 0x3120), a3 = __byte_perm(a3, 0, 0x3120);
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              MmaOp<__half>::run(acc[c][nn], cvt_lo(a0), cvt_hi(a0), cvt_lo(a1), cvt_hi(a1), pb[h][nn][0], pb[h][nn][1]);
#pragma unroll
            for (int nn = 0; nn < NT; ++nn)
              MmaOp<__half>::run(acc[c + 1][nn], cvt_lo(a2), cvt_hi(a2), cvt_lo(a3), cvt_hi(a3), pb[h][nn][0], pb[h][nn][1]);
          }
        }
      }
      // Refill the stage: its reads fed the MMAs above; generic writes need a proxy fence before
      // the TMA unit writes the same bytes.
      if (valid < kTile) fence_proxy_async_smem();
      __syncwarp();
      if (k + S < n) issue(k + S);
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
      float f[NT][2];
#pragma unroll
      for (int nn = 0; nn < NT; ++nn)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc)
          f[nn][cc] = l[nn][cc] > 0.f ? fast_exp2(my[nn][cc] - mx[nn][cc]) / l[nn][cc] : 0.f;
      write_out(t, acc, f);
    } else {
      const int which = (cb + lb0 == r.begin) ? 0 : 1;  // the unit's first segment or a later one
      float* rec = p.partials + (((size_t)head * r.parts + unit) * 2 + which) * Rec::kFloats;
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
          reinterpret_cast<uint2*>(rec)[(i * NT + nn) * 32 + lane] =
              make_uint2(pack2<__half>(acc[i][nn][0] * f0, acc[i][nn][1] * f1),
                         pack2<__half>(acc[i][nn][2] * f0, acc[i][nn][3] * f1));
        if (g8 == 0) {
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            rec[Rec::kM + nn * 8 + 2 * t4 + cc] = mx[nn][cc];
            rec[Rec::kL + nn * 8 + 2 * t4 + cc] = l[nn][cc];
            rec[Rec::kS + nn * 8 + 2 * t4 + cc] =
                l[nn][cc] > 0.f ? top[cc] * (fast_exp2(my[nn][cc] - mx[nn][cc]) / l[nn][cc]) : 0.f;
          }
        }
      }
      if (npend < 2) {  // counted in after the stream: a fence now would stall its refills
        pend_v[npend] = v;
        pend_cb[npend] = cb;
        pend_nt[npend] = ntl;
        ++npend;
      }
    }
    gidx = seg_end;
    if (lb1 == ntl) {
      cb += ntl;
      ++v;
    }
  }
  // Never leave with TMA writes in flight (only after an abort: every issued tile is waited for).
  if (lane == 0)
    for (int64_t kk = k; kk < issued; ++kk) mbar_wait_bounded(&full[kk % S], (uint32_t)((kk / S) & 1), nullptr);

  // ---- count this warp's partials in; the last one of a virtual sequence merges them
  int last_mask = 0;
  __syncwarp();
  if (lane == 0 && npend > 0) {
    asm volatile("fence.acq_rel.gpu;" ::: "memory");  // the warp's records before its counts
    int prev[2] = {0, 0};
    for (int j = 0; j < npend; ++j) prev[j] = atomicAdd(p.counters + (size_t)head * nv + pend_v[j], 1);
    for (int j = 0; j < npend; ++j) {
      const int64_t uf = unit_of(pend_cb[j], r.total, r.parts);
      const int64_t ul = unit_of(pend_cb[j] + pend_nt[j] - 1, r.total, r.parts);
      if (prev[j] == (int)(ul - uf)) {
        p.counters[(size_t)head * nv + pend_v[j]] = 0;
        last_mask |= 1 << j;
      }
    }
    if (last_mask) asm volatile("fence.acq_rel.gpu;" ::: "memory");
  }
  last_mask = __shfl_sync(0xffffffffu, last_mask, 0);
  for (int j = 0; j < npend; ++j) {
    if (!((last_mask >> j) & 1)) continue;
    const int64_t scb = pend_cb[j];
    const int64_t u0 = unit_of(scb, r.total, r.parts), u1 = unit_of(scb + pend_nt[j] - 1, r.total, r.parts);
    float M[NT][2], L[NT][2];
    float O[kChunks][NT][4];
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
      M[nn][0] = M[nn][1] = kNoMax;
      L[nn][0] = L[nn][1] = 0.f;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) O[i][nn][0] = O[i][nn][1] = O[i][nn][2] = O[i][nn][3] = 0.f;
    }
    constexpr int kBatch = NT == 1 ? 4 : NT == 2 ? 2 : 1;  // records loaded together (registers)
    for (int64_t ub = u0; ub <= u1; ub += kBatch) {
      float mv[kBatch][NT][2], lv[kBatch][NT][2], sv[kBatch][NT][2];
      uint2 ov[kBatch][kChunks][NT];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int64_t u = ub + b;
        const bool have = u <= u1;
        const int which = (u == u0 && unit_start(u, r.total, r.parts) != scb) ? 1 : 0;
        const float* pr = p.partials + (((size_t)head * r.parts + (have ? u : u0)) * 2 + which) * Rec::kFloats;
#pragma unroll
        for (int nn = 0; nn < NT; ++nn) {
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            mv[b][nn][cc] = have ? __ldcg(pr + Rec::kM + nn * 8 + 2 * t4 + cc) : kNoMax;
            lv[b][nn][cc] = have ? __ldcg(pr + Rec::kL + nn * 8 + 2 * t4 + cc) : 0.f;
            sv[b][nn][cc] = have ? __ldcg(pr + Rec::kS + nn * 8 + 2 * t4 + cc) : 0.f;
          }
#pragma unroll
          for (int i = 0; i < kChunks; ++i)
            ov[b][i][nn] = have ? __ldcg(reinterpret_cast<const uint2*>(pr) + (i * NT + nn) * 32 + lane) : make_uint2(0u, 0u);
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
#pragma unroll
        for (int nn = 0; nn < NT; ++nn) {
          float w[2], a[2];
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const float mn = fmaxf(M[nn][cc], mv[b][nn][cc]);
            a[cc] = fast_exp2(M[nn][cc] - mn);
            w[cc] = fast_exp2(mv[b][nn][cc] - mn) * lv[b][nn][cc];
            L[nn][cc] = L[nn][cc] * a[cc] + w[cc];
            M[nn][cc] = mn;
            w[cc] *= sv[b][nn][cc];
          }
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&ov[b][i][nn].x));
            const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&ov[b][i][nn].y));
            O[i][nn][0] = O[i][nn][0] * a[0] + lo.x * w[0];
            O[i][nn][1] = O[i][nn][1] * a[1] + lo.y * w[1];
            O[i][nn][2] = O[i][nn][2] * a[0] + hi.x * w[0];
            O[i][nn][3] = O[i][nn][3] * a[1] + hi.y * w[1];
          }
        }
    }
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
      L[nn][0] = L[nn][0] > 0.f ? 1.f / L[nn][0] : 0.f;
      L[nn][1] = L[nn][1] > 0.f ? 1.f / L[nn][1] : 0.f;
    }
    write_out(virtual_of<NC>(p, pend_v[j]), O, L);
  }
}

// ====================================================================== host side
struct Fp8Plan {
  const void* fn = nullptr;
  int smem = 0, warps = 0, columns = 0;
};

template <typename T, int D, int NT, int S, int W>
Fp8Plan make_fp8_plan() {
  static_assert(W <= 8 && NT <= 4 && D <= 128, "the workspace has room for these");
  Fp8Plan pl;
  pl.fn = reinterpret_cast<const void*>(&paged_rows_fp8<T, D, NT, S, W>);
  pl.smem = W * S * 4 * kSub * D + (NT > 2 ? W * (D / 16) * NT * 32 * 8 : 0) + W * S * 8 + 1024;
  pl.warps = W;
  pl.columns = NT * 8;
  return pl;
}

template <typename T>
bool select_fp8_plan(int head_dim, int columns, Fp8Plan& pl) {
  if (head_dim == 128)
    pl = columns <= 8 ? make_fp8_plan<T, 128, 1, 3, 8>()
         : columns <= 16 ? make_fp8_plan<T, 128, 2, 3, 8>()
                         : make_fp8_plan<T, 128, 4, 2, 8>();
  else if (head_dim == 64)
    pl = columns <= 8 ? make_fp8_plan<T, 64, 1, 4, 8>()
         : columns <= 16 ? make_fp8_plan<T, 64, 2, 4, 8>()
                         : make_fp8_plan<T, 64, 4, 4, 8>();
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
constexpr int kMostColumns = 32;   // per virtual sequence
constexpr int kMostUnits = 8;      // warps per CTA of any plan
constexpr int kRowColumns = 64;    // columns per sequence that calls here have at most

size_t records_bytes(int num_kv_heads) {
  const int64_t ctas = num_kv_heads > b2p_host::sm_count() ? num_kv_heads : b2p_host::sm_count();
  return (size_t)ctas * kMostUnits * 2 * Fp8Record<128, kMostColumns / 8>::kFloats * 4;
}

int column_groups(const Fp8Plan& pl, int group, int max_q_len) {
  return (int)(((int64_t)group * max_q_len + pl.columns - 1) / pl.columns);
}

}  // namespace

// Whether calls of this shape run here; rows beyond a few per sequence belong to the tile kernel.
bool b2p_rows_fp8_takes(int group, int head_dim, int block_size, int dtype, int max_q_len) {
  Fp8Plan pl;
  return (dtype == B2P_BF16 || dtype == B2P_F16) && block_size % kSub == 0 && max_q_len >= 1 &&
         (max_q_len > 1 || group <= 32) && (int64_t)group * max_q_len <= kRowColumns &&
         select_fp8_plan<__half>(head_dim, group * max_q_len, pl);
}

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
  p.layer = (int)layer_index;
  p.block_size = block_size;
  p.hkv = num_kv_heads;
  p.num_blocks = num_slots / block_size;
  p.k_scales = key_scales + layer_index * p.num_blocks * num_kv_heads;
  p.v_scales = value_scales + layer_index * p.num_blocks * num_kv_heads;
  p.scale_log2 = scale * kLog2e;
  p.partials = static_cast<float*>(workspace);
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
