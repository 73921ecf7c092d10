// K8 — verification of drafted tokens (speculative decoding).
//
// Sequence i drafted k_i tokens x_0 .. x_{k-1}; row j of its k_i + 1 target rows is the target
// model's distribution p_j for the token after x_{j-1}, and q_j is the distribution x_j was
// drafted from. Draft j is accepted while u_j * q_j(x_j) < p_j(x_j). Then one more token is
// drawn with v: with n accepted, the first index where the running sum of r exceeds v * sum(r),
//   r = max(p_n - q_n, 0) after a rejection (p_n itself where that is zero everywhere),
//   r = p_k               with all k accepted.
// Without draft probabilities the draft is certain: q_j is 1 at x_j and 0 elsewhere. The token
// stream this gives is distributed as the target model's own.
//
// Bytes: a handful of gathered values, then one row pair (p_n, q_n) per sequence, read once;
// everything else is latency. One cluster of CTAs owns a sequence: every CTA takes a slice of the
// vocabulary and every warp a contiguous piece of the slice, in 16-byte loads; the piece sums
// meet in distributed shared memory, and only the one piece that holds the crossing is read again
// (from L2) to find the index. All sums are fp64 in a fixed order: p - q and u * q of fp32
// inputs are exact there, and a token's interval is as narrow as its probability, so fp32
// sums over 150,000 entries would move draws across the borders of rare tokens. (The
// conversions to fp64, two per entry, are what an SM has least of: a quarter of the time that
// the entry's 8 bytes take from HBM.)
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

using namespace b2p;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMostRanks = 8;  // CTAs of a cluster

struct VerifyParams {
  const uint8_t* target;  // [total + num_seqs, vocab]
  int64_t t_row;          // element strides
  const uint8_t* draft;   // [total, vocab] or null
  int64_t d_row;
  const int64_t* tokens;  // [total]
  const int32_t* cu;      // [num_seqs + 1]
  const float* accept;    // [total]
  const float* sample;    // [num_seqs]
  int64_t total;
  int num_seqs, max_drafts, vocab;
  int64_t* out;  // [num_seqs, max_drafts + 1]
  int64_t out_row;
  int32_t* accepted;
  int32_t* err;
};

// What a CTA needs to know of its sequence.
struct Row {
  int begin, k, n;   // first draft, drafts, accepted
  int rejected;      // the rejected token, -1: none (or out of range)
};

// Entries of both rows pass through this before they are compared or subtracted (a NaN or a
// negative q takes nothing from p): 49.0 us for 256 sequences, 48.2 with p alone.
__device__ __forceinline__ double positive(double x) { return x > 0.0 ? x : 0.0; }  // NaN: 0

template <typename T>
__device__ __forceinline__ double residual(const T* p, const T* q, int drop, int v) {
  const double x = positive((double)to_f32<T>(p[v]));
  if (q != nullptr) return positive(x - positive((double)to_f32<T>(q[v])));
  return v == drop ? 0.0 : x;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Sum of the residual over [v0, v1) of one warp's piece, in 16-byte loads where both rows start on
// a 16-byte boundary (pieces do within a row).
template <typename T, bool kDraft>
__device__ __forceinline__ double piece_sum(const T* p, const T* q, int drop, int v0, int v1, int lane) {
  constexpr int kPer = 16 / sizeof(T);
  double s = 0.0;
  if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0) {
    constexpr int kAhead = 4;  // loads of each row in flight per lane
    const int whole = v0 + (v1 - v0) / kPer * kPer;  // the row's last piece may end unaligned
    for (int v = v0 + lane * kPer; v < whole; v += 32 * kPer * kAhead) {
      uint4 a[kAhead], b[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int at = v + k * 32 * kPer;
        a[k] = b[k] = make_uint4(0, 0, 0, 0);
        if (at < whole) {
          a[k] = __ldcs(reinterpret_cast<const uint4*>(p + at));
          if (kDraft) b[k] = __ldcs(reinterpret_cast<const uint4*>(q + at));
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const T* x = reinterpret_cast<const T*>(&a[k]);
        const T* y = reinterpret_cast<const T*>(&b[k]);
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          float u = to_f32<T>(x[e]);
          if (kDraft) {
            float w = fmaxf(to_f32<T>(y[e]), 0.f);  // NaN: 0
            const bool more = u > w;  // false for NaN and for what is not positive
            u = more ? u : 0.f;
            w = more ? w : 0.f;
            s += (double)u - (double)w;
          } else {
            s += (double)(u > 0.f && v + k * 32 * kPer + e != drop ? u : 0.f);
          }
        }
      }
    }
    if (whole + lane < v1) s += residual<T>(p, kDraft ? q : nullptr, drop, whole + lane);
  } else {
    for (int v = v0 + lane; v < v1; v += 32) s += residual<T>(p, kDraft ? q : nullptr, drop, v);
  }
  return warp_sum(s);
}

// kLoads * 16 bytes of both rows from entry a on, kept as they come.
template <typename T, int kLoads>
struct Run {
  static constexpr int kPer = 16 / sizeof(T);
  static constexpr int kEntries = kLoads * kPer;
  uint4 u[kLoads], w[kLoads];

  // Zeros from w1 on; 16-byte loads where both rows start on a 16-byte boundary (a is a multiple
  // of as much).
  __device__ __forceinline__ void load(const T* p, const T* q, int a, int w1) {
    const bool wide = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0;
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
      const int at = a + c * kPer;
      u[c] = w[c] = make_uint4(0, 0, 0, 0);
      if (wide && at + kPer <= w1) {
        u[c] = __ldg(reinterpret_cast<const uint4*>(p + at));
        if (q != nullptr) w[c] = __ldg(reinterpret_cast<const uint4*>(q + at));
      } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          if (at + k < w1) {
            reinterpret_cast<T*>(&u[c])[k] = p[at + k];
            if (q != nullptr) reinterpret_cast<T*>(&w[c])[k] = q[at + k];
          }
        }
      }
    }
  }
  __device__ __forceinline__ double residual(int e) const {  // of entry a + e (not the dropped one)
    const float p = to_f32<T>(reinterpret_cast<const T*>(&u[e / kPer])[e % kPer]);
    const float q = to_f32<T>(reinterpret_cast<const T*>(&w[e / kPer])[e % kPer]);
    return positive((double)fmaxf(p, 0.f) - (double)fmaxf(q, 0.f));
  }
};

// The first entry of [w0, w1) at which the running sum, `at` before w0, passes goal goes to *pick
// (which no later entry then replaces), the last one with anything to *tail. The piece is read once,
// a contiguous run per thread and round that stays in registers between the scan and the search.
template <typename T, int kLoads>
__device__ __forceinline__ void find_crossing(const T* prow, const T* qrow, int drop, int w0, int w1, double at,
                                              double goal, bool crossing, double* scan, int* pick, int* tail) {
  constexpr int kNone = 0x7fffffff;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r0 = w0; r0 < w1; r0 += kThreads * Run<T, kLoads>::kEntries) {
    const int a = r0 + (int)threadIdx.x * Run<T, kLoads>::kEntries;
    Run<T, kLoads> x;
    x.load(prow, qrow, a, w1);
    double mine = 0.0;
#pragma unroll
    for (int e = 0; e < Run<T, kLoads>::kEntries; ++e) mine += a + e == drop ? 0.0 : x.residual(e);
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    double before = at;
    for (int k = 0; k < kWarps; ++k) {
      if (k < warp) before += scan[k];
      at += scan[k];
    }
    before += incl - mine;
    int first = kNone, last_one = -1;
#pragma unroll
    for (int e = 0; e < Run<T, kLoads>::kEntries; ++e) {
      const double r = a + e == drop ? 0.0 : x.residual(e);
      before += r;
      if (r > 0.0) {
        last_one = a + e;
        if (crossing && before > goal) first = min(first, a + e);
      }
    }
    first = __reduce_min_sync(0xffffffffu, first);
    last_one = __reduce_max_sync(0xffffffffu, last_one);
    if (lane == 0) {
      atomicMin(pick, first);
      atomicMax(tail, last_one);
    }
    __syncthreads();
    if (*pick < kNone) return;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) verify_drafts(const VerifyParams p) {
  __shared__ Row row;
  __shared__ double piece[kWarps];  // sums over the warps' pieces
  __shared__ double total;          // this CTA's
  __shared__ double scan[kWarps];
  __shared__ int pick, tail;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int ranks = (int)cluster.num_blocks();
  const int seq = blockIdx.x / ranks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {  // how many drafts stand (every CTA of the cluster finds the same)
    Row r;
    r.begin = __ldg(p.cu + seq);
    const int end = __ldg(p.cu + seq + 1);
    r.k = end - r.begin;
    r.n = 0;
    r.rejected = -1;
    if (r.begin < 0 || r.k < 0 || r.k > p.max_drafts || end > p.total) {
      if (rank == 0 && lane == 0) set_device_error(p.err, B2P_DEV_LENGTH);
      r.k = -1;
    }
    for (int base = 0; base < r.k; base += 32) {
      const int j = base + lane;
      bool ok = false;
      int64_t x = -1;
      if (j < r.k) {
        x = p.tokens[r.begin + j];
        if (x < 0 || x >= p.vocab) {
          if (rank == 0) set_device_error(p.err, B2P_DEV_TOKEN_RANGE);
          x = -1;
        } else {
          const T* prow = reinterpret_cast<const T*>(p.target) + ((int64_t)r.begin + seq + j) * p.t_row;
          const T* qrow = reinterpret_cast<const T*>(p.draft) + (int64_t)(r.begin + j) * p.d_row;
          const double qx = p.draft != nullptr ? positive((double)to_f32<T>(qrow[x])) : 1.0;
          ok = (double)p.accept[r.begin + j] * qx < positive((double)to_f32<T>(prow[x]));
        }
      }
      const unsigned stop = __ballot_sync(0xffffffffu, j < r.k && !ok);
      if (stop) {
        const int first = __ffs(stop) - 1;
        r.n = base + first;
        r.rejected = (int)__shfl_sync(0xffffffffu, x, first);
        break;
      }
      r.n = min(base + 32, r.k);
    }
    if (lane == 0) row = r;
    if (rank == 0) {
      int64_t* out = p.out + (int64_t)seq * p.out_row;
      for (int j = lane; j <= p.max_drafts; j += 32)
        if (j != r.n || r.k < 0) out[j] = j < r.n ? p.tokens[r.begin + j] : -1;
      if (lane == 0) p.accepted[seq] = r.n;
    }
  }
  if (threadIdx.x == 0) {
    pick = 0x7fffffff;
    tail = -1;
  }
  __syncthreads();
  if (row.k < 0) return;  // the whole cluster returns

  const bool rejected = row.n < row.k;
  const T* prow = reinterpret_cast<const T*>(p.target) + ((int64_t)row.begin + seq + row.n) * p.t_row;
  const T* qrow = rejected && p.draft != nullptr
                      ? reinterpret_cast<const T*>(p.draft) + (int64_t)(row.begin + row.n) * p.d_row
                      : nullptr;
  int drop = rejected && p.draft == nullptr ? row.rejected : -1;
  // the vocabulary in ranks * kWarps pieces, in index order, each a multiple of 16 bytes
  constexpr int kPer = 16 / sizeof(T);
  const int len = ((p.vocab + ranks * kWarps - 1) / (ranks * kWarps) + kPer - 1) / kPer * kPer;
  const int v0 = min(p.vocab, (rank * kWarps + warp) * len), v1 = min(p.vocab, v0 + len);
  double part[kMostRanks];
  double all = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    const double s = qrow != nullptr ? piece_sum<T, true>(prow, qrow, -1, v0, v1, lane)
                                     : piece_sum<T, false>(prow, nullptr, drop, v0, v1, lane);
    if (lane == 0) piece[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double t = 0.0;
      for (int w = 0; w < kWarps; ++w) t += piece[w];
      total = t;
    }
    cluster.sync();
    all = 0.0;
#pragma unroll
    for (int c = 0; c < kMostRanks; ++c) {
      part[c] = c < ranks ? *cluster.map_shared_rank(&total, c) : 0.0;
      all += part[c];
    }
    cluster.sync();  // nobody leaves or writes again while its total may still be read
    if (all > 0.0 || (qrow == nullptr && drop < 0)) break;
    qrow = nullptr;  // nothing left over (p <= q everywhere): the target row itself
    drop = -1;
  }
  const double goal = (double)p.sample[seq] * all;
  // the CTA that holds the crossing; where rounding or a draw outside [0, 1) leaves none, the
  // last one with anything in it
  int owner = -1, last = -1;
  double run = 0.0, base = 0.0;
#pragma unroll
  for (int c = 0; c < kMostRanks; ++c) {
    if (c == rank) base = run;
    run += part[c];
    if (part[c] > 0.0) {
      last = c;
      if (owner < 0 && run > goal) owner = c;
    }
  }
  if (owner < 0) owner = last;
  if (owner < 0) {  // a row without a positive entry
    if (rank == 0 && threadIdx.x == 0) p.out[(int64_t)seq * p.out_row + row.n] = 0;
    return;
  }
  if (owner != rank) return;
  // the same inside the CTA, over its warps' pieces
  int ow = -1, lw = -1;
  double start = base;
  for (int w = 0; w < kWarps; ++w) {
    const double next = base + piece[w];
    if (piece[w] > 0.0) {
      lw = w;
      if (ow < 0) start = base;
      if (ow < 0 && next > goal) ow = w;
    }
    base = next;
  }
  const bool crossing = ow >= 0;
  if (!crossing) ow = lw;
  // The piece again. One load of each row per thread where two rounds of that cover it: long runs
  // of few threads take longer than a round saves (one sequence 10.3 us with three, 8.7 with one;
  // 256 of them, whose pieces are longer, 47 with three).
  const int w0 = min(p.vocab, (rank * kWarps + ow) * len), w1 = min(p.vocab, w0 + len);
  if (len <= 2 * kThreads * Run<T, 1>::kEntries)
    find_crossing<T, 1>(prow, qrow, drop, w0, w1, start, goal, crossing, scan, &pick, &tail);
  else
    find_crossing<T, 3>(prow, qrow, drop, w0, w1, start, goal, crossing, scan, &pick, &tail);
  if (threadIdx.x == 0)
    p.out[(int64_t)seq * p.out_row + row.n] = pick != 0x7fffffff ? pick : tail;
}

// Greedy form: the target rows are given by their arg-max ids; a draft stands while it equals
// the id of its row, and the id of the first row that differs (or of the last one) follows.
__global__ void __launch_bounds__(128) verify_drafts_greedy(const int64_t* ids, const int64_t* tokens,
                                                            const int32_t* cu, int64_t total,
                                                            int num_seqs, int max_drafts, int64_t* out,
                                                            int64_t out_row, int32_t* accepted,
                                                            int32_t* err) {
  const int seq = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (seq >= num_seqs) return;
  const int begin = __ldg(cu + seq), end = __ldg(cu + seq + 1);
  int k = end - begin, n = 0;
  if (begin < 0 || k < 0 || k > max_drafts || end > total) {
    if (lane == 0) set_device_error(err, B2P_DEV_LENGTH);
    k = -1;
  }
  for (int base = 0; base < k; base += 32) {
    const int j = base + lane;
    const bool ok = j < k && tokens[begin + j] == ids[begin + seq + j];
    const unsigned stop = __ballot_sync(0xffffffffu, j < k && !ok);
    if (stop) {
      n = base + __ffs(stop) - 1;
      break;
    }
    n = min(base + 32, k);
  }
  for (int j = lane; j <= max_drafts; j += 32)
    out[(int64_t)seq * out_row + j] =
        k < 0 ? -1 : j < n ? tokens[begin + j] : j == n ? ids[begin + seq + n] : -1;
  if (lane == 0) accepted[seq] = n;
}

}  // namespace

extern "C" int b2p_verify_drafts(const void* target_probs, int64_t target_row_stride,
                                 const void* draft_probs, int64_t draft_row_stride,
                                 const int64_t* draft_tokens, const int32_t* cu_drafts,
                                 const float* accept_draws, const float* sample_draws,
                                 int num_seqs, int64_t total_drafts, int max_drafts, int vocab,
                                 int dtype, int64_t* out_tokens, int64_t out_row_stride,
                                 int32_t* out_accepted, int32_t* err_flag, void* stream) {
  if (num_seqs < 0 || total_drafts < 0 || max_drafts < 0 || vocab <= 0 ||
      dtype < B2P_BF16 || dtype > B2P_F32)
    return B2P_EINVAL;
  if (num_seqs > (1 << 27) || total_drafts > 0x7fffffffLL || vocab > (1 << 30))
    return B2P_EUNSUPPORTED;
  if (num_seqs == 0) return B2P_OK;
  if (!target_probs || !cu_drafts || !sample_draws || !out_tokens || !out_accepted ||
      (total_drafts > 0 && (!draft_tokens || !accept_draws)) || out_row_stride < max_drafts + 1)
    return B2P_EINVAL;
  VerifyParams p;
  p.target = static_cast<const uint8_t*>(target_probs);
  p.t_row = target_row_stride;
  p.draft = static_cast<const uint8_t*>(draft_probs);
  p.d_row = draft_row_stride;
  p.tokens = draft_tokens;
  p.cu = cu_drafts;
  p.accept = accept_draws;
  p.sample = sample_draws;
  p.total = total_drafts;
  p.num_seqs = num_seqs;
  p.max_drafts = max_drafts;
  p.vocab = vocab;
  p.out = out_tokens;
  p.out_row = out_row_stride;
  p.accepted = out_accepted;
  p.err = err_flag;
  cudaLaunchConfig_t cfg = {};
  // CTAs per sequence: as many as fill the GPU with one wave (two CTAs per SM). More only repeat
  // the search for the first rejected draft: 256 sequences over 151,936 entries took 48.6 us with
  // one CTA each, 52 with two, 76 with eight; one sequence 21.7, 14.2 and 8.3 us.
  int ranks = kMostRanks;
  while (ranks > 1 && (int64_t)num_seqs * ranks > 2LL * b2p_host::sm_count()) ranks /= 2;
  cfg.gridDim = dim3((unsigned)(num_seqs * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const void* fn = dtype == B2P_BF16  ? reinterpret_cast<const void*>(&verify_drafts<__nv_bfloat16>)
                   : dtype == B2P_F16 ? reinterpret_cast<const void*>(&verify_drafts<__half>)
                                      : reinterpret_cast<const void*>(&verify_drafts<float>);
  void* args[] = {&p};
  const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
  if (e != cudaSuccess) return b2p_host::record_error(e);
  return b2p_host::check_launch();
}

extern "C" int b2p_verify_drafts_greedy(const int64_t* target_ids, const int64_t* draft_tokens,
                                        const int32_t* cu_drafts, int num_seqs,
                                        int64_t total_drafts, int max_drafts, int64_t* out_tokens,
                                        int64_t out_row_stride, int32_t* out_accepted,
                                        int32_t* err_flag, void* stream) {
  if (num_seqs < 0 || total_drafts < 0 || max_drafts < 0) return B2P_EINVAL;
  if (num_seqs == 0) return B2P_OK;
  if (!target_ids || !cu_drafts || !out_tokens || !out_accepted ||
      (total_drafts > 0 && !draft_tokens) || out_row_stride < max_drafts + 1)
    return B2P_EINVAL;
  verify_drafts_greedy<<<(unsigned)((num_seqs + 3) / 4), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      target_ids, draft_tokens, cu_drafts, total_drafts, num_seqs, max_drafts, out_tokens,
      out_row_stride, out_accepted, err_flag);
  return b2p_host::check_launch();
}
