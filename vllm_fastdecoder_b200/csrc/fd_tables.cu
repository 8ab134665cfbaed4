// Block tables, slots and positions of a step from the requests' lengths.
//
//   need_r = ceil((prior_r + new_r) / BS) - ceil(prior_r / BS)
//   block j of the step (requests in order, positions in order) is
//     stack0[c0 - 1 - j]          for j < c0
//     stack1[c1 - 1 - (j - c0)]   else,
//   c0, c1 the free counts after the ended requests' blocks were pushed.
//
// Integer work on a few bytes per request and 16 per new token, so the launch
// and a handful of dependent memory round trips bound it, not bandwidth.  One
// cluster does all: every CTA loads all lengths into shared memory and scans
// them (the redundant work is one pass over 8 bytes per request), so each can
// place any request, block or token by itself, and the writes are dealt out
// over the CTAs.  Two cluster barriers order what has to be ordered: every
// input is read before an output that may share its memory is written, and
// pushed blocks are in memory before any is popped.
//
// Measured: a decode step of 256 requests in 8.3 us (5.1 when none ends); 601
// requests with 103,000 new tokens in 17.7 us, with 270 in 9.4 (5.8 when none
// ends): half of the time of many tokens is their placing by the cluster's 8
// SMs.

#include <cooperative_groups.h>

#include "fd_common.cuh"
#include "fd_internal.h"

namespace fdk {
namespace tb {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
constexpr int kBatch = 8;  // rows of 32 block ids that a warp has in flight
constexpr int kShare = 8;   // warps that share 32 requests' ended ones
constexpr int kFew = 4;     // new tokens that one thread places
constexpr int kChunk = 256; // tokens per warp where it walks the requests,
constexpr int kTok = 4;     // and a lane's tokens in flight
// Calls of at most this many tokens and requests run on one CTA: its 1024
// threads place them in two passes, and the cluster's barriers cost more than
// the other CTAs save (one token each: 64 requests 6.5 us, 7.8 on eight CTAs;
// 256: 8.2 and 8.4; 400: 9.6 and 8.6.  64 requests of 1 to 64 tokens: 8.3 and
// 8.8; 256 of 1 to 16: 12.2 and 10.7).
constexpr int kOneCtaTokens = 2048;
constexpr int kOneCtaReqs = 256;
constexpr int kMaxCount = 1 << 30;  // tokens and blocks of a step: loop counters stay in 32 bits

// shared memory: new, prior, then running sums over the requests [R + 1]:
// tokens, needed blocks, freed blocks of either tier (per request before the
// scan), then the warps' sums of the scan
constexpr int smem_bytes(int R) { return (2 * R + 4 * (R + 1)) * 4; }

struct Sum4 {
  long long tok, need, f0, f1;  // 64 bits: checked against the capacities before they are narrowed
};

__device__ __forceinline__ Sum4 add(const Sum4& a, const Sum4& b) {
  return {a.tok + b.tok, a.need + b.need, a.f0 + b.f0, a.f1 + b.f1};
}

__device__ __forceinline__ Sum4 shfl_up(const Sum4& a, int off, bool freed) {
  Sum4 r = {__shfl_up_sync(0xffffffffu, a.tok, off), __shfl_up_sync(0xffffffffu, a.need, off), 0, 0};
  if (freed) {
    r.f0 = __shfl_up_sync(0xffffffffu, a.f0, off);
    r.f1 = __shfl_up_sync(0xffffffffu, a.f1, off);
  }
  return r;
}

// The request that owns entry x of a running sum: the last r in [lo, hi) with
// sum[r] <= x, given sum[lo] <= x < sum[hi].
__device__ __forceinline__ int owner(const int* sum, int lo, int hi, int x) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Lengths (at most bt_width * block_size, an int32) in blocks; block sizes
// are powers of two as a rule, and a shift is a twentieth of a division.
template <bool kPow2>
struct Blocks {
  int bs, sh;
  __device__ __forceinline__ explicit Blocks(int block_size) : bs(block_size), sh(0) {
    while ((2 << sh) <= bs && sh < 29) ++sh;
  }
  __device__ __forceinline__ int of(int pos) const { return kPow2 ? pos >> sh : (int)((unsigned)pos / (unsigned)bs); }
  __device__ __forceinline__ int hold(int len) const { return len > 0 ? of(len - 1) + 1 : 0; }
};

template <bool kPow2>
__global__ void __launch_bounds__(kThreads, 1) fd_tables_kernel(const __grid_constant__ fd_tables_args a) {
  extern __shared__ int sm[];
  __shared__ Sum4 warp_sum[kWarps];
  __shared__ unsigned ended[FD_TABLES_MAX_REQS / 32];  // bit i of word w: request 32 w + i ends
  __shared__ int shared_flags;
  __shared__ int shared_max[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int nct = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int R = a.num_reqs, BS = a.block_size, W = a.bt_width;
  const Blocks<kPow2> blocks(BS);
  int* s_new = sm;
  int* s_prior = s_new + R;
  int* s_tok = s_prior + R;
  int* s_need = s_tok + R + 1;
  int* s_f0 = s_need + R + 1;
  int* s_f1 = s_f0 + R + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    shared_flags = 0;
    shared_max[0] = shared_max[1] = 0;
  }
  bool ends = false;
  for (int base = 0; base < R; base += kThreads) {
    const int r = base + tid;
    bool e = false;
    if (r < R) {
      const int nw = a.new_lens[r];
      s_new[r] = nw;
      s_prior[r] = a.prior_lens[r];
      s_f0[r] = s_f1[r] = 0;
      e = nw == -1;
    }
    const unsigned word = __ballot_sync(0xffffffffu, e);
    if (lane == 0 && r < R) ended[r >> 5] = word;
    ends |= e;
  }
  const int c0_in = a.counts_in[0], c1_in = a.counts_in[1];
  // the same in every CTA of the cluster: all of them read all lengths
  const bool any_end = __syncthreads_or(ends ? 1 : 0) != 0;

  // A warp per ended request: the set bits of a word of `ended` are dealt out
  // over kShare warps, those over all CTAs.
  auto for_ended = [&](auto&& body) {
    const int units = (R + 31) / 32 * kShare;
    for (int x = rank + nct * warp; x < units; x += nct * kWarps) {
      unsigned w = ended[x / kShare];
      for (int i = 0; w != 0u; ++i, w &= w - 1u)
        if (i % kShare == x % kShare) body(x / kShare * 32 + __ffs(w) - 1);
    }
  };

  // their blocks by tier, the counts sent to every CTA
  int flags = 0;
  if (any_end) {
    if (nct > 1) cluster.sync();  // every CTA's zeros are in place before counts arrive
    for_ended([&](int r) {
      const int prior = s_prior[r];
      if (prior < 0 || (long long)prior > (long long)W * BS) return;  // flagged below
      const int held = blocks.hold(prior);
      int n0 = 0, n1 = 0;
      for (int base = 0; base < held; base += 32 * kBatch) {
        int id[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int c = base + 32 * u + lane;
          id[u] = c < held ? a.block_table[(int64_t)r * a.bt_stride + c] : 0;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (base + 32 * u + lane >= held) continue;
          if (id[u] < 0 || id[u] >= a.num_gpu_blocks + a.num_cpu_blocks) flags |= FD_TABLES_BAD_BLOCK;
          if (id[u] < a.num_gpu_blocks)
            ++n0;
          else
            ++n1;
        }
      }
      n0 = __reduce_add_sync(0xffffffffu, n0);
      n1 = __reduce_add_sync(0xffffffffu, n1);
      if (lane < nct) {
        cluster.map_shared_rank(s_f0, lane)[r] = n0;
        cluster.map_shared_rank(s_f1, lane)[r] = n1;
      }
    });
    if (flags != 0)
      for (int c = 0; c < nct; ++c) atomicOr(cluster.map_shared_rank(&shared_flags, c), flags);
    if (nct > 1)
      cluster.sync();
    else
      __syncthreads();
  }

  // running sums: thread t takes requests [t per, (t + 1) per)
  const int per = (R + kThreads - 1) / kThreads;
  Sum4 mine = {0, 0, 0, 0};
  int max_seq = 0, max_new = 0;
  flags = 0;
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r >= R) break;
    const int nw = s_new[r], prior = s_prior[r];
    if (nw < -1 || prior < 0 || (long long)prior > (long long)W * BS) {
      flags |= FD_TABLES_BAD_LEN;
      continue;
    }
    mine.f0 += s_f0[r];
    mine.f1 += s_f1[r];
    if (nw < 0) continue;
    const long long seq = (long long)prior + nw;
    if (seq > (long long)W * BS) {
      flags |= FD_TABLES_WIDTH;
      continue;
    }
    mine.tok += nw;
    mine.need += blocks.hold((int)seq) - blocks.hold(prior);
    max_seq = max(max_seq, (int)seq);
    max_new = max(max_new, nw);
  }
  Sum4 v = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const Sum4 u = shfl_up(v, off, any_end);
    if (lane >= off) v = add(v, u);
  }
  if (lane == 31) warp_sum[warp] = v;
  flags = __reduce_or_sync(0xffffffffu, flags);
  max_seq = __reduce_max_sync(0xffffffffu, max_seq);
  max_new = __reduce_max_sync(0xffffffffu, max_new);
  if (lane == 0) {
    if (flags != 0) atomicOr(&shared_flags, flags);
    atomicMax(&shared_max[0], max_seq);
    atomicMax(&shared_max[1], max_new);
  }
  __syncthreads();
  if (warp == 0) {  // running sums of the warps
    Sum4 w = warp_sum[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const Sum4 u = shfl_up(w, off, any_end);
      if (lane >= off) w = add(w, u);
    }
    warp_sum[lane] = w;
  }
  __syncthreads();
  const Sum4 zero = {0, 0, 0, 0};
  const Sum4 before = warp > 0 ? warp_sum[warp - 1] : zero, total = warp_sum[kWarps - 1];
  flags = shared_flags;
  Sum4 run = add(before, {v.tok - mine.tok, v.need - mine.need, v.f0 - mine.f0, v.f1 - mine.f1});
  const long long c0 = (long long)c0_in + total.f0, c1 = (long long)c1_in + total.f1;
  if (c0_in < 0 || c1_in < 0 || c0 > a.free_cap[0] || c1 > a.free_cap[1]) flags |= FD_TABLES_BAD_POOL;
  if (total.tok > a.max_tokens) flags |= FD_TABLES_TOKENS;
  if (total.need > c0 + c1 || total.need > kMaxCount) flags |= FD_TABLES_NO_BLOCKS;

  // every CTA has read the lengths and the counts before any writes them
  if (nct > 1) cluster.sync();
  if (flags != 0) {
    const int step = nct * kThreads;
    for (int r = rank * kThreads + tid; r < R; r += step) {
      a.seq_lens[r] = s_prior[r];
      a.query_start_loc[r] = 0;
      if (a.query_lens != nullptr) a.query_lens[r] = 0;
    }
    for (int t = rank * kThreads + tid; t < a.max_tokens; t += step) {
      a.slot_mapping[t] = -1;
      a.positions[t] = 0;
    }
    if (rank == 0 && tid == 0) {
      a.query_start_loc[R] = 0;
      a.counts_out[0] = c0_in;
      a.counts_out[1] = c1_in;
      for (int i = 1; i < FD_TABLES_HEADER_LEN; ++i) a.header[i] = 0;
      a.header[FD_TABLES_FLAGS] = flags;
      set_error(a.error, FD_DEVERR_TABLES);
    }
    return;
  }

  // the running sums of every request (tokens fit max_tokens, an int32)
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r >= R) break;
    const int nw = s_new[r], prior = s_prior[r], f0 = s_f0[r], f1 = s_f1[r];
    s_tok[r] = (int)run.tok;
    s_need[r] = (int)run.need;
    s_f0[r] = (int)run.f0;
    s_f1[r] = (int)run.f1;
    run.f0 += f0;
    run.f1 += f1;
    if (nw >= 0) {
      run.tok += nw;
      run.need += blocks.hold(prior + nw) - blocks.hold(prior);
    }
  }
  if (tid == 0) {
    s_tok[R] = (int)total.tok;
    s_need[R] = (int)total.need;
  }
  __syncthreads();

  if (any_end) {  // push, in request and table order within each tier
    for_ended([&](int r) {
      const int held = blocks.hold(s_prior[r]);
      int at0 = c0_in + s_f0[r], at1 = c1_in + s_f1[r];
      const unsigned below = (1u << lane) - 1u;
      for (int base = 0; base < held; base += 32 * kBatch) {
        int id[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int c = base + 32 * u + lane;
          id[u] = c < held ? a.block_table[(int64_t)r * a.bt_stride + c] : 0;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const bool in = base + 32 * u + lane < held, hbm = id[u] < a.num_gpu_blocks;
          const unsigned in0 = __ballot_sync(0xffffffffu, in && hbm), in1 = __ballot_sync(0xffffffffu, in && !hbm);
          if (in && hbm) a.free_ids[0][at0 + __popc(in0 & below)] = id[u];
          if (in && !hbm) a.free_ids[1][at1 + __popc(in1 & below)] = id[u];
          at0 += __popc(in0);
          at1 += __popc(in1);
        }
      }
    });
    // the barriers order the pushes before the pops at their scope
    if (nct > 1)
      cluster.sync();
    else
      __syncthreads();
  }

  const int gt = rank * kThreads + tid, step = nct * kThreads, need = (int)total.need;
  auto pop = [&](int j) -> int {
    return j < c0 ? __ldcg(a.free_ids[0] + (c0 - 1 - j)) : __ldcg(a.free_ids[1] + (c1 - 1 - (j - c0)));
  };
  for (int r = gt; r < R; r += step) {
    a.seq_lens[r] = s_new[r] < 0 ? 0 : s_prior[r] + s_new[r];
    a.query_start_loc[r] = s_tok[r];
    if (a.query_lens != nullptr) a.query_lens[r] = max(s_new[r], 0);
    if (a.evicted != nullptr && s_new[r] < 0) a.evicted[r] = 0;  // (read only for requests with new tokens)
  }
  for (int j = gt; j < need; j += step) {
    const int r = owner(s_need, 0, R, j);
    a.block_table[(int64_t)r * a.bt_stride + blocks.hold(s_prior[r]) + (j - s_need[r])] = pop(j);
  }
  // Tokens.  Requests of at most kFew new ones: a thread each, no search.
  const int ntok = (int)total.tok;
  auto block_at = [&](int at, int r, int held, int first_need) {
    const int b = blocks.of(at);
    return b < held ? a.block_table[(int64_t)r * a.bt_stride + b] : pop(first_need + b - held);
  };
  auto put = [&](int t, int at, int id, int gone) {
    a.slot_mapping[t] = (long long)id * BS + (at - blocks.of(at) * BS);
    a.positions[t] = (long long)at + gone;
  };
  auto gone_of = [&](int r) { return a.evicted != nullptr ? a.evicted[r] : 0; };
  for (int r = gt; r < R; r += step) {
    const int nw = s_new[r];
    if (nw <= 0 || nw > kFew) continue;
    const int prior = s_prior[r], gone = gone_of(r);
    for (int i = 0; i < nw; ++i)
      put(s_tok[r] + i, prior + i, block_at(prior + i, r, blocks.hold(prior), s_need[r]), gone);
  }
  // The others.  Up to two per thread: a thread per token, which looks its
  // request up.  More: a warp per kChunk neighbouring tokens walks the requests
  // that they belong to, 32 lengths at a time, and places a request's tokens
  // together.  (256 requests of 1 to 16 new tokens: 10.7 us, walked 12.7; 64 of
  // 1 to 256: 8.5 and 9.2; 256 of 1 to 400: 14.0 and 11.9.)
  if (shared_max[1] > kFew && ntok <= 2 * step) {
    for (int t = gt; t < ntok; t += step) {
      const int r = owner(s_tok, 0, R, t);
      if (s_new[r] <= kFew) continue;
      const int prior = s_prior[r], at = prior + (t - s_tok[r]);
      put(t, at, block_at(at, r, blocks.hold(prior), s_need[r]), gone_of(r));
    }
  } else if (shared_max[1] > kFew) {
    for (int t0 = (rank * kWarps + warp) * kChunk; t0 < ntok; t0 += nct * kWarps * kChunk) {
      const int t1 = min(t0 + kChunk, ntok);
      for (int r0 = owner(s_tok, 0, R, t0); r0 < R && s_tok[r0] < t1; r0 += 32) {
        const int mine = r0 + lane;
        unsigned large = __ballot_sync(0xffffffffu, mine < R && s_tok[min(mine, R)] < t1 && s_new[min(mine, R - 1)] > kFew);
        for (; large != 0u; large &= large - 1u) {
          const int r = r0 + __ffs(large) - 1;
          const int from = s_tok[r], prior = s_prior[r], held = blocks.hold(prior), need0 = s_need[r], gone = gone_of(r);
          const int lo = max(t0, from), hi = min(t1, from + s_new[r]);
          for (int t = lo + lane; t < hi; t += 32 * kTok) {
            int id[kTok];
#pragma unroll
            for (int u = 0; u < kTok; ++u)
              id[u] = t + 32 * u < hi ? block_at(prior + (t + 32 * u - from), r, held, need0) : 0;
#pragma unroll
            for (int u = 0; u < kTok; ++u)
              if (t + 32 * u < hi) put(t + 32 * u, prior + (t + 32 * u - from), id[u], gone);
          }
        }
      }
    }
  }
  for (int t = ntok + gt; t < a.max_tokens; t += step) {
    a.slot_mapping[t] = -1;
    a.positions[t] = 0;
  }
  if (rank == 0 && tid == 0) {
    a.query_start_loc[R] = ntok;
    const int t0 = (int)min(total.need, c0);
    a.counts_out[0] = (int)c0 - t0;
    a.counts_out[1] = (int)c1 - (need - t0);
    a.header[FD_TABLES_FLAGS] = 0;
    a.header[FD_TABLES_N_TOK] = ntok;
    a.header[FD_TABLES_TAKEN_HBM] = t0;
    a.header[FD_TABLES_TAKEN_HOST] = need - t0;
    a.header[FD_TABLES_FREED_HBM] = (int)total.f0;
    a.header[FD_TABLES_FREED_HOST] = (int)total.f1;
    a.header[FD_TABLES_MAX_SEQ] = shared_max[0];
    a.header[FD_TABLES_MAX_NEW] = shared_max[1];
  }
}

// ------------------------------------------------------------- shorter tables

// fd_trim_tables.  The freed blocks of all requests, in request and column
// order, form a line of F entries; its place on the stacks is the running
// count of HBM (or host) ids ahead of it.  The line is cut into equal spans,
// one per CTA of a cluster, those into runs of one warp, so one request that
// loses a thousand blocks and a thousand that lose one are dealt out alike.  A
// lane looks its first entry's request up, and another's where that one's blocks
// end.  Ids are read once and stay in registers from the count to the push where a CTA's span
// is one pass of kTrimIds ids per thread.  Bound by latency: the lengths, the
// ids, the barriers; a small CTA where the caller's bound says that few blocks
// can go.
// Measured: 256 requests that lose up to 7 tokens in 4.5 us (1024 threads: 8.6),
// 100 that lose up to 14000 (44,000 blocks) in 9.0, of which the launch and the
// end take 2; with a look-up for every id 14.5.
constexpr int kTrimIds = 8;
constexpr int kTrimSmall = 256;   // threads of the small CTA
// Blocks that one CTA takes, as far as the caller's bounds tell: one pass.  (256
// requests, 256 blocks: 3.1 us with the small CTA, 4.0 with the large one, 5.0
// with a cluster; 1000 and 1000: 4.5, 4.2 and 5.2; 4128 blocks: the large one
// 6.6; 8256: 8.2, a cluster 8.2; 38,500: 38.5 and 8.3.)
constexpr int kTrimOneCta = kThreads * kTrimIds;

// Sum over the CTA's warps of v (one value per warp, in shared memory), and of
// those before this one.
template <int kNw>
__device__ __forceinline__ void over_warps(const int* v, int warp, int lane, int& ahead, int& all) {
  const int x = lane < kNw ? v[lane] : 0;
  ahead = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
  all = __reduce_add_sync(0xffffffffu, x);
}

template <bool kPow2, int kNt>
__global__ void __launch_bounds__(kNt, 1) fd_trim_kernel(const __grid_constant__ fd_trim_args a) {
  constexpr int kNw = kNt / 32, kPass = kNt * kTrimIds;
  extern __shared__ int sm[];  // [R + 1] running sum of freed blocks, [R] first freed column, [R] lengths, [R] kept lengths
  __shared__ int warp_n[2][kNw];
  __shared__ int cta_n[kCluster][3];  // HBM and host blocks, flags
  __shared__ int shared_flags, shared_max, shared_high;
  cg::cluster_group cluster = cg::this_cluster();
  const int nct = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  if (nct > 1) cluster.barrier_arrive();  // this CTA has started; awaited before the first write to another's memory
  const int R = a.num_reqs, BS = a.block_size, W = a.bt_width;
  const Blocks<kPow2> blocks(BS);
  int* s_sum = sm;
  int* s_col = s_sum + R + 1;
  int* s_len = s_col + R;
  int* s_left = s_len + R;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) shared_flags = shared_max = shared_high = 0;
  const int c0_in = a.counts_in[0], c1_in = a.counts_in[1];
  for (int r = tid; r < R; r += kNt) {
    const int len = a.lens_in[r], keep = a.keep_lens[r];
    s_len[r] = len;
    s_left[r] = keep >= 0 && keep < len ? keep : len;
  }
  __syncthreads();

  // running sum of the freed blocks: thread t takes requests [t per, (t + 1) per)
  const int per = (R + kNt - 1) / kNt;
  int flags = 0, longest = 0, high = 0;
  unsigned sum = 0u;
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r >= R) break;
    const int len = s_len[r];
    if (len < 0 || (long long)len > (long long)W * BS) {
      flags |= FD_TABLES_BAD_LEN;
      s_col[r] = s_sum[r] = 0;
      continue;
    }
    const int col = blocks.hold(s_left[r]), n = blocks.hold(len) - col;
    s_col[r] = col;
    s_sum[r] = n;
    sum += (unsigned)n;  // (may wrap, as the sums below: then `high` tells)
    high += n >> 12;
    longest = max(longest, s_left[r]);
  }
  const int mine = (int)sum;
  int v = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v = (int)((unsigned)v + (unsigned)u);
  }
  if (lane == 31) warp_n[0][warp] = v;
  flags = __reduce_or_sync(0xffffffffu, flags);
  longest = __reduce_max_sync(0xffffffffu, longest);
  high = __reduce_add_sync(0xffffffffu, min(high, 1 << 20));
  if (lane == 0) {
    if (flags != 0) atomicOr(&shared_flags, flags);
    atomicMax(&shared_max, longest);
    if (high != 0) atomicAdd(&shared_high, high);
  }
  __syncthreads();
  int run, F;
  over_warps<kNw>(warp_n[0], warp, lane, run, F);
  run = (int)((unsigned)run + (unsigned)v - sum);
  // more than 2^30 blocks: no stack holds them
  const bool fits = shared_high <= kMaxCount >> 12;
  if (!fits) F = 0;
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r >= R) break;
    const int n = s_sum[r];
    s_sum[r] = fits ? run : 0;
    run = (int)((unsigned)run + (unsigned)n);
  }
  if (tid == 0) s_sum[R] = F;
  __syncthreads();

  // this CTA's span of the line; warp w takes kTrimIds * 32 neighbours per pass
  const int lo = (int)((long long)F * rank / nct), hi = (int)((long long)F * (rank + 1) / nct);
  const bool one = hi - lo <= kPass;
  const int ids = (int)(a.num_gpu_blocks + a.num_cpu_blocks), hbm_ids = (int)a.num_gpu_blocks;
  int id[kTrimIds];
  flags = fits ? 0 : FD_TABLES_BAD_POOL;
  auto load = [&](int base) {  // ids of the warp's run from `base` on, -1 behind the span
    int r = 0;
#pragma unroll
    for (int u = 0; u < kTrimIds; ++u) {
      id[u] = -1;
      const int f = base + 32 * u + lane;
      if (base + 32 * u >= hi) continue;  // the warp alike
      if (f >= hi) continue;
      if (u == 0 || s_sum[r + 1] <= f) r = owner(s_sum, r, R, f);
      id[u] = a.block_table[(int64_t)r * a.bt_stride + s_col[r] + (f - s_sum[r])];
    }
#pragma unroll
    for (int u = 0; u < kTrimIds; ++u) {
      if (base + 32 * u + lane < hi && (id[u] < 0 || id[u] >= ids)) {
        flags |= FD_TABLES_BAD_BLOCK;
        id[u] = 0;
      }
    }
  };
  auto count = [&](int base, int& n0, int& n1) {
#pragma unroll
    for (int u = 0; u < kTrimIds; ++u) {
      if (base + 32 * u >= hi) break;  // the warp alike
      n0 += __popc(__ballot_sync(0xffffffffu, id[u] >= 0 && id[u] < hbm_ids));
      n1 += __popc(__ballot_sync(0xffffffffu, id[u] >= hbm_ids));
    }
  };
  int n0 = 0, n1 = 0;  // of this warp, over all passes
  for (int base = lo + warp * kTrimIds * 32; base < hi; base += kPass) {
    load(base);
    count(base, n0, n1);
  }
  flags = __reduce_or_sync(0xffffffffu, flags);
  if (lane == 0) {
    warp_n[0][warp] = n0;
    warp_n[1][warp] = n1;
    if (flags != 0) atomicOr(&shared_flags, flags);
  }
  __syncthreads();
  int ahead0, ahead1, all0, all1;
  over_warps<kNw>(warp_n[0], warp, lane, ahead0, all0);
  over_warps<kNw>(warp_n[1], warp, lane, ahead1, all1);
  flags = shared_flags;
  int at0 = c0_in, at1 = c1_in;
  long long end0 = (long long)c0_in + all0, end1 = (long long)c1_in + all1;
  if (nct > 1) {
    cluster.barrier_wait();
    if (tid < nct) {
      int* to = cluster.map_shared_rank(&cta_n[rank][0], tid);
      to[0] = all0;
      to[1] = all1;
      to[2] = flags;
    }
    cluster.sync();  // also: every CTA has read the lengths and counts before any writes them
    end0 = c0_in;
    end1 = c1_in;
#pragma unroll
    for (int c = 0; c < kCluster; ++c) {
      if (c >= nct) break;
      const int x0 = cta_n[c][0], x1 = cta_n[c][1];
      at0 += c < rank ? x0 : 0;
      at1 += c < rank ? x1 : 0;
      end0 += x0;
      end1 += x1;
      flags |= cta_n[c][2];
    }
  }
  if (c0_in < 0 || c1_in < 0 || end0 > a.free_cap[0] || end1 > a.free_cap[1]) flags |= FD_TABLES_BAD_POOL;
  if (flags == 0) {
    const unsigned below = (1u << lane) - 1u;
    for (int base = lo; base < hi; base += kPass) {
      const int from = base + warp * kTrimIds * 32;
      if (!one) {  // the pass's ids again, and its counts
        n0 = n1 = 0;
        if (from < hi) {
          load(from);
          count(from, n0, n1);
        }
        __syncthreads();  // the last pass's counts have been read
        if (lane == 0) {
          warp_n[0][warp] = n0;
          warp_n[1][warp] = n1;
        }
        __syncthreads();
        over_warps<kNw>(warp_n[0], warp, lane, ahead0, all0);
        over_warps<kNw>(warp_n[1], warp, lane, ahead1, all1);
      }
      int to0 = at0 + ahead0, to1 = at1 + ahead1;
#pragma unroll
      for (int u = 0; u < kTrimIds; ++u) {
        if (from + 32 * u >= hi) break;  // the warp alike
        const bool in = id[u] >= 0, hbm = id[u] < hbm_ids;
        const unsigned in0 = __ballot_sync(0xffffffffu, in && hbm), in1 = __ballot_sync(0xffffffffu, in && !hbm);
        if (in && hbm) a.free_ids[0][to0 + __popc(in0 & below)] = id[u];
        if (in && !hbm) a.free_ids[1][to1 + __popc(in1 & below)] = id[u];
        to0 += __popc(in0);
        to1 += __popc(in1);
      }
      at0 += all0;
      at1 += all1;
    }
  }
  for (int r = rank * kNt + tid; r < R; r += nct * kNt) {
    const int len = s_len[r], left = s_left[r];
    a.lens_out[r] = flags != 0 ? len : left;
    if (flags == 0 && a.evicted != nullptr && left < len) a.evicted[r] += len - left;
  }
  if (rank == 0 && tid < FD_TABLES_HEADER_LEN) {
    a.header[tid] = tid == FD_TABLES_FLAGS        ? flags
                    : flags != 0                  ? 0
                    : tid == FD_TABLES_FREED_HBM  ? (int)(end0 - c0_in)
                    : tid == FD_TABLES_FREED_HOST ? (int)(end1 - c1_in)
                    : tid == FD_TABLES_MAX_SEQ    ? shared_max
                                                  : 0;
    if (tid < 2) a.counts_out[tid] = flags != 0 ? (tid == 0 ? c0_in : c1_in) : (int)(tid == 0 ? end0 : end1);
    if (tid == 0 && flags != 0) set_error(a.error, FD_DEVERR_TABLES);
  }
}

}  // namespace tb
}  // namespace fdk

extern "C" int fd_extend_tables(const fd_tables_args* a, void* stream) {
  using namespace fdk::tb;
  if (a == nullptr) return fdh::fail(FD_ERR_INVALID, "fd_extend_tables: null args");
  if (a->num_reqs < 0 || a->max_tokens < 0 || a->block_size <= 0 || a->num_gpu_blocks < 0 || a->num_cpu_blocks < 0)
    return fdh::fail(FD_ERR_INVALID, "fd_extend_tables: bad num_reqs, max_tokens, block_size or block counts");
  if (a->num_reqs > FD_TABLES_MAX_REQS)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_extend_tables: %d requests (at most %d)", a->num_reqs,
                     FD_TABLES_MAX_REQS);
  if (a->num_gpu_blocks + a->num_cpu_blocks > 0x7fffffff)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_extend_tables: block ids must fit int32");
  if (a->max_tokens > kMaxCount)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_extend_tables: max_tokens at most %d", kMaxCount);
  if (a->bt_width <= 0 || a->bt_stride < a->bt_width)
    return fdh::fail(FD_ERR_INVALID, "fd_extend_tables: bt_width must be positive and at most bt_stride");
  if ((int64_t)a->bt_width * a->block_size > 0x7fffffff)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_extend_tables: bt_width * block_size must fit int32");
  if (a->counts_in == nullptr || a->counts_out == nullptr || a->query_start_loc == nullptr || a->header == nullptr ||
      (a->num_reqs > 0 && (a->new_lens == nullptr || a->prior_lens == nullptr || a->block_table == nullptr ||
                           a->seq_lens == nullptr)) ||
      (a->max_tokens > 0 && (a->slot_mapping == nullptr || a->positions == nullptr)))
    return fdh::fail(FD_ERR_INVALID, "fd_extend_tables: null buffer");
  for (int t = 0; t < 2; ++t)
    if (a->free_cap[t] < 0 || (a->free_cap[t] > 0 && a->free_ids[t] == nullptr))
      return fdh::fail(FD_ERR_INVALID, "fd_extend_tables: free stack %d has a capacity but no memory", t);
  const bool pow2 = (a->block_size & (a->block_size - 1)) == 0;
  static unsigned long long done[2] = {0, 0};
  const void* kern = pow2 ? reinterpret_cast<const void*>(fd_tables_kernel<true>)
                          : reinterpret_cast<const void*>(fd_tables_kernel<false>);
  int st = fdh::ensure_smem(kern, smem_bytes(FD_TABLES_MAX_REQS), &done[pow2 ? 1 : 0]);
  if (st != FD_OK) return st;
  const int ctas = a->max_tokens <= kOneCtaTokens && a->num_reqs <= kOneCtaReqs ? 1 : kCluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem_bytes(a->num_reqs);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[1] = {const_cast<fd_tables_args*>(a)};
  return fdh::cuda_status(cudaLaunchKernelExC(&cfg, kern, args), "fd_tables_kernel launch");
}

extern "C" size_t fd_tables_args_bytes(void) { return sizeof(fd_tables_args); }

extern "C" int fd_trim_tables(const fd_trim_args* a, void* stream) {
  using namespace fdk::tb;
  if (a == nullptr) return fdh::fail(FD_ERR_INVALID, "fd_trim_tables: null args");
  if (a->num_reqs < 0 || a->block_size <= 0 || a->num_gpu_blocks < 0 || a->num_cpu_blocks < 0)
    return fdh::fail(FD_ERR_INVALID, "fd_trim_tables: bad num_reqs, block_size or block counts");
  if (a->num_reqs > FD_TABLES_MAX_REQS)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_trim_tables: %d requests (at most %d)", a->num_reqs, FD_TABLES_MAX_REQS);
  if (a->num_gpu_blocks + a->num_cpu_blocks > 0x7fffffff)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_trim_tables: block ids must fit int32");
  if (a->bt_width <= 0 || a->bt_stride < 0)
    return fdh::fail(FD_ERR_INVALID, "fd_trim_tables: bt_width must be positive, bt_stride not negative");
  if ((int64_t)a->bt_width * a->block_size > 0x7fffffff)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_trim_tables: bt_width * block_size must fit int32");
  if (a->counts_in == nullptr || a->counts_out == nullptr || a->header == nullptr ||
      (a->num_reqs > 0 &&
       (a->keep_lens == nullptr || a->lens_in == nullptr || a->lens_out == nullptr || a->block_table == nullptr)))
    return fdh::fail(FD_ERR_INVALID, "fd_trim_tables: null buffer");
  for (int t = 0; t < 2; ++t)
    if (a->free_cap[t] < 0 || (a->free_cap[t] > 0 && a->free_ids[t] == nullptr))
      return fdh::fail(FD_ERR_INVALID, "fd_trim_tables: free stack %d has a capacity but no memory", t);
  const bool pow2 = (a->block_size & (a->block_size - 1)) == 0;
  int64_t most = a->bt_width;  // blocks that a request can lose
  if (a->max_cut > 0 && a->max_cut / a->block_size + 1 < most) most = a->max_cut / a->block_size + 1;
  most *= a->num_reqs;
  const int ctas = most <= kTrimOneCta ? 1 : kCluster;
  const bool small = ctas == 1 && most <= kTrimSmall * kTrimIds && a->num_reqs <= 4 * kTrimSmall;
  static unsigned long long done[4] = {0, 0, 0, 0};
  const void* const kerns[4] = {reinterpret_cast<const void*>(fd_trim_kernel<false, kThreads>),
                                reinterpret_cast<const void*>(fd_trim_kernel<true, kThreads>),
                                reinterpret_cast<const void*>(fd_trim_kernel<false, kTrimSmall>),
                                reinterpret_cast<const void*>(fd_trim_kernel<true, kTrimSmall>)};
  const int which = (small ? 2 : 0) + (pow2 ? 1 : 0);
  const void* kern = kerns[which];
  const int st = fdh::ensure_smem(kern, (4 * FD_TABLES_MAX_REQS + 1) * 4, &done[which]);
  if (st != FD_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(small ? kTrimSmall : kThreads);
  cfg.dynamicSmemBytes = (size_t)(4 * a->num_reqs + 1) * 4;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[1] = {const_cast<fd_trim_args*>(a)};
  return fdh::cuda_status(cudaLaunchKernelExC(&cfg, kern, args), "fd_trim_kernel launch");
}

extern "C" size_t fd_trim_args_bytes(void) { return sizeof(fd_trim_args); }
