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
  auto put = [&](int t, int at, int id) {
    a.slot_mapping[t] = (long long)id * BS + (at - blocks.of(at) * BS);
    a.positions[t] = at;
  };
  for (int r = gt; r < R; r += step) {
    const int nw = s_new[r];
    if (nw <= 0 || nw > kFew) continue;
    const int prior = s_prior[r];
    for (int i = 0; i < nw; ++i)
      put(s_tok[r] + i, prior + i, block_at(prior + i, r, blocks.hold(prior), s_need[r]));
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
      put(t, at, block_at(at, r, blocks.hold(prior), s_need[r]));
    }
  } else if (shared_max[1] > kFew) {
    for (int t0 = (rank * kWarps + warp) * kChunk; t0 < ntok; t0 += nct * kWarps * kChunk) {
      const int t1 = min(t0 + kChunk, ntok);
      for (int r0 = owner(s_tok, 0, R, t0); r0 < R && s_tok[r0] < t1; r0 += 32) {
        const int mine = r0 + lane;
        unsigned large = __ballot_sync(0xffffffffu, mine < R && s_tok[min(mine, R)] < t1 && s_new[min(mine, R - 1)] > kFew);
        for (; large != 0u; large &= large - 1u) {
          const int r = r0 + __ffs(large) - 1;
          const int from = s_tok[r], prior = s_prior[r], held = blocks.hold(prior), need0 = s_need[r];
          const int lo = max(t0, from), hi = min(t1, from + s_new[r]);
          for (int t = lo + lane; t < hi; t += 32 * kTok) {
            int id[kTok];
#pragma unroll
            for (int u = 0; u < kTok; ++u)
              id[u] = t + 32 * u < hi ? block_at(prior + (t + 32 * u - from), r, held, need0) : 0;
#pragma unroll
            for (int u = 0; u < kTok; ++u)
              if (t + 32 * u < hi) put(t + 32 * u, prior + (t + 32 * u - from), id[u]);
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
