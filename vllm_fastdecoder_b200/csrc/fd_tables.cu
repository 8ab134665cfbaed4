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

#include <cooperative_groups.h>

#include "fd_common.cuh"
#include "fd_internal.h"

namespace fdk {
namespace tb {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
// Calls of at most this many tokens and requests run on one CTA: its 1024
// threads place them in two passes, and the cluster's barriers cost more than
// the other CTAs save.
constexpr int kOneCtaTokens = 2048;
constexpr int kOneCtaReqs = 1024;
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

__device__ __forceinline__ Sum4 shfl_up(const Sum4& a, int off) {
  return {__shfl_up_sync(0xffffffffu, a.tok, off), __shfl_up_sync(0xffffffffu, a.need, off),
          __shfl_up_sync(0xffffffffu, a.f0, off), __shfl_up_sync(0xffffffffu, a.f1, off)};
}

// The request that owns entry x of a running sum: the last r with sum[r] <= x
// (sum[R] > x).
__device__ __forceinline__ int owner(const int* sum, int R, int x) {
  int lo = 0, hi = R;  // sum[lo] <= x < sum[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int ceil_div(long long a, int b) { return (int)((a + b - 1) / b); }

__global__ void __launch_bounds__(kThreads, 1) fd_tables_kernel(const __grid_constant__ fd_tables_args a) {
  extern __shared__ int sm[];
  __shared__ Sum4 warp_sum[kWarps];
  __shared__ int shared_flags;
  __shared__ int shared_max[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int nct = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int R = a.num_reqs, BS = a.block_size, W = a.bt_width;
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
  for (int r = tid; r < R; r += kThreads) {
    s_new[r] = a.new_lens[r];
    s_prior[r] = a.prior_lens[r];
    s_f0[r] = s_f1[r] = 0;
    ends |= s_new[r] == -1;
  }
  const int c0_in = a.counts_in[0], c1_in = a.counts_in[1];
  // the same in every CTA of the cluster: all of them read all lengths
  const bool any_end = __syncthreads_or(ends ? 1 : 0) != 0;

  // blocks of ended requests by tier: one warp per request, requests dealt
  // out over the CTAs, the counts sent to all of them
  int flags = 0;
  if (any_end) {
    if (nct > 1) cluster.sync();  // every CTA's zeros are in place before counts arrive
    for (int r = rank + nct * warp; r < R; r += nct * kWarps) {
      if (s_new[r] != -1) continue;
      const int prior = s_prior[r];
      if (prior < 0 || (long long)prior > (long long)W * BS) continue;  // flagged below
      const int held = ceil_div(prior, BS);
      int n0 = 0, n1 = 0;
      for (int c = lane; c < held; c += 32) {
        const long long id = a.block_table[(int64_t)r * a.bt_stride + c];
        if (id < 0 || id >= a.num_gpu_blocks + a.num_cpu_blocks) flags |= FD_TABLES_BAD_BLOCK;
        if (id < a.num_gpu_blocks)
          ++n0;
        else
          ++n1;
      }
      n0 = __reduce_add_sync(0xffffffffu, n0);
      n1 = __reduce_add_sync(0xffffffffu, n1);
      if (lane < nct) {
        cluster.map_shared_rank(s_f0, lane)[r] = n0;
        cluster.map_shared_rank(s_f1, lane)[r] = n1;
      }
    }
    if (flags != 0 && lane < 32)
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
    mine.need += ceil_div(seq, BS) - ceil_div(prior, BS);
    max_seq = max(max_seq, (int)seq);
    max_new = max(max_new, nw);
  }
  Sum4 v = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const Sum4 u = shfl_up(v, off);
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
  Sum4 before = {0, 0, 0, 0}, total = {0, 0, 0, 0};
#pragma unroll 4
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = total;
    total = add(total, warp_sum[w]);
  }
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
      run.need += ceil_div((long long)prior + nw, BS) - ceil_div(prior, BS);
    }
  }
  if (tid == 0) {
    s_tok[R] = (int)total.tok;
    s_need[R] = (int)total.need;
  }
  __syncthreads();

  if (any_end) {  // push, in request and table order within each tier
    for (int r = rank + nct * warp; r < R; r += nct * kWarps) {
      if (s_new[r] != -1) continue;
      const int held = ceil_div(s_prior[r], BS);
      int at0 = c0_in + s_f0[r], at1 = c1_in + s_f1[r];
      for (int base = 0; base < held; base += 32) {
        const int c = base + lane;
        const int id = c < held ? a.block_table[(int64_t)r * a.bt_stride + c] : 0;
        const bool hbm = id < a.num_gpu_blocks;
        const unsigned in0 = __ballot_sync(0xffffffffu, c < held && hbm);
        const unsigned in1 = __ballot_sync(0xffffffffu, c < held && !hbm);
        const unsigned below = (1u << lane) - 1u;
        if (c < held) {
          if (hbm)
            a.free_ids[0][at0 + __popc(in0 & below)] = id;
          else
            a.free_ids[1][at1 + __popc(in1 & below)] = id;
        }
        at0 += __popc(in0);
        at1 += __popc(in1);
      }
    }
    __threadfence();
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
  }
  for (int j = gt; j < need; j += step) {
    const int r = owner(s_need, R, j);
    a.block_table[(int64_t)r * a.bt_stride + ceil_div(s_prior[r], BS) + (j - s_need[r])] = pop(j);
  }
  int r = 0;
  const int ntok = (int)total.tok;
  for (int t = gt; t < a.max_tokens; t += step) {
    long long slot = -1, pos = 0;
    if (t < ntok) {
      if (t >= s_tok[r + 1] || t < s_tok[r]) r = owner(s_tok, R, t);
      const int prior = s_prior[r];
      const int at = prior + (t - s_tok[r]);
      const int held = ceil_div(prior, BS), b = at / BS;
      const int id = b < held ? a.block_table[(int64_t)r * a.bt_stride + b] : pop(s_need[r] + b - held);
      slot = (long long)id * BS + (at - b * BS);
      pos = at;
    }
    a.slot_mapping[t] = slot;
    a.positions[t] = pos;
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
  static unsigned long long done = 0;
  const void* kern = reinterpret_cast<const void*>(fd_tables_kernel);
  int st = fdh::ensure_smem(kern, smem_bytes(FD_TABLES_MAX_REQS), &done);
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
