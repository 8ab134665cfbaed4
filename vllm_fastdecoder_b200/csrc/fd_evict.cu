// A cache cut to a budget: which keys stay (fd_select_keys) and their move to
// the front of their request's blocks (fd_move_keys).
//
// Select.  A key's place in the order that the choice wants is one 64-bit
// number: its weight as an ordered 32-bit number (guarded keys above all, a NaN
// below all), then its index, the lowest first.  No two are equal, so the
// keep-th greatest, T, splits the keys without a rule for ties.  It is found by
// narrowing: the window from the least to the greatest is cut into 512 equal
// bins, the bin that holds T becomes the window, until few enough candidates
// are left to rank each against all.  (Weights are spread over exponents and
// order like their bits, so the bins are filled evenly: two rounds, seldom
// three.)  Then one running count in index order, of the places that become
// free and of the keys that move, gives each pair its place, so src and dst
// ascend and no result depends on timing.  The keys are read once, into shared
// memory, by one CTA, or by a cluster that adds its counters up through
// distributed shared memory where one CTA would be slow.
// Bound by the latency of that chain (lengths, table, weights, then the
// exchanges), not by its 8 bytes per key.
// Measured: 32 requests x 8 heads of 2050 keys in 16.4 us, 4 x 8 of 11,000 to
// 32,000 in 24.6.
//
// Move.  Only what lies behind the budget moves, into what goes before it, so
// no pair reads what another writes, and the pairs are dealt out over the GPU
// in any order.  A CTA takes kPairs pairs of one request and head at a time:
// their rows' places first, then all 16-byte pieces of K and V, several per
// thread in flight.  Bound by the bytes of the rows, read and written once.
// Measured: 32 requests x 8 heads of up to 32 pairs of 512 bytes in 9.4 us, 4 x
// 8 of 1500 in 16.4.

#include <cooperative_groups.h>

#include "fd_common.cuh"
#include "fd_internal.h"

namespace fdk {
namespace ev {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxKeys = 40 * 1024;  // keys of a CTA in shared memory; more are read again in every round
constexpr int kCtaKeys = 4096;       // keys of a CTA from which on more CTAs are taken
constexpr int kBinBits = 9, kBins = 1 << kBinBits;
static_assert(kBins == kThreads, "a bin per thread");
constexpr int kCand = 128;           // candidates that are ranked one by one
constexpr unsigned kGuarded = 0xffffffffu;

struct SelectParams {
  fd_select_args a;
  int cap;  // keys that fit the CTA's shared memory
};

// Weights in order as unsigned numbers: -0 equals 0, a NaN is below all.
__device__ __forceinline__ unsigned ordered(float w) {
  if (w != w) return 0u;
  const unsigned u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kThreads, 2) fd_select_kernel(const __grid_constant__ SelectParams sp) {
  const fd_select_args& a = sp.a;
  typedef unsigned long long u64;
  extern __shared__ unsigned s_keys[];
  __shared__ int hist[2][kBins];
  __shared__ u64 cand[kCand];
  __shared__ unsigned ends[kMaxCluster][3];   // least key, greatest key, a bad block, of every CTA
  __shared__ int cta_n[2][kMaxCluster];       // free places, moving keys of every CTA
  __shared__ unsigned warp_u[3][kWarps];
  __shared__ int warp_n[2][kWarps];
  __shared__ int found[3];                    // the round's bin, the keys above it, the keys in it
  __shared__ int taken;
  __shared__ u64 s_T;
  cg::cluster_group cluster = cg::this_cluster();
  const int nct = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int unit = blockIdx.x / nct, KVH = a.num_kv_heads, r = unit / KVH, h = unit - r * KVH;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (nct > 1) cluster.barrier_arrive();  // this CTA has started; awaited before the first write to another's memory
  const int n = a.lens[r], keep = a.keep_lens[r], BS = a.block_size;
  auto sync = [&]() {
    if (nct > 1)
      cluster.sync();
    else
      __syncthreads();
  };

  // the whole cluster alike
  const bool cut = keep >= 0 && keep < n;
  bool ok = true;
  if (n < 0 || (long long)n > (long long)a.bt_width * BS || (cut && min(keep, n - keep) > a.room)) {
    if (rank == 0 && tid == 0) set_error(a.error, FD_DEVERR_LEN);
    ok = false;
  }
  if (!ok || !cut || keep == 0) {
    if (rank == 0 && tid == 0) a.counts[unit] = 0;
    if (nct > 1) cluster.barrier_wait();
    return;
  }
  const int per = ((n + nct - 1) / nct + 31) / 32 * 32;  // keys of a CTA
  const int lo = min(n, rank * per), hi = min(n, lo + per);
  const long long newest = (long long)n + (a.evicted != nullptr ? a.evicted[r] : 0) - a.recent;
  const int32_t* table = a.block_table + (int64_t)r * a.bt_stride;
  auto load = [&](int j, unsigned& bad) -> unsigned {
    const int page = (int)((unsigned)j / (unsigned)BS);
    const int64_t id = table[page];
    if (id < 0 || id >= a.stats.num_blocks) {
      bad = 1u;
      return 0u;
    }
    const int64_t at = (id * KVH + h) * BS + (j - page * BS);
    const float w = a.stats.weights[at];
    const int pos = a.stats.positions[at];
    return pos < a.sinks || pos >= newest ? kGuarded : ordered(w);
  };
  const bool kept = per <= sp.cap;
  unsigned least = 0xffffffffu, most = 0u, bad = 0u;
#pragma unroll 4
  for (int j = lo + tid; j < hi; j += kThreads) {
    const unsigned k = load(j, bad);
    if (kept) s_keys[j - lo] = k;
    least = min(least, k);
    most = max(most, k);
  }
  auto key = [&](int j) {
    unsigned ignored;
    return kept ? s_keys[j - lo] : load(j, ignored);
  };
  auto place = [&](int j) { return (u64)key(j) << 32 | (0xffffffffu - (unsigned)j); };
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  bad = __reduce_or_sync(0xffffffffu, bad);
  if (lane == 0) {
    warp_u[0][warp] = least;
    warp_u[1][warp] = most;
    warp_u[2][warp] = bad;
  }
  for (int i = tid; i < 2 * kBins; i += kThreads) hist[i / kBins][i % kBins] = 0;
  if (tid == 0) taken = 0;
  __syncthreads();
  if (nct > 1) cluster.barrier_wait();
  if (warp == 0) {
    const int w = lane % kWarps;
    least = __reduce_min_sync(0xffffffffu, warp_u[0][w]);
    most = __reduce_max_sync(0xffffffffu, warp_u[1][w]);
    bad = __reduce_or_sync(0xffffffffu, warp_u[2][w]);
    if (lane < nct) {
      unsigned* to = cluster.map_shared_rank(&ends[rank][0], lane);
      to[0] = least;
      to[1] = most;
      to[2] = bad;
    }
  }
  sync();
  least = 0xffffffffu;
  most = bad = 0u;
  for (int c = 0; c < nct; ++c) {
    least = min(least, ends[c][0]);
    most = max(most, ends[c][1]);
    bad |= ends[c][2];
  }
  if (bad != 0u) {  // all threads of the cluster alike
    if (rank == 0 && tid == 0) {
      a.counts[unit] = 0;
      set_error(a.error, FD_DEVERR_BLOCK_ID);
    }
    return;
  }

  // the window [base, base + 2^bits) holds the want-th greatest of its keys
  u64 base = (u64)least << 32, T;
  int bits = 64 - __clzll((u64)(most - least) << 32 | 0xffffffffu), want = keep;
#pragma unroll 1
  for (int round = 0;; ++round) {
    int* const mine = hist[round & 1];
    const int sh = max(0, bits - kBinBits);
    for (int j = lo + tid; j < hi; j += kThreads) {
      const u64 x = place(j) - base;  // wraps below the window
      if (bits == 64 || x >> bits == 0) atomicAdd(&mine[x >> sh], 1);
    }
    sync();
    // bins from the greatest down, a thread each: those above, and the window's next
    const int bin = kBins - 1 - tid;
    int c = 0;
    for (int x = 0; x < nct; ++x) c += cluster.map_shared_rank(mine, x)[bin];
    int above = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, above, off);
      if (lane >= off) above += o;
    }
    if (lane == 31) warp_n[0][warp] = above;
    hist[(round + 1) & 1][bin] = 0;  // the last round's: every CTA has read it
    __syncthreads();
    above -= c;
    for (int w = 0; w < warp; ++w) above += warp_n[0][w];
    if (above < want && want <= above + c) {  // one thread
      found[0] = bin;
      found[1] = above;
      found[2] = c;
    }
    __syncthreads();
    const int at = found[0], m = found[2];
    base += (u64)at << sh;
    bits = sh;
    want -= found[1];
    if (want == m || bits == 0) {  // all of the window's (of one key alone, it)
      T = base;
      break;
    }
    if (m > kCand) continue;
    // few: every CTA gets them all, and ranks them by itself
    if (tid == 0) {
      int ahead = 0;
      for (int x = 0; x < rank; ++x) ahead += cluster.map_shared_rank(mine, x)[at];
      taken = ahead;
    }
    __syncthreads();
    for (int j = lo + tid; j < hi; j += kThreads) {
      const u64 p = place(j);
      if ((p - base) >> bits != 0) continue;
      const int slot = atomicAdd(&taken, 1);
      for (int x = 0; x < nct; ++x) cluster.map_shared_rank(cand, x)[slot] = p;
    }
    sync();
    if (tid < m) {
      const u64 p = cand[tid];
      int greater = 0;
#pragma unroll 8
      for (int i = 0; i < m; ++i) greater += cand[i] > p;
      if (greater == want - 1) s_T = p;
    }
    __syncthreads();
    T = s_T;
    break;
  }

  // Places that become free, and keys that move there, in index order: a warp
  // has a run of neighbours.
  const int wper = ((hi - lo + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int from = min(hi, lo + warp * wper), to = min(hi, from + wper);
  const unsigned below = (1u << lane) - 1u;
  int n0 = 0, n1 = 0;
  for (int b = from; b < to; b += 32) {
    const int j = b + lane;
    const bool stay = j < to && place(j) >= T;
    n0 += __popc(__ballot_sync(0xffffffffu, j < to && j < keep && !stay));
    n1 += __popc(__ballot_sync(0xffffffffu, j >= keep && stay));
  }
  if (lane == 0) {
    warp_n[0][warp] = n0;
    warp_n[1][warp] = n1;
  }
  __syncthreads();
  int all0 = 0, all1 = 0;
  n0 = n1 = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      n0 += warp_n[0][w];
      n1 += warp_n[1][w];
    }
    all0 += warp_n[0][w];
    all1 += warp_n[1][w];
  }
  if (tid < nct) {
    cluster.map_shared_rank(&cta_n[0][0], tid)[rank] = all0;
    cluster.map_shared_rank(&cta_n[1][0], tid)[rank] = all1;
  }
  sync();
  all0 = 0;
  for (int c = 0; c < nct; ++c) {
    if (c < rank) {
      n0 += cta_n[0][c];
      n1 += cta_n[1][c];
    }
    all0 += cta_n[0][c];
  }
  int32_t* const dst = a.dst + (int64_t)unit * a.room;
  int32_t* const src = a.src + (int64_t)unit * a.room;
  for (int b = from; b < to; b += 32) {
    const int j = b + lane;
    const bool stay = j < to && place(j) >= T;
    const bool hole = j < to && j < keep && !stay, mover = j >= keep && stay;
    const unsigned m0 = __ballot_sync(0xffffffffu, hole), m1 = __ballot_sync(0xffffffffu, mover);
    if (hole) dst[n0 + __popc(m0 & below)] = j;
    if (mover) src[n1 + __popc(m1 & below)] = j;
    n0 += __popc(m0);
    n1 += __popc(m1);
  }
  if (rank == 0 && tid == 0) a.counts[unit] = all0;
}

// ------------------------------------------------------------------ move

constexpr int kMoveThreads = 256;
constexpr int kPairs = 32;   // pairs of a CTA at a time
constexpr int kInFlight = 4; // 16-byte pieces per thread

struct MoveParams {
  const int32_t* src;
  const int32_t* dst;
  const int32_t* counts;
  unsigned char* k[2];
  unsigned char* v[2];
  int64_t blk_sb[2], head_sb[2], tok_sb[2], nblk[2];  // bytes
  int64_t split;
  const int32_t* bt;
  int64_t bt_stride;
  fd_key_stats stats;
  int W, KVH, BS, room, vec;  // vec: 16-byte pieces of a row of K
  int32_t* err;
};

struct Place {
  unsigned char* k;  // null: the pair is passed over
  unsigned char* v;
  int64_t stat;
};

__device__ __forceinline__ Place place_of(const MoveParams& p, int r, int h, int j) {
  Place x = {nullptr, nullptr, 0};
  if (j < 0 || (long long)j >= (long long)p.W * p.BS) {
    set_error(p.err, FD_DEVERR_LEN);
    return x;
  }
  const int page = (int)((unsigned)j / (unsigned)p.BS), off = j - page * p.BS;
  const int64_t id = p.bt[(int64_t)r * p.bt_stride + page];
  const int t = id >= p.split ? 1 : 0;
  const int64_t b = id - (t ? p.split : 0);
  if (b < 0 || b >= p.nblk[t] || (p.stats.weights != nullptr && id >= p.stats.num_blocks)) {
    set_error(p.err, FD_DEVERR_BLOCK_ID);
    return x;
  }
  const int64_t at = b * p.blk_sb[t] + h * p.head_sb[t] + off * p.tok_sb[t];
  x.k = p.k[t] + at;
  x.v = p.v[t] + at;
  x.stat = (id * p.KVH + h) * p.BS + off;
  return x;
}

__global__ void __launch_bounds__(kMoveThreads) fd_move_kernel(const __grid_constant__ MoveParams p) {
  __shared__ Place from[kPairs], to[kPairs];
  const int unit = blockIdx.x, r = unit / p.KVH, h = unit - r * p.KVH, tid = threadIdx.x;
  int n = p.counts[unit];
  if (n < 0 || n > p.room) {
    if (tid == 0) set_error(p.err, FD_DEVERR_LEN);
    n = 0;
  }
  for (int i0 = blockIdx.y * kPairs; i0 < n; i0 += gridDim.y * kPairs) {
    const int m = min(kPairs, n - i0);
    __syncthreads();  // the last round's places have been read
    if (tid < 2 * kPairs) {
      const int i = tid & (kPairs - 1);
      if (i < m) {
        const int j = (tid < kPairs ? p.src : p.dst)[(int64_t)unit * p.room + i0 + i];
        (tid < kPairs ? from : to)[i] = place_of(p, r, h, j);
      }
    }
    __syncthreads();
    if (tid < m && p.stats.weights != nullptr && from[tid].k != nullptr && to[tid].k != nullptr) {
      p.stats.weights[to[tid].stat] = p.stats.weights[from[tid].stat];
      p.stats.positions[to[tid].stat] = p.stats.positions[from[tid].stat];
    }
    const int total = m * 2 * p.vec;
    for (int x0 = tid; x0 < total; x0 += kMoveThreads * kInFlight) {
      uint4 v[kInFlight];
      unsigned char* out[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int x = x0 + u * kMoveThreads;
        out[u] = nullptr;
        if (x >= total) continue;
        const int row = x / p.vec, c = (x - row * p.vec) * 16, i = row >> 1;
        if (from[i].k == nullptr || to[i].k == nullptr) continue;
        v[u] = *reinterpret_cast<const uint4*>(((row & 1) ? from[i].v : from[i].k) + c);
        out[u] = ((row & 1) ? to[i].v : to[i].k) + c;
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
        if (out[u] != nullptr) *reinterpret_cast<uint4*>(out[u]) = v[u];
    }
  }
}

}  // namespace ev
}  // namespace fdk

extern "C" int fd_select_keys(const fd_select_args* a, void* stream) {
  using namespace fdk::ev;
  if (a == nullptr) return fdh::fail(FD_ERR_INVALID, "fd_select_keys: null args");
  if (a->num_reqs < 0 || a->num_kv_heads <= 0 || a->block_size <= 0 || a->room < 0 || a->stats.num_blocks < 0 ||
      a->sinks < 0 || a->recent < 0)
    return fdh::fail(FD_ERR_INVALID, "fd_select_keys: bad num_reqs, num_kv_heads, block_size, room, num_blocks, sinks or recent");
  if (a->num_reqs > 65535 || a->num_kv_heads > 4096)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_select_keys: %d requests (at most 65535) of %d kv heads (at most 4096)", a->num_reqs,
                     a->num_kv_heads);
  if (a->num_reqs == 0) return FD_OK;
  if (a->bt_width <= 0 || a->bt_stride < 0)
    return fdh::fail(FD_ERR_INVALID, "fd_select_keys: bt_width must be positive, bt_stride not negative");
  const int64_t most = (int64_t)a->bt_width * a->block_size;
  if (most > 0x7fffffff - 512)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_select_keys: bt_width * block_size must fit int32");
  if (a->block_table == nullptr || a->lens == nullptr || a->keep_lens == nullptr || a->counts == nullptr ||
      (a->stats.num_blocks > 0 && (a->stats.weights == nullptr || a->stats.positions == nullptr)) ||
      (a->room > 0 && (a->src == nullptr || a->dst == nullptr)))
    return fdh::fail(FD_ERR_INVALID, "fd_select_keys: null buffer");
  const int64_t len = a->max_len > 0 && a->max_len < most ? a->max_len : most;
  const int64_t units = (int64_t)a->num_reqs * a->num_kv_heads;
  int ctas = 1;
  while (ctas < kMaxCluster && units * ctas < 296 && len > (int64_t)ctas * kCtaKeys) ctas *= 2;
  SelectParams sp;
  sp.a = *a;
  const int64_t per = ((len + ctas - 1) / ctas + 31) / 32 * 32;
  sp.cap = (int)(per < kMaxKeys ? per : kMaxKeys);
  static unsigned long long done = 0;
  const void* kern = reinterpret_cast<const void*>(fd_select_kernel);
  const int st = fdh::ensure_smem(kern, kMaxKeys * 4, &done);
  if (st != FD_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)sp.cap * 4;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[1] = {&sp};
  return fdh::cuda_status(cudaLaunchKernelExC(&cfg, kern, args), "fd_select_kernel launch");
}

extern "C" size_t fd_select_args_bytes(void) { return sizeof(fd_select_args); }

extern "C" int fd_move_keys(const fd_move_args* a, void* stream) {
  using namespace fdk::ev;
  if (a == nullptr) return fdh::fail(FD_ERR_INVALID, "fd_move_keys: null args");
  const int es = fdh::elem_size(a->dtype);
  if (es == 0) return fdh::fail(FD_ERR_UNSUPPORTED, "fd_move_keys: unsupported dtype %d", a->dtype);
  if (a->num_reqs < 0 || a->num_kv_heads <= 0 || a->head_size <= 0 || a->block_size <= 0 || a->room < 0 ||
      a->stats.num_blocks < 0)
    return fdh::fail(FD_ERR_INVALID, "fd_move_keys: bad num_reqs, num_kv_heads, head_size, block_size, room or num_blocks");
  if (a->num_reqs > 65535 || a->num_kv_heads > 4096 || a->head_size > 65536)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_move_keys: %d requests (at most 65535), %d kv heads (4096), head size %d (65536)",
                     a->num_reqs, a->num_kv_heads, a->head_size);
  if ((int64_t)a->head_size * es % 16 != 0)
    return fdh::fail(FD_ERR_ALIGN, "fd_move_keys: head_size*elem_size must be a multiple of 16");
  if (a->num_reqs == 0 || a->room == 0) return FD_OK;
  if (a->bt_width <= 0 || a->bt_stride < 0)
    return fdh::fail(FD_ERR_INVALID, "fd_move_keys: bt_width must be positive, bt_stride not negative");
  if (a->src == nullptr || a->dst == nullptr || a->counts == nullptr || a->block_table == nullptr ||
      (a->stats.weights != nullptr && a->stats.positions == nullptr))
    return fdh::fail(FD_ERR_INVALID, "fd_move_keys: null buffer");
  MoveParams p{};
  for (int t = 0; t < 2; ++t) {
    const fd_kv_tier& tr = a->tier[t];
    p.nblk[t] = tr.num_blocks > 0 ? tr.num_blocks : 0;
    if (p.nblk[t] == 0) continue;
    if (tr.k == nullptr || tr.v == nullptr)
      return fdh::fail(FD_ERR_INVALID, "fd_move_keys: tier %d has blocks but no K/V pointer", t);
    if (!fdh::aligned16(tr.k) || !fdh::aligned16(tr.v) || (tr.blk_stride * es) % 16 != 0 ||
        (tr.head_stride * es) % 16 != 0 || (tr.tok_stride * es) % 16 != 0)
      return fdh::fail(FD_ERR_ALIGN, "fd_move_keys: tier %d pointers/strides must be 16-byte aligned", t);
    p.k[t] = static_cast<unsigned char*>(const_cast<void*>(static_cast<const void*>(tr.k)));
    p.v[t] = static_cast<unsigned char*>(const_cast<void*>(static_cast<const void*>(tr.v)));
    p.blk_sb[t] = tr.blk_stride * es;
    p.head_sb[t] = tr.head_stride * es;
    p.tok_sb[t] = tr.tok_stride * es;
  }
  p.src = a->src;
  p.dst = a->dst;
  p.counts = a->counts;
  p.split = a->tier_split;
  p.bt = a->block_table;
  p.bt_stride = a->bt_stride;
  p.stats = a->stats;
  p.W = a->bt_width;
  p.KVH = a->num_kv_heads;
  p.BS = a->block_size;
  p.room = a->room;
  p.vec = a->head_size * es / 16;
  p.err = a->error;
  // CTAs per request and head: as many as its pairs could fill, but no more
  // than fill the GPU eight times over (most of a large room stays unused)
  const int64_t units = (int64_t)a->num_reqs * a->num_kv_heads;
  int64_t y = (a->room + kPairs - 1) / kPairs;
  const int64_t few = (148 * 8 * 8 + units - 1) / units;
  if (y > few) y = few;
  fd_move_kernel<<<dim3((unsigned)units, (unsigned)y), kMoveThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return fdh::cuda_status(cudaGetLastError(), "fd_move_kernel launch");
}

extern "C" size_t fd_move_args_bytes(void) { return sizeof(fd_move_args); }
