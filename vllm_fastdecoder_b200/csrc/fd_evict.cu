// A cache cut to a budget: which keys stay (fd_select_keys) and their move to
// the front of their request's blocks (fd_move_keys).
//
// Select.  A key's place in the order that the choice wants is one 64-bit
// number: its weight as an ordered 32-bit number (guarded keys above all, a NaN
// below all), then its index, the lowest first.  No two are equal, so the
// keep-th greatest, T, splits the keys without a rule for ties.  It is found by
// narrowing: a window, at first of all 64-bit numbers, is cut into 512 equal
// bins, and the bin that holds T becomes the window, until few enough candidates
// are left to rank each against all.  The first round tells exponents apart, each
// other one nine more bits.  A CTA by itself ranks after the first as a rule; a
// cluster, where ranking costs two rounds, goes on until the window holds no more
// keys than are wanted of it (two or three rounds), and ranks only among equal
// weights.  Then one running count in index order, of the places that become free
// and of the keys that move, gives each pair its place, so src and dst ascend and
// no result depends on timing.  The keys are read once and stay in registers (in
// shared memory where a CTA has more than 4096), in one CTA, or in a cluster that
// adds its counters up through distributed shared memory.
// Bound by the latency of that chain (lengths, table, weights, then the
// exchanges), not by its 8 bytes per key.
// Measured: 32 requests x 8 heads of up to 2080 keys in 8.9 us, 13.3 where the
// border falls among a hundred keys that tie; 4 x 8 of 11,000 to 32,000 in 16.2 on
// clusters of 8 (four or five cluster barriers: the start, two or three rounds, the
// counts), of which a round with its exchange takes 1.6 to 2.4.
//
// Move.  Only what lies behind the budget moves, into what goes before it, so
// no pair reads what another writes, and the pairs are dealt out over the GPU
// in any order.  A CTA takes kPairs pairs of one request and head at a time:
// their rows' places first, then all 16-byte pieces of K and V, several per
// thread in flight.  The rows' bytes are its floor; what bounds it is latency, of
// one wave of CTAs that go through count, pair and table before any row moves
// (a warp's cycles are half waits for loads, DRAM is busy a quarter of the time).
// Measured: 32 requests x 8 heads of up to 32 pairs of 512 bytes in 3.9 us, 4 x
// 8 of 1400 in 13.2 (48.8 MB, read and written in pieces of 512 bytes, at 3.7
// TB/s); with half of their blocks in the host tier 25 and 366, the link's time.
// With 16, 32 and 128 pairs per CTA: 18.4, 14.2 and 13.7; with 2 and 8
// pieces per thread 13.2 and 15.0; a warp by itself with eight pairs 15.0.

#include <cooperative_groups.h>

#include "fd_common.cuh"
#include "fd_internal.h"

namespace fdk {
namespace ev {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kPer = 8;                   // keys of a thread:
constexpr int kTile = kThreads * kPer;    // a CTA of one tile keeps them in registers
constexpr int kMaxKeys = 40 * 1024;       // keys of a CTA of several tiles in shared memory; more are read again in every pass
constexpr int kBinBits = 9, kBins = 1 << kBinBits;
static_assert(kBins == kThreads, "a bin per thread");
constexpr int kCand = kThreads / 4;       // candidates that are ranked one by one
constexpr unsigned kGuarded = 0xffffffffu;

struct SelectParams {
  fd_select_args a;
  int cap;  // keys that fit the CTA's shared memory (several tiles)
  int sh;   // log2 of the block size, or -1
};

// Weights in order as unsigned numbers: -0 equals 0, a NaN is below all.
__device__ __forceinline__ unsigned ordered(float w) {
  if (w != w) return 0u;
  const unsigned u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}

template <bool kMany>  // several CTAs per request and head
__global__ void __launch_bounds__(kThreads, 2) fd_select_kernel(const __grid_constant__ SelectParams sp) {
  const fd_select_args& a = sp.a;
  typedef unsigned long long u64;
  extern __shared__ unsigned s_keys[];
  __shared__ int hist[kBins];                 // of the CTA's own keys
  // Of the cluster's: a CTA adds its bins that are not empty to every CTA's copy
  // (few; reading all of every other's took 5000 cycles a round).  Three take
  // turns: the next round's is clean before any CTA can write to it.
  __shared__ int whole[kMany ? 3 : 1][kMany ? kBins : 1];
  __shared__ u64 cand[kMany ? kMaxCluster : 1][kCand];  // of every CTA,
  __shared__ int cand_n[kMaxCluster];                   // and how many
  __shared__ int cta_n[kMaxCluster][2];       // free places, moving keys of every CTA
  __shared__ int warp_n[2][kWarps];
  __shared__ __align__(16) int counts[kPer * kWarps];  // of 32 keys each, in index order: free places, moving keys << 16
  __shared__ int found[3];                    // the round's bin, the keys above it, the keys in it
  __shared__ int taken, any_bad;
  __shared__ u64 s_T;
  cg::cluster_group cluster = cg::this_cluster();
  const int nct = kMany ? (int)cluster.num_blocks() : 1, rank = kMany ? (int)cluster.block_rank() : 0;
  const int unit = blockIdx.x / nct, KVH = a.num_kv_heads, r = unit / KVH, h = unit - r * KVH;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = a.lens[r], keep = a.keep_lens[r], BS = a.block_size;
  auto sync = [&]() {
    if constexpr (kMany)
      cluster.sync();
    else
      __syncthreads();
  };
  auto at_rank = [&](auto* p, int c) {  // CTA c's copy of a shared variable
    if constexpr (kMany)
      return cluster.map_shared_rank(p, c);
    else
      return p;
  };

  // the whole cluster alike
  const bool cut = keep >= 0 && keep < n;
  bool ok = true;
  if (n < 0 || (long long)n > (long long)a.bt_width * BS || (cut && min(keep, n - keep) > a.room)) {
    if (rank == 0 && tid == 0) set_error(a.error, FD_DEVERR_LEN);
    ok = false;
  }
  if (ok && cut && a.stats.num_blocks == 0) {
    if (rank == 0 && tid == 0) set_error(a.error, FD_DEVERR_BLOCK_ID);
    ok = false;
  }
  if (!ok || !cut || keep == 0) {
    if (rank == 0 && tid == 0) a.counts[unit] = 0;
    return;
  }
  const int span = ((n + nct - 1) / nct + 31) / 32 * 32;  // keys of a CTA
  const int lo = min(n, rank * span), hi = min(n, lo + span);
  // positions from here on are guarded (its bounds are int32's)
  const int newest = (int)min(max((long long)n + (a.evicted != nullptr ? a.evicted[r] : 0) - a.recent, -0x80000000ll), 0x7fffffffll);
  const int32_t* table = a.block_table + (int64_t)r * a.bt_stride;
  const unsigned nblk = (unsigned)(a.stats.num_blocks < 0x7fffffff ? a.stats.num_blocks : 0x7fffffff);
  const int line = KVH * BS, row0 = h * BS;
  unsigned bad = 0u;
  // The thread's keys of the tile from t0 on: t0 + u kThreads + tid.
  unsigned k[kPer];
  auto load = [&](int t0) {
    // a level at a time: all its loads are under way before the first is used
    int id[kPer], off[kPer], pos[kPer];
    float w[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if (t0 + u * kThreads >= hi) break;  // the CTA alike
      const int j = t0 + u * kThreads + tid;
      const int page = sp.sh >= 0 ? j >> sp.sh : (int)((unsigned)j / (unsigned)BS);
      off[u] = row0 + j - page * BS;
      id[u] = j < hi ? table[page] : 0;
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if (t0 + u * kThreads >= hi) break;
      const bool in = t0 + u * kThreads + tid < hi, have = (unsigned)id[u] < nblk;
      const int64_t at = in && have ? (int64_t)id[u] * line + off[u] : 0;
      w[u] = a.stats.weights[at];
      pos[u] = a.stats.positions[at];
      bad |= in && !have ? 1u : 0u;
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if (t0 + u * kThreads >= hi) break;
      k[u] = pos[u] < a.sinks || pos[u] >= newest ? kGuarded : ordered(w[u]);
    }
  };
  const bool one = hi - lo <= kTile, kept = hi - lo <= sp.cap;
  auto fetch = [&](int t0) {  // again, for a pass over several tiles
    if (one) return;
    if (!kept) return load(t0);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int j = t0 + u * kThreads + tid;
      if (j < hi) k[u] = s_keys[j - lo];
    }
  };
  // body(key, j) for the CTA's keys
  auto each = [&](int t0, auto&& body) {
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if (t0 + u * kThreads >= hi) break;
      const int j = t0 + u * kThreads + tid;
      if (j < hi) body(k[u], j);
    }
  };
  if (tid == 0) taken = any_bad = 0;
  hist[tid] = 0;
  if constexpr (kMany) {
    whole[0][tid] = whole[1][tid] = whole[2][tid] = 0;
    cluster.barrier_arrive();  // awaited before the first write to another CTA's counters: they are clean by then
  }
  __syncthreads();
  for (int t0 = lo; t0 < hi; t0 += kTile) {
    load(t0);
    each(t0, [&](unsigned x, int j) {
      if (!one && kept) s_keys[j - lo] = x;
      atomicAdd(&hist[x >> (32 - kBinBits)], 1);  // the first round's bins
    });
  }
  if constexpr (kMany) cluster.barrier_wait();
  if (bad != 0u)
    for (int c = 0; c < nct; ++c) *at_rank(&any_bad, c) = 1;

  auto place = [](unsigned x, int j) { return (u64)x << 32 | (0xffffffffu - (unsigned)j); };
  // the window [base, base + 2^bits) holds the want-th greatest of its places
  u64 base = 0ull, T;
  int bits = 64, want = keep;
#pragma unroll 1
  for (int round = 0;; ++round) {
    const int sh = max(0, bits - kBinBits);
    if (round > 0) {  // (its own counters have been read: two barriers ago)
      hist[tid] = 0;
      __syncthreads();
      for (int t0 = lo; t0 < hi; t0 += kTile) {
        fetch(t0);
        each(t0, [&](unsigned x, int j) {
          const u64 y = place(x, j) - base;  // wraps below the window
          if (y >> bits == 0) atomicAdd(&hist[y >> sh], 1);
        });
      }
    }
    __syncthreads();
    // bins from the greatest down, a thread each: the keys above them, and theirs
    const int bin = kBins - 1 - tid;
    int c = hist[bin];
    if constexpr (kMany) {
      if (c > 0)
        for (int x = 0; x < nct; ++x) atomicAdd(cluster.map_shared_rank(&whole[round % 3][bin], x), c);
      cluster.sync();
      c = whole[round % 3][bin];
      whole[(round + 2) % 3][bin] = 0;
    }
    if (round == 0 && any_bad != 0) {  // all threads of the cluster alike
      if (rank == 0 && tid == 0) {
        a.counts[unit] = 0;
        set_error(a.error, FD_DEVERR_BLOCK_ID);
      }
      return;
    }
    int above = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, above, off);
      if (lane >= off) above += o;
    }
    if (lane == 31) warp_n[0][warp] = above;
    __syncthreads();
    above += __reduce_add_sync(0xffffffffu, lane < warp ? warp_n[0][lane] : 0) - c;
    if (above < want && want <= above + c) {  // one thread
      found[0] = bin;
      found[1] = above;
      found[2] = c;
    }
    __syncthreads();
    const int m = found[2];
    base += (u64)found[0] << sh;
    bits = sh;
    want -= found[1];
    if (want == m || bits == 0) {  // all of the window's (of one key alone, it)
      T = base;
      break;
    }
    if (m > kCand || (kMany && bits > 32)) continue;
    // few: every CTA gets them all, and ranks them by itself (in a cluster another round costs half of that, and as a
    // rule tells keys of different weights apart)
    for (int t0 = lo; t0 < hi; t0 += kTile) {
      fetch(t0);
      unsigned who[kPer];
      int mine = 0;
      const unsigned base_key = (unsigned)(base >> 32);
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        who[u] = 0u;
        if (t0 + u * kThreads >= hi) continue;  // the CTA alike
        const int j = t0 + u * kThreads + tid;
        const bool in = bits >= 32 ? (k[u] - base_key) >> (bits - 32) == 0u : (place(k[u], j) - base) >> bits == 0;
        who[u] = __ballot_sync(0xffffffffu, in && j < hi);
        mine += __popc(who[u]);
      }
      if (mine == 0) continue;
      int slot = 0;
      if (lane == 0) slot = atomicAdd(&taken, mine);
      slot = __shfl_sync(0xffffffffu, slot, 0);
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        if (who[u] == 0u) continue;
        if ((who[u] >> lane) & 1u) {
          const int to = slot + __popc(who[u] & ((1u << lane) - 1u));
          for (int x = 0; x < nct; ++x) at_rank(&cand[rank][0], x)[to] = place(k[u], t0 + u * kThreads + tid);
        }
        slot += __popc(who[u]);
      }
    }
    __syncthreads();
    if (tid < nct) *at_rank(&cand_n[rank], tid) = taken;
    sync();
    if (warp < (m + 7) / 8) {  // four threads per candidate
      int x = tid >> 2, of = 0;
      while (of < nct && x >= cand_n[of]) x -= cand_n[of++];
      const u64 y = of < nct ? cand[of][x] : ~0ull;
      int greater = 0;
      for (int q = 0; q < nct; ++q) {
        const int many = cand_n[q];
#pragma unroll 4
        for (int i = tid & 3; i < many; i += 4) greater += cand[q][i] > y ? 1 : 0;
      }
      greater += __shfl_xor_sync(0xffffffffu, greater, 1);
      greater += __shfl_xor_sync(0xffffffffu, greater, 2);
      if (of < nct && greater == want - 1) s_T = y;
    }
    __syncthreads();
    T = s_T;
    break;
  }

  // Places that become free, and keys that move there, in index order.
  const unsigned T_key = (unsigned)(T >> 32), T_j = 0xffffffffu - (unsigned)T;
  auto stays = [&](unsigned x, int j) { return x > T_key || (x == T_key && (unsigned)j <= T_j); };
  unsigned hole[kPer], mover[kPer];  // the warp's 32 keys of each
  auto look = [&](int t0) {
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      hole[u] = mover[u] = 0u;
      if (t0 + u * kThreads >= hi) continue;  // the CTA alike
      const int j = t0 + u * kThreads + tid;
      const bool in = j < hi, stay = in && stays(k[u], j);
      hole[u] = __ballot_sync(0xffffffffu, in && !stay && j < keep);
      mover[u] = __ballot_sync(0xffffffffu, stay && j >= keep);
    }
  };
  int at0 = 0, at1 = 0;  // pairs ahead of this CTA
  if constexpr (kMany) {
    int n0 = 0, n1 = 0;
    for (int t0 = lo; t0 < hi; t0 += kTile) {
      fetch(t0);
      look(t0);
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        n0 += __popc(hole[u]);
        n1 += __popc(mover[u]);
      }
    }
    if (lane == 0) {
      warp_n[0][warp] = n0;
      warp_n[1][warp] = n1;
    }
    __syncthreads();
    n0 = __reduce_add_sync(0xffffffffu, lane < kWarps ? warp_n[0][lane] : 0);
    n1 = __reduce_add_sync(0xffffffffu, lane < kWarps ? warp_n[1][lane] : 0);
    if (tid < nct) {
      int* to = cluster.map_shared_rank(&cta_n[rank][0], tid);
      to[0] = n0;
      to[1] = n1;
    }
    cluster.sync();
    int all = 0;
    for (int c = 0; c < nct; ++c) {
      if (c < rank) {
        at0 += cta_n[c][0];
        at1 += cta_n[c][1];
      }
      all += cta_n[c][0];
    }
    if (rank == 0 && tid == 0) a.counts[unit] = all;
  }
  int32_t* const dst = a.dst + (int64_t)unit * a.room;
  int32_t* const src = a.src + (int64_t)unit * a.room;
  const unsigned below = (1u << lane) - 1u;
  for (int t0 = lo; t0 < hi; t0 += kTile) {
    if (!(kMany && one)) {  // (else they are there from the count)
      fetch(t0);
      look(t0);
    }
    // a running sum over the tile's groups of 32: group 16 u + warp is this warp's u-th
    int mine = 0;
#pragma unroll
    for (int u = 0; u < kPer; ++u)
      if (lane == u) mine = __popc(hole[u]) | __popc(mover[u]) << 16;
    if (t0 > lo) __syncthreads();  // the last tile's counts have been read
    if (lane < kPer) counts[lane * kWarps + warp] = mine;
    __syncthreads();
    const int4 c = reinterpret_cast<const int4*>(counts)[lane];
    const int own = c.x + c.y + c.z + c.w;
    int incl = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    const int x = warp & 3;  // of the lane's four groups, the one that a warp with these low bits has
    const int ahead = incl - own + (x > 0 ? c.x : 0) + (x > 1 ? c.y : 0) + (x > 2 ? c.z : 0);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if ((hole[u] | mover[u]) == 0u) continue;  // the warp alike
      const int p = __shfl_sync(0xffffffffu, ahead, (u * kWarps + warp) >> 2);
      const int j = t0 + u * kThreads + tid;
      if ((hole[u] >> lane) & 1u) dst[at0 + (p & 0xffff) + __popc(hole[u] & below)] = j;
      if ((mover[u] >> lane) & 1u) src[at1 + (p >> 16) + __popc(mover[u] & below)] = j;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    at0 += total & 0xffff;
    at1 += total >> 16;
  }
  if constexpr (!kMany) {
    if (tid == 0) a.counts[unit] = at0;
  }
}

// ------------------------------------------------------------------ move

constexpr int kMoveThreads = 256;
constexpr int kPairs = 64;   // pairs of a CTA at a time
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
  int vec_sh;                 // its log2, or -1
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
        const int row = p.vec_sh >= 0 ? x >> p.vec_sh : x / p.vec, c = (x - row * p.vec) * 16, i = row >> 1;
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
  if (most > 0x7fffffff - 2 * kTile || (int64_t)a->num_kv_heads * a->block_size > 0x7fffffff)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_select_keys: bt_width * block_size and num_kv_heads * block_size must fit int32");
  if (a->block_table == nullptr || a->lens == nullptr || a->keep_lens == nullptr || a->counts == nullptr ||
      (a->stats.num_blocks > 0 && (a->stats.weights == nullptr || a->stats.positions == nullptr)) ||
      (a->room > 0 && (a->src == nullptr || a->dst == nullptr)))
    return fdh::fail(FD_ERR_INVALID, "fd_select_keys: null buffer");
  const int64_t len = a->max_len > 0 && a->max_len < most ? a->max_len : most;
  const int64_t units = (int64_t)a->num_reqs * a->num_kv_heads;
  // CTAs per request and head: enough that each has one tile, as long as they run at once (32 of 8000 keys: 12.1 us
  // on clusters of 2, one CTA with two tiles 23.9; of 32,000: 17.1 on 8, 34, 60 and 84 on 4, 2 and 1; 8 of 32,000, a
  // CTA per SM: 12.9 on 8)
  int ctas = 1;
  while (ctas < kMaxCluster && units * ctas < 296 && len > (int64_t)ctas * kTile) ctas *= 2;
  SelectParams sp;
  sp.a = *a;
  const int64_t per = ((len + ctas - 1) / ctas + 31) / 32 * 32;
  sp.cap = per <= kTile ? 0 : (int)(per < kMaxKeys ? per : kMaxKeys);
  sp.sh = -1;
  for (int sh = 0; sh < 31; ++sh)
    if (a->block_size == 1 << sh) sp.sh = sh;
  static unsigned long long done[2] = {0, 0};
  const void* kern = ctas > 1 ? reinterpret_cast<const void*>(fd_select_kernel<true>)
                              : reinterpret_cast<const void*>(fd_select_kernel<false>);
  const int st = fdh::ensure_smem(kern, kMaxKeys * 4, &done[ctas > 1 ? 1 : 0]);
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
  p.vec_sh = -1;
  for (int sh = 0; sh < 20; ++sh)
    if (p.vec == 1 << sh) p.vec_sh = sh;
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
