// Attention weight per cached key: what the CUDA-core kernel (fd_keyw.cu) and
// the tensor-core kernel (fd_keyw_mma.cu) share: parameters, the schedule, and
// how a key's weight is written.
//
//   w[j] = sum_{i, h} exp(scale q[i,h] . k[j] - lse[h, i])
//
// The products are turned over: keys are rows, queries columns, so a key's sum
// stays with one thread (or one row of threads) while the queries stream by,
// and no softmax has to be found, since lse is known.
//
// Schedule.  An ITEM is one tile of KT keys of one request and kv head; its
// work is the query tiles (CHUNKS of tq tokens times the G heads) that see any
// of them: those from token i0 = max(0, key0 - (klen - qlen)) on.  Items of all
// requests, kv heads and key tiles in that order form a line on which an item
// takes kW positions (K's load, the epilogue) and one per chunk.  The line is
// cut into equal ranges, one per CTA; an item that a range's end cuts leaves
// its keys' sums as partials, which the combine adds up in ascending order, or,
// with `snap`, belongs whole to the CTA in whose range it starts.  A call of few
// items on the CUDA cores has a grid of them instead (kDirect: key tile, kv
// head, request), whose CTAs need not look for their work.
#pragma once

#include "fd_attn.cuh"

namespace fdk {
namespace kw {

using at::AttnParams;
using at::Req;

constexpr int kMaxCtas = 320;
constexpr int kMaxKeys = 256;  // keys per item, at most

// One cut item, written by the CTA that holds its first segment.
struct Cut {
  int nparts;  // 0: none
  int r, kh, kt;
};

struct KwParams {
  AttnParams a;
  float* weights;
  int32_t* positions;
  int64_t nstat;
  const int32_t* evicted;
  Cut* cuts;     // [ctas], or null where no item is cut
  float* parts;  // [ctas][2][kMaxKeys]
};

__host__ __device__ constexpr size_t cut_bytes() { return kMaxCtas * sizeof(Cut); }
__host__ __device__ constexpr size_t workspace_bytes() { return cut_bytes() + (size_t)kMaxCtas * 2 * kMaxKeys * 4; }

// Key j of request r gets the weight w: set, with its position, where the key
// is one of the newest qlen, else added.  One addition per key and call, so an
// atomic add (which needs no read by the thread) makes nothing depend on time.
__device__ __forceinline__ void give(const KwParams& p, const Req& rq, int r, int kh, int j, int64_t id, float w) {
  const int t = id >= p.a.split ? 1 : 0;
  const int64_t b = id - (t ? p.a.split : 0);
  if (b < 0 || b >= p.a.nblk[t] || id < 0 || id >= p.nstat) {
    set_error(p.a.err, FD_DEVERR_BLOCK_ID);
    return;
  }
  const int64_t at = (id * p.a.KVH + kh) * p.a.BS + (int)((unsigned)j % (unsigned)p.a.BS);
  if (j < rq.klen - rq.qlen) {
    atomicAdd(p.weights + at, w);
  } else {
    p.weights[at] = w;
    p.positions[at] = j + (p.evicted != nullptr ? p.evicted[r] : 0);
  }
}

template <int kKT, int kW, bool kDirect>
struct Walk {
  struct Seg {
    int r, kh, kt;
    int c0;        // first chunk of the segment
    int n;         // chunks of the segment
    bool whole;
    bool head;     // holds the item's first chunk
    int nparts;    // a cut item's first segment: its parts
  };

  const AttnParams& p;
  int len, per;
  int s;           // the current item, relative to the start of this CTA's range
  int r, kh, item;
  Req rq;
  bool behind;

  __device__ __forceinline__ Walk(const AttnParams& params) : p(params) {}

  __device__ __forceinline__ static int tiles(const Req& q) { return q.qlen > 0 ? (q.klen + kKT - 1) / kKT : 0; }
  __device__ __forceinline__ static int last_chunk(const AttnParams& p, const Req& q) { return (q.qlen + p.tq - 1) / p.tq; }
  __device__ __forceinline__ static int first_chunk(const AttnParams& p, const Req& q, int kt) {
    const int i0 = kt * kKT - (q.klen - q.qlen);
    return i0 > 0 ? i0 / p.tq : 0;
  }
  // positions of key tiles 0 .. i - 1 of a request and kv head
  __device__ static long long before(const AttnParams& p, const Req& q, int i) {
    long long sum = (long long)i * (kW + last_chunk(p, q));
    const int base = q.klen - q.qlen;
    const int k0 = base > 0 ? (base + kKT - 1) / kKT : 0;  // tiles that every query sees
    if (i > k0) sum -= at::staircase((uint32_t)(i - k0), (uint32_t)p.tq, kKT, (uint32_t)(k0 * kKT - base));
    return sum;
  }
  __device__ __forceinline__ static long long cost(const AttnParams& p, const Req& q) {
    return q.qlen > 0 ? before(p, q, tiles(q)) : 0;
  }
  __device__ __forceinline__ static long long quot(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
  }

  struct Scratch {
    long long warp_sum[32];
    long long start, per_head;
    int found;
    Req rq;
  };

  // The range of CTA `c`, given the cost of all requests.  False: no work.
  __device__ __forceinline__ bool range(long long total, int c, int min_per, long long& p0) {
    if (total > (long long)at::kMaxLen * p.ctas) {  // positions of a range are 32 bits
      set_error(p.err, FD_DEVERR_LEN);
      return false;
    }
    per = (int)quot(total + p.ctas - 1, p.ctas);
    if (per < min_per) per = min_per;
    p0 = (long long)c * per;
    if (p0 >= total) return false;
    len = (int)min((long long)per, total - p0);
    return true;
  }

  // A warp together: the item of request r (cost per_head for each kv head) at
  // position off of the request's.
  __device__ __forceinline__ void find(long long off, long long per_head) {
    const int lane = threadIdx.x & 31;
    kh = (int)quot(off, per_head);
    const long long x = off - (long long)kh * per_head;
    int lo = 0, hi = tiles(rq);
    long long at_lo = 0;
    while (hi - lo > 1) {  // the last item that starts at or before x, 32 candidates at a time
      const int gap = (hi - lo + 31) / 32;
      const int i = lo + lane * gap;
      const long long v = i < hi ? before(p, rq, i) : 0;
      const unsigned in = __ballot_sync(0xffffffffu, i < hi && v <= x);
      const int last = 31 - __clz(in);  // lane 0 always: before(lo) <= x
      at_lo = __shfl_sync(0xffffffffu, v, last);
      lo += last * gap;
      hi = min(hi, lo + gap);
    }
    item = lo;
    s = (int)(at_lo - x);
  }

  // All NT threads of the block together: the range of CTA `c` and the item
  // it starts in.  False: no work.
  template <int NT>
  __device__ bool init(Scratch* sc, int c, int min_per) {
    if constexpr (kDirect) {
      r = blockIdx.z;
      kh = blockIdx.y;
      rq = at::load_req(p, r);
      item = blockIdx.x;
      behind = false;
      return item < tiles(rq);
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kWarps = NT / 32;
    behind = false;
    if (p.n <= 32) {  // every warp by itself, a lane per request: no barriers (32 requests: 2 us of a call less)
      Req mine = {0, 0, 0, 0};
      if (lane < p.n) mine = at::load_req(p, lane);
      long long per_head = cost(p, mine), at = per_head * p.KVH, p0;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, at, off);
        if (lane >= off) at += y;
      }
      if (!range(__shfl_sync(0xffffffffu, at, 31), c, min_per, p0)) return false;
      at -= per_head * p.KVH;
      r = __ffs(__ballot_sync(0xffffffffu, at <= p0 && p0 < at + per_head * p.KVH)) - 1;
      rq.qlen = __shfl_sync(0xffffffffu, mine.qlen, r);
      rq.klen = __shfl_sync(0xffffffffu, mine.klen, r);
      rq.qst = __shfl_sync(0xffffffffu, mine.qst, r);
      rq.kbase = __shfl_sync(0xffffffffu, mine.kbase, r);
      find(p0 - __shfl_sync(0xffffffffu, at, r), __shfl_sync(0xffffffffu, per_head, r));
      return true;
    }
    long long total = 0, mine = 0, mine_at = 0, per_head = 0, p0 = 0;
    Req mine_rq = {0, 0, 0, 0};
    const bool one = p.n <= NT;
    if (tid == 0) sc->found = -1;
    for (int pass = 0; pass < 2; ++pass) {  // the sum of all requests' costs, then the request at this range's start
      long long carry = 0;
      for (int base = 0; base < p.n; base += NT) {
        if (pass == 0 || !one) {
          const int i = base + tid;
          mine_rq.qlen = 0;
          if (i < p.n) mine_rq = at::load_req(p, i);
          per_head = cost(p, mine_rq);
          mine = per_head * p.KVH;
          long long x = mine;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off) x += y;
          }
          if (lane == 31) sc->warp_sum[warp] = x;
          __syncthreads();
          long long ahead = 0, all = 0;
          for (int w = 0; w < kWarps; ++w) {
            if (w == warp) ahead = all;
            all += sc->warp_sum[w];
          }
          mine_at = carry + ahead + x - mine;
          carry += all;
          __syncthreads();
        }
        if (pass == 1 && mine > 0 && mine_at <= p0 && p0 < mine_at + mine) {
          sc->found = base + tid;
          sc->start = mine_at;
          sc->per_head = per_head;
          sc->rq = mine_rq;
        }
      }
      if (pass == 0) {
        total = carry;
        if (!range(total, c, min_per, p0)) return false;
      }
    }
    __syncthreads();
    r = sc->found;
    rq = sc->rq;
    find(p0 - sc->start, sc->per_head);  // (every warp by itself)
    return true;
  }

  // The next segment of this CTA's range.
  __device__ __forceinline__ bool next(Seg& g) {
    if constexpr (kDirect) {  // (more than one item only where the keys are more than the caller's bound)
      if (behind) item += gridDim.x;
      behind = true;
      if (item >= tiles(rq)) return false;
      g.r = r;
      g.kh = kh;
      g.kt = item;
      g.c0 = first_chunk(p, rq, item);
      g.n = last_chunk(p, rq) - g.c0;
      g.whole = g.head = true;
      g.nparts = 0;
      return true;
    } else while (true) {
      if (behind) {
        s += kW + last_chunk(p, rq) - first_chunk(p, rq, item);
        if (++item == tiles(rq)) {
          item = 0;
          if (++kh == p.KVH) {
            kh = 0;
            while (s < len) {  // the next request with work
              rq = at::load_req(p, ++r);
              if (tiles(rq) > 0) break;
            }
          }
        }
      }
      if (s >= len) return false;
      behind = true;
      if (p.snap && s < 0) continue;  // the CTA before has it
      const int first = first_chunk(p, rq, item), n = last_chunk(p, rq) - first;
      const int x0 = p.snap ? 0 : max(0, min(n, -s - kW)), x1 = p.snap ? n : max(0, min(n, len - s - kW));
      if (x0 >= x1) continue;
      g.r = r;
      g.kh = kh;
      g.kt = item;
      g.c0 = first + x0;
      g.n = x1 - x0;
      g.whole = x0 == 0 && x1 == n;
      g.head = x0 == 0;
      g.nparts = !g.whole && x0 == 0 ? (s + kW + n - 1) / per + 1 : 0;
      return true;
    }
  }
};

// The kernel of a call, as far as the caller's bounds tell (a wrong one costs
// time, not the result).
struct Plan {
  int cols;   // query rows per chunk of the tensor-core kernel (its N), 0: the CUDA-core kernel
  int ctas;
  bool whole; // no item is cut
  int tiles;  // > 0: a grid of items, this many key tiles wide (CUDA cores)
};
Plan plan_of(const fd_attn_args* a);
// The tensor-core kernel: fp16 and bf16 heads of 64 to 128 dims.
int mma_launch(KwParams& p, const fd_attn_args* a, const Plan& plan, cudaStream_t s);
// Adds up the cut items' partials, KT keys per item.
int combine_launch(const KwParams& p, int kt, cudaStream_t s);

}  // namespace kw
}  // namespace fdk
