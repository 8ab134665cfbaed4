// Chunk and cross attention: what the tensor-core kernel (fd_attn_mma.cu), the
// CUDA-core kernel and the combine (fd_attn.cu) share: parameters, the
// schedule, and the layout of the partials.
//
// Work.  The query tokens of a request are cut into tiles of `tq` tokens times
// the G query heads of a kv head (row = token * G + head).  An ITEM is one
// tile (or, with kPairs, two neighbouring tiles that share every K/V tile; an
// odd last tile is an item of its own) of one request and kv head, over the n
// key tiles of kt keys that its last query sees.  Items of all requests, kv
// heads and tiles in that order form a line of POSITIONS: an item takes w
// (its fixed cost: the query load, the pipeline's start, the epilogue) plus u
// per key tile (u = 2 for a pair, else 1).
//
// Schedule.  The line is cut into equal ranges, one per CTA of a grid that
// fills the GPU once, so a call with few queries over long keys and one with
// many queries both load all SMs, and no CTA waits for another.  An item cut by a range's end leaves fp32
// partials (O, m, l) of its rows that the combine kernel joins in ascending
// CTA order: results do not depend on timing.  A CTA's range holds at most
// one segment of an item that began earlier (slot 0) and one of an item that
// ends later (slot 1); all others are whole and written directly.  The
// lengths are device data, so each CTA finds its start itself: the cost of a
// request is a closed form (staircase), one thread per request, then one scan.
#pragma once

#include <math.h>

#include "fd_common.cuh"
#include "fd_internal.h"

namespace fdk {
namespace at {

constexpr int kMaxLen = 1 << 30;  // q_len and k_len: the closed forms stay in 32 bits

// One cut item, written by the CTA that holds its first segment.
struct Cut {
  int nparts;   // 0: none
  int row0;     // first query row (token) of the item in q / out
  int rows;     // token * G + head rows of the item
  int kh;
};

struct AttnParams {
  const unsigned char* q;
  unsigned char* out;
  float* lse;
  int64_t q_st, q_sh, o_st, o_sh;  // bytes
  int64_t lse_sh, lse_st;          // elements
  // the tiers, and third the copies of host blocks (stage_w > 0: block j <
  // stage_w of request r is block r * stage_w + j there)
  const unsigned char* k[3];
  const unsigned char* v[3];
  int64_t blk_sb[3], head_sb[3], tok_sb[3], nblk[3];  // bytes
  int stage_w;
  int64_t split;
  const int32_t* bt;       // null: cross attention (k[0], v[0] are rows, nblk[0] of them)
  int64_t bt_stride;
  const int32_t* bt_row;
  const int32_t* k_start;
  const int32_t *q_start, *q_len, *k_len;
  int bt_width, bt_rows;   // bt_rows 0: not known
  int n, T, H, KVH, G, D, BS;
  int host[2];             // tier is mapped host memory
  float sl2;               // scale * log2(e)
  int tq;                  // tokens per query tile
  int ctas;
  int snap;                // no item is cut: each is its start's CTA's (whole_items)
  Cut* cuts;               // [ctas]
  float* part_ml;          // [ctas][2][rows per item][2]: m (log2 domain), l
  float* part_o;           // [ctas][2][D / 4][rows per item][4]
  int out32;               // rows of out are 32-byte aligned (fd_attn_mma.cu)
  int32_t* err;
};

// 1 / l, and the natural log-sum-exp, of a row with maximum m (log2 domain) and
// sum l: 0 and -inf where no key is seen (l = 0), and a NaN stays a NaN.
__device__ __forceinline__ float row_inv(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float row_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

// 2^x by the SFU's ex2 instruction (relative error a few ulp; 2^-inf = 0).
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The sum of floor((a i + b) / m) over 0 <= i < n, for a n + b + m < 2^32: a
// staircase of key tiles.  The whole multiples of m in a and b are added at
// once.  What is left is the number of points (i, y) with 1 <= y and m y <=
// a i + b, none of them above `top`.  It is n top less the points above the
// line, and at height y those are the i below ceil((m y - b) / a) =
// floor((m (y - 1) + m - b + a - 1) / a): a staircase again, over top steps
// and with a and m exchanged, so that the numbers shrink as in Euclid's
// division.
__device__ __forceinline__ long long staircase(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  long long sum = 0;
  for (bool minus = false; n > 0; minus = !minus) {
    long long part = 0;
    if (a >= m) {
      part = (long long)(a / m) * ((long long)n * (n - 1) / 2);
      a %= m;
    }
    if (b >= m) {
      part += (long long)(b / m) * n;
      b %= m;
    }
    const uint32_t top = (a * (n - 1) + b) / m;
    part += (long long)n * top;
    sum += minus ? -part : part;
    const uint32_t was_m = m;
    b = m - b + a - 1;
    m = a;
    a = was_m;
    n = top;  // 0: no point is left (m may be 0 then)
  }
  return sum;
}

// A request's lengths, or qlen = 0 when it has no work (or does not fit its
// rows: FD_DEVERR_LEN).
struct Req {
  int qlen, klen, qst, kbase;  // kbase: table row, or first state row
};

__device__ __forceinline__ Req load_req(const AttnParams& p, int r) {
  Req q;
  q.qlen = p.q_len[r];
  q.klen = p.k_len[r];
  q.qst = p.q_start[r];
  q.kbase = p.bt != nullptr ? (p.bt_row != nullptr ? p.bt_row[r] : r) : p.k_start[r];
  bool ok = q.qlen >= 0 && q.qlen <= kMaxLen && q.klen >= 0 && q.klen <= kMaxLen;
  if (q.qlen > 0) {
    ok = ok && q.qst >= 0 && (long long)q.qst + q.qlen <= p.T;
    if (p.bt != nullptr)
      ok = ok && ((long long)q.klen + p.BS - 1) / p.BS <= p.bt_width && q.kbase >= 0 &&
           (p.bt_rows == 0 || q.kbase < p.bt_rows);
    else
      ok = ok && (q.klen == 0 || (q.kbase >= 0 && (long long)q.kbase + q.klen <= p.nblk[0]));
  }
  if (!ok) {
    set_error(p.err, FD_DEVERR_LEN);
    q.qlen = 0;
  }
  return q;
}

// kKT keys per tile, items of two query tiles with kPairs, fixed cost kW.
template <int kKT, bool kPairs, int kW>
struct Sched {
  struct Seg {
    int kh, tile0;   // kv head, first query tile of the item
    bool pair;
    int j0, j1;      // key tiles of this segment
    bool whole;
    int nparts;      // slot 1 segments: parts of the cut item
  };

  const AttnParams& p;
  // positions relative to the start of this CTA's range (the current item may
  // have begun before it): 32 bits, the line itself has 64
  int len, per;  // positions of this CTA, and of every CTA
  int s;         // the current item
  int r, kh, item;
  Req rq;        // of request r
  bool behind;   // the current item has been returned: step to the next one first

  __device__ __forceinline__ Sched(const AttnParams& params) : p(params) {}

  __device__ __forceinline__ static int tiles(const AttnParams& p, const Req& q) { return (q.qlen + p.tq - 1) / p.tq; }
  __device__ __forceinline__ static int items(const AttnParams& p, const Req& q) {
    const int t = tiles(p, q);
    return kPairs ? (t + 1) >> 1 : t;
  }
  __device__ __forceinline__ static bool is_pair(const AttnParams& p, const Req& q, int i) {
    return kPairs && 2 * i + 1 < tiles(p, q);
  }
  // keys, and key tiles, that the queries before token `te` of the request see
  __device__ __forceinline__ static int visible(const AttnParams& p, const Req& q, int te) {
    return max(0, p.bt != nullptr ? q.klen - q.qlen + te : q.klen);
  }
  __device__ __forceinline__ static int ntiles(const AttnParams& p, const Req& q, int te) {
    return (visible(p, q, te) + kKT - 1) / kKT;
  }
  __device__ __forceinline__ static int item_end(const AttnParams& p, const Req& q, int i) {
    return (int)min((long long)(i + 1) * (kPairs ? 2 : 1) * p.tq, (long long)q.qlen);
  }
  // positions of items 0 .. i - 1 of a request and kv head
  __device__ static long long before(const AttnParams& p, const Req& q, int i) {
    const int ni = items(p, q);
    long long ans = (long long)i * kW;
    // the last item may end early, or be a single tile
    const int reg = min(i, ni - 1);
    constexpr int u = kPairs ? 2 : 1;
    if (reg > 0) {
      if (p.bt == nullptr) {
        ans += (long long)u * reg * ntiles(p, q, 0);
      } else {
        const int st = u * p.tq, b = q.klen - q.qlen;
        const int m0 = b + st > 0 ? 0 : min(reg, -b / st);  // items whose queries see nothing
        if (reg > m0)
          ans += u * staircase((uint32_t)(reg - m0), kKT, (uint32_t)st,
                               (uint32_t)((long long)b + (long long)(m0 + 1) * st + kKT - 1));
      }
    }
    if (i == ni) ans += (is_pair(p, q, ni - 1) ? 2 : 1) * (long long)ntiles(p, q, q.qlen);
    return ans;
  }
  __device__ __forceinline__ static long long cost(const AttnParams& p, const Req& q) {
    return q.qlen > 0 ? before(p, q, items(p, q)) : 0;
  }

  struct Scratch {
    long long warp_sum[32];
    long long start, per_head;  // position of the request found; its cost per kv head
    long long item_start;
    int found, item;
    Req rq;
  };

  // a / b (b > 0), in 32 bits where they fit: a 64-bit division is a routine of hundreds of cycles
  __device__ __forceinline__ static long long quot(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
  }

  // All threads of the block (NT of them) together: the range of CTA `c` and
  // the item it starts in.  False: no work.
  template <int NT>
  __device__ bool init(Scratch* sc, int c, int min_per) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kWarps = NT / 32;
    long long total = 0, mine = 0, mine_at = 0, per_head = 0, p0 = 0;
    Req mine_rq = {0, 0, 0, 0};
    // pass 0 adds up all requests, pass 1 finds this CTA's (from the values
    // that pass 0 left when one round holds all requests)
    const bool one = p.n <= NT;
    if (tid == 0) sc->found = -1;
    for (int pass = 0; pass < 2; ++pass) {
      long long carry = 0;
      for (int base = 0; base < p.n; base += NT) {
        if (pass == 0 || !one) {
          const int i = base + tid;
          mine_rq.qlen = 0;
          if (i < p.n) mine_rq = load_req(p, i);
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
        if (total > (long long)kMaxLen * p.ctas) {  // positions of a range are 32 bits
          set_error(p.err, FD_DEVERR_LEN);
          return false;
        }
        per = (int)quot(total + p.ctas - 1, p.ctas);
        if (per < min_per) per = min_per;
        p0 = (long long)c * per;
        if (p0 >= total) return false;
        len = (int)min((long long)per, total - p0);
      }
    }
    __syncthreads();
    r = sc->found;
    rq = sc->rq;
    per_head = sc->per_head;
    const long long off = p0 - sc->start;
    kh = (int)quot(off, per_head);
    const long long x = off - (long long)kh * per_head;
    if (warp == 0) {  // the last item that starts at or before x, 32 candidates at a time
      int lo = 0, hi = items(p, rq);
      long long at = 0;
      while (hi - lo > 1) {
        const int gap = (hi - lo + 31) / 32;
        const int i = lo + lane * gap;
        const long long v = i < hi ? before(p, rq, i) : 0;
        const unsigned in = __ballot_sync(0xffffffffu, i < hi && v <= x);
        const int last = 31 - __clz(in);  // lane 0 always: before(lo) <= x
        at = __shfl_sync(0xffffffffu, v, last);
        lo += last * gap;
        hi = min(hi, lo + gap);
      }
      if (lane == 0) {
        sc->item = lo;
        sc->item_start = at - x;
      }
    }
    __syncthreads();
    item = sc->item;
    s = (int)sc->item_start;
    behind = false;
    return true;
  }

  // The next segment of this CTA's range.  (Stepping on is left to the next
  // call: it may read the next request's lengths, which the first segment's
  // loads need not wait for.)
  __device__ __forceinline__ bool next(Seg& g) {
    while (true) {
      if (behind) {
        s += kW + (is_pair(p, rq, item) ? 2 : 1) * ntiles(p, rq, item_end(p, rq, item));
        if (++item == items(p, rq)) {
          item = 0;
          if (++kh == p.KVH) {
            kh = 0;
            while (s < len) {  // the next request with work
              rq = load_req(p, ++r);
              if (rq.qlen > 0) break;
            }
          }
        }
      }
      if (s >= len) return false;
      behind = true;
      const bool pr = is_pair(p, rq, item);
      const int u = pr ? 2 : 1;
      const int n = ntiles(p, rq, item_end(p, rq, item));
      if (p.snap && s < 0) continue;  // the CTA before has it
      const int a = p.snap ? -kW : -s - kW, b = p.snap ? u * n : len - s - kW;
      // tile j belongs to the range that holds position s + kW + u j
      g.j0 = max(0, min(n, (a + u - 1) >> (u - 1)));
      g.j1 = max(0, min(n, (b + u - 1) >> (u - 1)));
      g.kh = kh;
      g.tile0 = (kPairs ? 2 : 1) * item;
      g.pair = pr;
      g.whole = g.j0 == 0 && g.j1 == n;
      g.nparts = 0;
      // the range that holds the last tile (ranges start at multiples of per)
      if (!g.whole && g.j0 == 0 && g.j1 > 0) g.nparts = (s + kW + u * (n - 1)) / per + 1;
      if (g.j0 < g.j1 || (n == 0 && s >= 0)) return true;
    }
  }
};

// Where block `j` of a request lies, given its entry `id` of the block table:
// the tier (2: its staged copy) and, in `id`, the block within it; -1: id is
// outside both tiers.
__device__ __forceinline__ int locate(const AttnParams& p, int r, int j, int64_t& id) {
  int t = 0;
  if (id >= p.split) {
    t = 1;
    id -= p.split;
  }
  if (id < 0 || id >= p.nblk[t]) {
    set_error(p.err, FD_DEVERR_BLOCK_ID);
    return -1;
  }
  if (t == 1 && j < p.stage_w) {
    id = (int64_t)r * p.stage_w + j;
    t = 2;
  }
  return t;
}

// Shared checks and parameters of the entry points over fd_attn_args; `what`
// names one in messages.  *empty: there is nothing to do.
enum Kind { kChunk, kCross, kWeights };
int fill_params(const fd_attn_args* a, Kind kind, const char* what, AttnParams& p, bool* empty);
// Copies of host blocks (K, or K and V) `base` bytes into the workspace, where
// they fit, and the bytes that they take.
int stage_launch(AttnParams& p, const fd_attn_args* a, size_t base, bool k_only, cudaStream_t s);
size_t stage_bytes(const fd_attn_args* a);

// The kernels' entry points for the host code in fd_attn.cu.
bool mma_covers(const fd_attn_args* a);
size_t mma_workspace(const fd_attn_args* a);
int mma_launch(AttnParams& p, const fd_attn_args* a, cudaStream_t s);
// At most kFewRows query rows (tokens x heads of a kv head) per request, as
// the caller says: `rows` of them (fd_attn_rows.cu; right for more, too).
constexpr int kFewRows = 32;
int rows_launch(AttnParams& p, const fd_attn_args* a, int rows, cudaStream_t s);
// Whether to give every item to one CTA whole, as far as the caller's bounds
// tell: at most one item per CTA, and cutting would take at most `most` key
// tiles off the longest CTA, less than the partials and the combine cost.
// (fd_attn_mma, 144 items of 64 tokens: 700 keys 26.9 us, cut 41.7; 1500 keys
// 40.0 and 55.2; fd_attn_rows, 112 items of 1024 keys 20.0 and 23.5; fd_attn,
// 288 items of 128 keys 23.4 and 24.2.)
bool whole_items(const fd_attn_args* a, int ctas, int item_rows, int keys, int most);
// Joins the cut items: `rows` rows per item at most.
int combine_launch(const AttnParams& p, int dtype, int rows, cudaStream_t s);

}  // namespace at
}  // namespace fdk
