// Chunk and cross attention on the 5th-generation tensor cores (tcgen05): fp16
// and bf16, head sizes 64 to 128 (padded to 64 or 128 dims in shared memory).
//
//   S [128 rows x 64 keys] = Q . K^T,  P = 2^(scale log2(e) S - m),
//   l = sum P,  O [128 rows x D] += P . V,  o = O / l, lse = ln 2 (m + log2 l)
//
// A CTA walks its range of the schedule (fd_attn.cuh) segment by segment and
// runs two STREAMS of such products.  In a pair (256 rows and more) the
// streams are two neighbouring query tiles and share every K/V tile; in a
// single tile (few query rows: bound by the bytes of the cache) stream A
// takes the first 64 keys of every key tile and stream B the second 64, for
// the same query tile, and the two are joined in registers at the end.  Either
// way both streams wait for every tile and release it: a stream that waited
// only for every other one would, in a ring of 3 or 5 slots, see every other
// phase of a slot's barrier, and the parity of the phase before the last
// would let it pass before the tile between has landed.
//
// What would bound a stream that takes one step after the other is its chain
// (scores, softmax, P.V, scores ...), with the tensor cores and the SFU each
// idle half of the time.  So a stream works on 64 keys at a time with two S
// buffers: q.K^T of step i + 2 is issued right behind P.V of step i, and the
// softmax of step i + 1 finds its scores ready.  Twelve warps:
//   8      schedule, Q tiles and K tiles  } TMA boxes of 8 to 128 keys (what
//   10     V tiles                        } divides a block) with the 128-byte
//          swizzle the MMA reads, or 16-byte loads stored in the same layout
//          where a box is in the host tier, spans blocks (block sizes that are
//          no multiple of 8), or is cut by the end of a request's V (rows
//          behind it must be 0: P is 0 there, and 0 x NaN is not)
//   9, 11  one thread each issues the MMAs of stream A, B (one thread alone
//          issues an MMA per ~70 cycles, more than a 64-key step leaves)
//   0-3, 4-7  softmax of stream A, B: one thread per row.  P overwrites the
//          first half of its S buffer in TMEM as 16-bit values (the A operand
//          of P.V); O stays in TMEM over a segment and is rescaled only when a
//          row's maximum passes its reference m by more than 2^8, so P stays
//          below 2^8; row sums add the fp32 values of P.
// TMEM: S/P of A [0, 128), of B [128, 256), two buffers of 64 columns each; O
// of A [256, 384), of B [384, 512).
// Scores, sums and O are fp32; P is rounded to the input type (the tensor
// core's operand type), the result once.  Every wait is bounded, and a role
// that gives up raises the CTA's abort flag for the others.
//
// Measured: 2 x 2048 tokens of 32 heads over up to 12288 keys of 8 heads x 128
// in 594 us, 995 TFLOP/s (over 8192: 440 us, 1093).  The tensor pipe is busy
// for 67% of the time: q.K^T of 64 keys is held up by the shared memory that
// feeds it (48 cycles per MMA for 32 of arithmetic, ~68 beside the other
// stream's and the TMA's writes), and a step of both streams takes 1750 cycles
// where 1270 of MMAs alone would do and the SFU needs 1024.  Tried and slower:
// q.K^T of 128 keys into both buffers at once (the streams fall into step: 700
// us), a quarter of the exponentials by a polynomial on the FMA pipe (623 us);
// as fast: the row maximum found in the SFU's shadow (605 us), fewer commits
// (602 us).

#include <type_traits>

#include "fd_attn_mma.cuh"

namespace fdk {
namespace at {
namespace mm {

constexpr int kM = 128;             // rows per query tile (MMA M)
constexpr int kHalf = 64;           // keys per step of a stream
constexpr int kWarpK = 8, kWarpMmaA = 9, kWarpV = 10, kWarpMmaB = 11;
constexpr int kThreads = 12 * 32;
constexpr int kSegs = 4;            // segments in flight between the roles
constexpr int kSegReaders = 11;     // MMA threads, V producer, eight softmax warps
constexpr int kItemRows = 2 * kM;
constexpr int kMaxCtas = 160;
constexpr int kFixed = 3;           // an item's fixed cost in key tiles of a single (of 2, 5 and 8 none is better throughout)
// Least positions of a CTA: 64 tokens of 32 heads over 1500 and 2048 keys 23.4
// and 24.2 us; with 2, 23.8 and 25.5; with 5, 24.6 and 25.2; with 7, 26.6 and
// 25.9.
constexpr int kMinPer = 4;
typedef Sched<kKT, true, kFixed> Walk;

template <int KD>
struct Geo {
  static constexpr int kPanels = KD / 64;
  static constexpr int kTile = kPanels * kPanel;
  static constexpr int kRingK = KD == 128 ? 3 : 5;
  static constexpr int kRingV = KD == 128 ? 2 : 5;
  static constexpr int kOffK = 2 * kTile;
  static constexpr int kOffV = kOffK + kRingK * kTile;
  static constexpr int kOffBar = kOffV + kRingV * kTile;
  // q full/empty, k full/empty, v full/empty, s_full[2][2], p_full[2][2], pv_done[2],
  // o_full[2], o_both, o_empty, ml_full, seg full/empty, drain
  static constexpr int kNumBars = 2 + 2 * kRingK + 2 * kRingV + 4 + 4 + 2 + 2 + 3 + 2 * kSegs + 1;
  static constexpr int kOffSeg = (kOffBar + kNumBars * 8 + 15) / 16 * 16;
  static constexpr int kOffMl = kOffSeg + kSegs * 64;   // [2 streams][128 rows] float2 (before that: Walk::Scratch)
  static constexpr int kOffMisc = kOffMl + 2 * kM * 8;  // abort flag, TMEM address
  static constexpr int kSmem = kOffMisc + 16;
  static_assert(kSmem <= 227 * 1024, "smem budget");
};

// One segment as the roles see it.
struct SegInfo {
  int live;      // 0: no more segments
  int pair;
  int j0, m;     // first key tile, key tiles
  int n0, n1;    // steps (64 keys) of stream A, B
  int tok0;      // first query token of the item within the request
  int req, qst, qlen, klen, kbase, kh;
  int slot;      // -1: whole, else its slot of the partials
  int pad[2];
};
static_assert(sizeof(SegInfo) == 64, "segment record");

// The end of a segment for one softmax warp of stream x: o and lse of its
// rows, or their partials.  A pair's stream has its own tile and all dims; in
// a single the two warpgroups take half of the dims each of the joined
// streams.  nkey: segments with keys before this one.  Not inlined: what it
// needs stays out of the main loop's registers.
template <typename T, int KD>
__device__ __noinline__ bool finish_rows(const AttnParams& p, const SegInfo& seg, int x, uint32_t t_s, float m, float l,
                                         bool any_row, int nkey, uint32_t* phases, float2* ml, uint64_t* o_empty,
                                         volatile int* misc) {
  uint64_t* o_full = o_empty - 3;  // [2], then o_both, o_empty, ml_full
  uint64_t* o_both = o_empty - 1;
  uint64_t* ml_full = o_empty + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = x ? seg.n1 : seg.n0;
  uint32_t ph = *phases;
  const bool pair = seg.pair != 0, single = !pair;
  const int row = (warp & 3) * 32 + lane;  // row of the tile = TMEM lane
  const int tg = row / p.G, hg = row % p.G;
  const uint32_t t_o = t_s - x * kKT + 2 * kKT;  // O of stream A; B's 128 columns on
  const int m_tiles = seg.m, slot = seg.slot;
  const int qi = seg.tok0 + (pair ? x * p.tq : 0) + tg;
  const bool row_ok = tg < p.tq && qi < seg.qlen;
  float wa = 1.f, wb = 0.f;  // weights of stream A's and B's O
  // everyone has read the m and l of the segment with keys before
  if (m_tiles > 0 && nkey > 0 &&
      !__all_sync(0xffffffffu, wait_or_abort(o_empty, (uint32_t)(nkey - 1) & 1u, misc, p.err)))
    return false;
  if (single && m_tiles > 0) {
    ml[x * kM + row] = make_float2(m, l);
    __syncwarp();
    if (lane == 0) mbar_arrive(ml_full);
    if (!__all_sync(0xffffffffu, wait_or_abort(ml_full, (ph >> 3) & 1u, misc, p.err) &&
                                     wait_or_abort(o_both, (ph >> 3) & 1u, misc, p.err)))
      return false;
    ph ^= 8u;
    const float2 other = ml[(x ^ 1) * kM + row];
    const float mm = fmaxf(m, other.x);
    const float base = mm == -INFINITY ? 0.f : mm;
    const float wo = exp2f(m - base), wt = exp2f(other.x - base);
    wa = x ? wt : wo;
    wb = x ? wo : wt;
    l = l * wo + other.y * wt;
    m = mm;
  } else if (m_tiles > 0) {
    if (!__all_sync(0xffffffffu, wait_or_abort(&o_full[x], (ph >> 2) & 1u, misc, p.err))) return false;
    ph ^= 4u;
  }
  tc_fence_after();
  const int64_t tok = seg.qst + qi;
  const int h = seg.kh * p.G + hg;
  const bool have_b = single && seg.n1 > 0;
  const bool have = single ? m_tiles > 0 : n > 0;
  const float inv = slot >= 0 ? 1.f : row_inv(l);
  wa *= inv;
  wb *= inv;
  const int item_row = (pair ? x * p.tq * p.G : 0) + row;
  if (row_ok && (!single || x == 0)) {
    if (slot >= 0) {
      reinterpret_cast<float2*>(p.part_ml)[(int64_t)slot * kItemRows + item_row] = make_float2(m, l);
    } else if (p.lse != nullptr) {
      p.lse[h * p.lse_sh + tok * p.lse_st] = row_lse(m, l);
    }
  }
  __syncwarp();
  const int c_lo = single ? x * (KD / 32) : 0, c_hi = single ? c_lo + KD / 32 : KD / 16;  // 16 dims each
  if (any_row) {
#pragma unroll 1
    for (int c = c_lo; c < c_hi; ++c) {
      if (16 * c >= p.D) break;
      uint32_t oa[16], ob[16];
      float f[16];
      if (have) tmem_ld16_nowait(t_o + (single ? 0 : x * kM) + 16 * c, oa);
      if (have_b) tmem_ld16_nowait(t_o + kM + 16 * c, ob);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        f[e] = have ? __uint_as_float(oa[e]) * wa : 0.f;
        if (have_b) f[e] = fmaf(__uint_as_float(ob[e]), wb, f[e]);
      }
      if (row_ok && slot >= 0) {  // [dim / 4][row][dim % 4]: a warp's rows side by side
        float4* po = reinterpret_cast<float4*>(p.part_o) +
                     ((int64_t)slot * (p.D / 4) + 4 * c) * kItemRows + item_row;
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (16 * c + e < p.D) po[(e / 4) * kItemRows] = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
      } else if (row_ok) {
        unsigned char* po = p.out + tok * p.o_st + h * p.o_sh + 32 * c;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = pack2<T>(f[2 * e], f[2 * e + 1]);
        if (p.out32) {
          stg256(po, w);
        } else {
          *reinterpret_cast<uint4*>(po) = make_uint4(w[0], w[1], w[2], w[3]);
          if (16 * c + 8 < p.D) *reinterpret_cast<uint4*>(po + 16) = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
      __syncwarp();  // the TMEM loads are the whole warp's
    }
  }
  *phases = ph;
  return true;
}

template <typename T, int KD>
__global__ void __launch_bounds__(kThreads, 1) fd_attn_mma_kernel(const __grid_constant__ MmaParams mp) {
  typedef Geo<KD> Ge;
  constexpr int kTile = Ge::kTile, kRingK = Ge::kRingK, kRingV = Ge::kRingV;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdQK = instr_desc(kBF16, false, kM, kHalf);
  constexpr uint32_t kIdPV = instr_desc(kBF16, false, kM, KD, true);  // V: MN-major B
  const AttnParams& p = mp.a;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + Ge::kOffBar);
  uint64_t* q_empty = q_full + 1;         // both streams' MMA commits after a segment's last q.K^T
  uint64_t* k_full = q_empty + 1;         // [kRingK]
  uint64_t* k_empty = k_full + kRingK;    // [kRingK] two arrivals: both streams are done with the tile
  uint64_t* v_full = k_empty + kRingK;    // [kRingV]
  uint64_t* v_empty = v_full + kRingV;    // [kRingV] two arrivals
  uint64_t* s_full = v_empty + kRingV;    // [2][2] MMA commit: S of the stream's step is in its buffer
  uint64_t* p_full = s_full + 4;          // [2][2] the stream's four softmax warps wrote P there
  uint64_t* pv_done = p_full + 4;         // [2] MMA commit after each P.V of the stream
  uint64_t* o_full = pv_done + 2;         // [2] pairs: MMA commit after the stream's last P.V, if it has any
  uint64_t* o_both = o_full + 2;          // singles: both streams' last P.V, likewise
  // all eight softmax warps are done with a segment that has keys.  In such a
  // segment they await both MMA threads (o_full or o_both, also of a stream
  // without steps), so those never find this barrier a phase past the one
  // that they wait for; a segment without keys is left out
  uint64_t* o_empty = o_both + 1;
  uint64_t* ml_full = o_empty + 1;        // singles: both streams' m and l are in shared memory
  uint64_t* seg_full = ml_full + 1;       // [kSegs]
  uint64_t* seg_empty = seg_full + kSegs; // [kSegs]
  uint64_t* drain = seg_empty + kSegs;
  SegInfo* segs = reinterpret_cast<SegInfo*>(smem + Ge::kOffSeg);
  float2* ml = reinterpret_cast<float2*>(smem + Ge::kOffMl);
  volatile int* misc = reinterpret_cast<volatile int*>(smem + Ge::kOffMisc);  // [0] abort, [1] TMEM address

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;

  griddep_launch_dependents();  // the combine's CTAs may start, and wait for this grid's end
  prefetch_maps(mp, (int)threadIdx.x - 64);
  init_barriers(q_full, Ge::kNumBars, [&](int i) -> uint32_t {
    uint64_t* b = q_full + i;
    if (b == q_empty || b == o_both || b == drain || (b >= k_empty && b < v_full) || (b >= v_empty && b < s_full)) return 2;
    return b >= p_full && b < pv_done ? 4 : b == o_empty || b == ml_full ? 8 : b >= seg_empty ? kSegReaders : 1;
  });
  if (threadIdx.x == 0) {
    p.cuts[cta].nparts = 0;
    misc[0] = 0;
  }
  Walk walk(p);
  static_assert(sizeof(Walk::Scratch) <= 2 * kM * 8, "scratch of the schedule");
  if (!walk.init<kThreads>(reinterpret_cast<Walk::Scratch*>(ml), cta, kMinPer)) return;  // all threads alike, before any TMEM is held
  if (warp == kWarpMmaA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(smem + Ge::kOffMisc + 4)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)misc[1];

  if (warp == kWarpK) {
    // ------------------------------------------------ schedule, Q and K tiles
    const uint64_t pol_once = l2_evict_first_policy(), pol_again = l2_evict_normal_policy();
    auto steps = [](int vis, int j0, int j1) {
      return max(0, min(2 * j1, (vis + kHalf - 1) / kHalf) - 2 * j0);
    };
    int nseg = 0, nq = 0, st = 0;
    uint32_t tiles = 0, ph = 0;  // K tiles issued; phase parity of the ring's current round
    bool ok = true;
    Walk::Seg g;
    while (ok) {
      const bool more = walk.next(g);
      const int ss = nseg % kSegs;
      if (nseg >= kSegs)
        ok = __all_sync(0xffffffffu, wait_or_abort(&seg_empty[ss], (uint32_t)(nseg / kSegs - 1) & 1u, misc, p.err));
      if (!ok) break;
      const Req rq = walk.rq;
      const int tok0 = g.tile0 * p.tq;
      if (lane == 0) {
        SegInfo& i = segs[ss];
        i.live = more;
        if (more) {
          i.pair = g.pair;
          i.j0 = g.j0;
          i.m = g.j1 - g.j0;
          // steps of 64 keys: those that some query of the stream's tile sees
          const int last = Walk::visible(p, rq, min(tok0 + (g.pair ? 2 : 1) * p.tq, rq.qlen));
          if (g.pair) {
            i.n0 = steps(Walk::visible(p, rq, tok0 + p.tq), g.j0, g.j1);
            i.n1 = steps(last, g.j0, g.j1);
          } else {
            const int halves = steps(last, g.j0, g.j1);  // the last tile's second half may not be seen
            i.n0 = (halves + 1) >> 1;
            i.n1 = halves >> 1;
          }
          i.tok0 = tok0;
          i.qst = rq.qst;
          i.qlen = rq.qlen;
          i.klen = rq.klen;
          i.kbase = rq.kbase;
          i.kh = g.kh;
          i.slot = g.whole ? -1 : 2 * cta + (g.j0 > 0 ? 0 : 1);
          i.req = walk.r;
          if (g.nparts > 0)
            p.cuts[cta] = Cut{g.nparts, rq.qst + tok0, min((g.pair ? 2 : 1) * p.tq, rq.qlen - tok0) * p.G, g.kh};
        }
        mbar_arrive(&seg_full[ss]);
      }
      __syncwarp();
      ++nseg;
      if (!more) break;
      if (g.j0 >= g.j1) continue;  // no key is seen: the softmax warps write zeros
      if (nq > 0 && !__all_sync(0xffffffffu, wait_or_abort(q_empty, (uint32_t)(nq - 1) & 1u, misc, p.err))) {
        ok = false;
        break;
      }
      ++nq;
      int id = box_block(mp, false, rq.kbase, rq.klen, g.j0, lane);
      const int nt = g.pair ? 2 : 1;
      if (mp.q_tma) {
        if (lane == 0) {
          mbar_expect_tx(q_full, (uint32_t)(nt * Ge::kPanels * p.tq * p.G * 128));
          for (int x = 0; x < nt; ++x)
            for (int c = 0; c < Ge::kPanels; ++c)
              tma_load_4d(smem + x * kTile + c * kPanel, &mp.tmap_q, 64 * c, g.kh * p.G, rq.qst + tok0 + x * p.tq, 0,
                          q_full, 0ull);
          mbar_arrive(q_full);
        }
      } else {
        for (int x = 0; x < nt; ++x)
          load_q<KD>(p, smem + x * kTile, kPanel, g.kh, rq.qst + tok0 + x * p.tq, min(p.tq, rq.qlen - tok0 - x * p.tq), lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      // a pair's neighbours read the same keys again: they stay in L2
      const uint64_t pol = g.pair ? pol_again : pol_once;
      for (int j = g.j0; j < g.j1; ++j) {
        const int id_next = j + 1 < g.j1 ? box_block(mp, false, rq.kbase, rq.klen, j + 1, lane) : -1;
        if (tiles >= (uint32_t)kRingK) ok = __all_sync(0xffffffffu, wait_or_abort(&k_empty[st], ph ^ 1u, misc, p.err));
        if (!ok) break;
        load_tile<KD>(mp, false, smem + Ge::kOffK + st * kTile, &k_full[st], j, walk.r, rq.kbase, rq.klen, g.kh, id, lane, pol);
        id = id_next;
        ++tiles;
        if (++st == kRingK) {
          st = 0;
          ph ^= 1u;
        }
      }
    }
    if (!ok) misc[0] = 1;
    // no copy of this warp is in flight when the CTA ends: the last tile of
    // each slot and the last Q (at once on the normal path)
    for (uint32_t s = 0; s < (uint32_t)kRingK && s < tiles; ++s) {
      const uint32_t last = s + kRingK * ((tiles - 1 - s) / kRingK);
      mbar_wait(&k_full[s], (last / kRingK) & 1u, p.err);
    }
    if (nq > 0) mbar_wait(q_full, (uint32_t)(nq - 1) & 1u, p.err);
  } else if (warp == kWarpV) {
    // ------------------------------------------------ V tiles
    const uint64_t pol_once = l2_evict_first_policy(), pol_again = l2_evict_normal_policy();
    int st = 0;
    uint32_t tiles = 0, ph = 0;
    bool ok = true;
    for (int nseg = 0; ok; ++nseg) {
      const int ss = nseg % kSegs;
      ok = __all_sync(0xffffffffu, wait_or_abort(&seg_full[ss], (uint32_t)(nseg / kSegs) & 1u, misc, p.err));
      if (!ok) break;
      const SegInfo i = segs[ss];
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[ss]);
      if (!i.live) break;
      const uint64_t pol = i.pair ? pol_again : pol_once;
      int id = i.m > 0 ? box_block(mp, true, i.kbase, i.klen, i.j0, lane) : -1;
      for (int j = i.j0; j < i.j0 + i.m; ++j) {
        const int id_next = j + 1 < i.j0 + i.m ? box_block(mp, true, i.kbase, i.klen, j + 1, lane) : -1;
        if (tiles >= (uint32_t)kRingV) ok = __all_sync(0xffffffffu, wait_or_abort(&v_empty[st], ph ^ 1u, misc, p.err));
        if (!ok) break;
        load_tile<KD>(mp, true, smem + Ge::kOffV + st * kTile, &v_full[st], j, i.req, i.kbase, i.klen, i.kh, id, lane, pol);
        id = id_next;
        ++tiles;
        if (++st == kRingV) {
          st = 0;
          ph ^= 1u;
        }
      }
    }
    if (!ok) misc[0] = 1;
    for (uint32_t s = 0; s < (uint32_t)kRingV && s < tiles; ++s) {
      const uint32_t last = s + kRingV * ((tiles - 1 - s) / kRingV);
      mbar_wait(&v_full[s], (last / kRingV) & 1u, p.err);
    }
  } else if (warp == kWarpMmaA || warp == kWarpMmaB) {
    // ------------------------------------------------ MMA issuer of stream x
    if (lane == 0) {
      const int x = warp == kWarpMmaB ? 1 : 0;
      const uint32_t t_s = tmem + x * kKT, t_o = tmem + 2 * kKT + x * kM;
      const uint32_t base = smem_u32(smem) >> 4;
      // 16-byte units: from one half (64 keys) of a K/V tile to the other, and between its panels
      const uint32_t half = (uint32_t)mp.group * 8 >> 4, panel = (uint32_t)mp.panel >> 4;
      const uint32_t q_hi = desc_hi(1024), kv_hi = desc_hi((uint32_t)mp.group);
      uint64_t* const my_s = s_full + 2 * x;
      uint64_t* const my_p = p_full + 2 * x;
      uint32_t nq = 0;  // segments with keys
      uint32_t pp = 0;  // phase parities of p_full's two buffers
      int ks_ = 0, vs_ = 0;  // ring slots (and phases) of the next K and V tile
      uint32_t kp = 0, vp = 0;
      bool ok = true;
      for (int nseg = 0; ok; ++nseg) {
        const int ss = nseg % kSegs;
        ok = poll_or_abort(&seg_full[ss], (uint32_t)(nseg / kSegs) & 1u, misc, p.err);
        if (!ok) break;
        const int live = segs[ss].live, pair = segs[ss].pair, m = segs[ss].m;
        const int n = x ? segs[ss].n1 : segs[ss].n0;
        mbar_arrive(&seg_empty[ss]);
        if (!live) break;
        // of a pair step i takes half i & 1 of tile i / 2, of a single half x of tile i
        auto first_of_tile = [&](int i) { return !pair || (i & 1) == 0; };
        auto last_of_tile = [&](int i) { return !pair || (i & 1) || i == n - 1; };
        const uint32_t q_lo = base + (uint32_t)((pair ? x : 0) * (kTile >> 4)) + (1u << 16);
        auto qk = [&](int i) {  // q.K^T of step i into its S buffer
          const int h = i & 1;
          if (first_of_tile(i) && !poll_or_abort(&k_full[ks_], kp, misc, p.err)) return false;
          tc_fence_after();
          const uint32_t k_lo = base + (uint32_t)((Ge::kOffK + ks_ * kTile) >> 4) + (uint32_t)(pair ? h : x) * half + (1u << 16);
#pragma unroll
          for (int ks = 0; ks < KD / 16; ++ks)
            umma_f16_lo(t_s + h * kHalf, q_lo + (uint32_t)(((ks >> 2) * kPanel + (ks & 3) * 32) >> 4), q_hi,
                        k_lo + (uint32_t)(ks >> 2) * panel + (uint32_t)((ks & 3) * 32 >> 4), kv_hi, kIdQK,
                        ks > 0 ? 1u : 0u);
          umma_commit(&my_s[h]);
          if (last_of_tile(i)) {
            umma_commit(&k_empty[ks_]);
            advance<kRingK>(ks_, kp);
            if (i == n - 1) umma_commit(q_empty);
          }
          return true;
        };
        if (m > 0) {
          ok = poll_or_abort(q_full, nq & 1u, misc, p.err);
          ++nq;
          if (ok && n == 0) mbar_arrive(q_empty);
        }
        if (ok && n > 0) ok = qk(0) && (n < 2 || qk(1));
        // the O of the segment with keys before has been read
        if (ok && m > 0 && nq > 1) ok = poll_or_abort(o_empty, (nq - 2) & 1u, misc, p.err);
        for (int i = 0; ok && i < n; ++i) {
          const int h = i & 1;
          if (first_of_tile(i)) ok = poll_or_abort(&v_full[vs_], vp, misc, p.err);
          ok = ok && poll_or_abort(&my_p[h], (pp >> h) & 1u, misc, p.err);
          if (!ok) break;
          pp ^= 1u << h;
          tc_fence_after();
          const uint32_t v_lo =
              base + (uint32_t)((Ge::kOffV + vs_ * kTile) >> 4) + (uint32_t)(pair ? h : x) * half + (panel << 16);
#pragma unroll
          for (int ks = 0; ks < kHalf / 16; ++ks)
            umma_f16_ts_lo(t_o, t_s + h * kHalf + 8 * ks, v_lo + (uint32_t)ks * (half / 4), kv_hi, kIdPV,
                           (i > 0 || ks > 0) ? 1u : 0u);
          umma_commit(&pv_done[x]);
          if (i + 2 < n) ok = qk(i + 2);
          if (last_of_tile(i)) {
            umma_commit(&v_empty[vs_]);
            advance<kRingV>(vs_, vp);
          }
        }
        if (!ok) break;
        if (m > 0) {
          uint64_t* const done = pair ? &o_full[x] : o_both;
          if (n == 0)
            mbar_arrive(done);
          else
            umma_commit(done);
          // tiles that only the other stream sees
          for (int t = pair ? (n + 1) >> 1 : n; ok && t < m; ++t) {
            ok = poll_or_abort(&k_full[ks_], kp, misc, p.err);
            if (ok) mbar_arrive(&k_empty[ks_]);
            ok = ok && poll_or_abort(&v_full[vs_], vp, misc, p.err);
            if (ok) mbar_arrive(&v_empty[vs_]);
            advance<kRingK>(ks_, kp);
            advance<kRingV>(vs_, vp);
          }
        }
      }
      if (!ok) misc[0] = 1;
      umma_commit(drain);  // all MMAs of both threads complete before TMEM is released
      mbar_wait(drain, 0u, p.err);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ softmax of stream x
    const int x = warp >> 2;
    const uint32_t t_s = tmem + ((uint32_t)((warp & 3) * 32) << 16) + x * kKT;
    // phase parities of s_full (bits 0, 1), o_full (2), o_both / ml_full (3),
    // pv_done of the step at hand (4)
    uint32_t ph = 0;
    int nkey = 0;  // segments with keys
    bool ok = true;
    for (int nseg = 0; ok; ++nseg) {
      const int ss = nseg % kSegs;
      ok = __all_sync(0xffffffffu, wait_or_abort(&seg_full[ss], (uint32_t)(nseg / kSegs) & 1u, misc, p.err));
      if (!ok) break;
      const SegInfo& seg = segs[ss];  // stays until this segment's end
      if (!seg.live) break;
      const int n = x ? seg.n1 : seg.n0;
      // step i's first key: of a pair half i & 1 of tile i / 2, of a single half x of tile i
      const int per = seg.pair ? 1 : 0, jfirst = seg.j0 * kKT + (seg.pair ? 0 : x * kHalf);
      bool any_row;
      int lim, lim_all;  // last key that this row sees, that all rows of the tile see
      {
        const int tg = ((warp & 3) * 32 + lane) / p.G;  // token of the row within the tile
        const int q0 = seg.tok0 + (seg.pair ? x * p.tq : 0), qi = q0 + tg;
        const bool row_ok = tg < p.tq && qi < seg.qlen;
        any_row = __any_sync(0xffffffffu, row_ok);
        lim = !row_ok ? -1 : p.bt != nullptr ? seg.klen - seg.qlen + qi : seg.klen - 1;
        lim_all = p.bt != nullptr ? seg.klen - seg.qlen + q0 : seg.klen - 1;
      }
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < n; ++i) {
        const int h = i & 1;
        ok = __all_sync(0xffffffffu, wait_or_abort(&s_full[2 * x + h], (ph >> h) & 1u, misc, p.err));
        if (!ok) break;
        ph ^= 1u << h;
        tc_fence_after();
        if (any_row) {
          const int key0 = jfirst + (i >> per) * kKT + (i & per) * kHalf;
          uint32_t ra[32], rb[32];
          tmem_ld32_nowait(t_s + h * kHalf, ra);
          tmem_ld32_nowait(t_s + h * kHalf + 32, rb);
          tmem_wait_ld();
          if (key0 + kHalf - 1 > lim_all) {
            hide(ra, lim - key0 + 1);
            hide(rb, lim - key0 + 1 - 32);
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            m4[0] = fmax3(m4[0], __uint_as_float(ra[e]), __uint_as_float(ra[e + 1]));
            m4[1] = fmax3(m4[1], __uint_as_float(rb[e]), __uint_as_float(rb[e + 1]));
            m4[2] = fmax3(m4[2], __uint_as_float(ra[e + 2]), __uint_as_float(ra[e + 3]));
            m4[3] = fmax3(m4[3], __uint_as_float(rb[e + 2]), __uint_as_float(rb[e + 3]));
          }
          const float mxs = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.sl2;
          const bool grow = m != -INFINITY && mxs > m + 8.f;
          if (__any_sync(0xffffffffu, grow)) {
            // O takes the earlier steps: the last one's P.V may still run (that
            // of the one before it is done: this S's q.K^T was issued behind
            // it, so the phase before the awaited one is known to have passed)
            ok = __all_sync(0xffffffffu, wait_or_abort(&pv_done[x], ((ph >> 4) & 1u) ^ 1u, misc, p.err));
            if (!ok) break;
            tc_fence_after();
            const float alpha = grow ? exp2f(m - mxs) : 1.f;
#pragma unroll 1
            for (int c = 0; c < KD / 16; ++c) {
              uint32_t o[16];
              tmem_ld16_nowait(t_s + 2 * kKT + 16 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(t_s + 2 * kKT + 16 * c, o);
            }
            l *= alpha;
          }
          if (grow || m == -INFINITY) m = mxs;
          const float neg_m = m == -INFINITY ? 0.f : -m;
          const f2_t sl2x2 = f2_pack(p.sl2, p.sl2), nm2 = f2_pack(neg_m, neg_m);
          f2_t ls[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
          auto expo = [&](const uint32_t (&r)[32], int col) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float a0, a1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), sl2x2, nm2), a0, a1);
              const float p0 = ex2_approx(a0), p1 = ex2_approx(a1);
              pk[e] = pack2<T>(p0, p1);
              ls[e & 1] = f2_add(ls[e & 1], f2_pack(p0, p1));
            }
            tmem_st16(t_s + h * kHalf + col, pk);
          };
          expo(ra, 0);
          expo(rb, 16);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * x + h]);
          float a0, a1;
          f2_unpack(f2_add(ls[0], ls[1]), a0, a1);
          l += a0 + a1;
        } else if (lane == 0) {
          mbar_arrive(&p_full[2 * x + h]);
        }
        ph ^= 16u;
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, finish_rows<T, KD>(p, seg, x, t_s, m, l, any_row, nkey, &ph, ml, o_empty, misc));
      if (!ok) break;
      tc_fence_before();
      const bool keyed = seg.m > 0;
      nkey += keyed ? 1 : 0;
      __syncwarp();
      if (lane == 0) {
        if (keyed) mbar_arrive(o_empty);
        mbar_arrive(&seg_empty[ss]);
      }
    }
    if (!ok) misc[0] = 1;
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpMmaA)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <typename T, int KD>
int launch(const MmaParams& mp, cudaStream_t s) {
  const void* kern = reinterpret_cast<const void*>(fd_attn_mma_kernel<T, KD>);
  static unsigned long long done = 0;
  const int st = fdh::ensure_smem(kern, Geo<KD>::kSmem, &done);
  if (st != FD_OK) return st;
  return fdh::launch_maybe_pdl(kern, dim3((unsigned)mp.a.ctas), dim3(kThreads), Geo<KD>::kSmem, s, false, mp,
                               "fd_attn_mma_kernel launch");
}

// {D, heads, tokens, blocks} (strides in bytes), box {64, box_heads, box_tokens, 1}.
bool encode_rows(CUtensorMap* m, const void* base, int dtype, int D, int heads, int tokens, int64_t blocks,
                 int64_t head_sb, int64_t tok_sb, int64_t blk_sb, int box_heads, int box_tokens) {
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)head_sb, (cuuint64_t)tok_sb, (cuuint64_t)blk_sb};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens, 1};
  return blocks <= 0x7fffffff && encode_map(m, base, dtype, 4, dims, strides, box);
}

// Heads of 128 dims: {64 dims, 8 tokens, 2 halves of the dims, BS / 8, lines},
// where a line is the BS tokens of one head of one block (line l at l *
// head_sb: heads and blocks in one dimension), box {64, 8, 2, box_tokens / 8,
// 1}: both halves of box_tokens rows in one copy.
bool encode_lines(CUtensorMap* m, const void* base, int dtype, int BS, int64_t lines, int64_t head_sb, int64_t tok_sb,
                  int box_tokens) {
  const cuuint64_t dims[5] = {64, 8, 2, (cuuint64_t)(BS / 8), (cuuint64_t)lines};
  const cuuint64_t strides[4] = {(cuuint64_t)tok_sb, 128, (cuuint64_t)(8 * tok_sb), (cuuint64_t)head_sb};
  const cuuint32_t box[5] = {64, 8, 2, (cuuint32_t)(box_tokens / 8), 1};
  return encode_map(m, base, dtype, 5, dims, strides, box);
}

void encode_maps(MmaParams& mp, const fd_attn_args* a, bool k_only) {
  const AttnParams& p = mp.a;
  const int D = p.D;
  mp.box_sh = 3;
  while (mp.box_sh < 7 && (p.bt == nullptr || p.BS % (2 << mp.box_sh) == 0)) ++mp.box_sh;
  // heads of 128 dims in small blocks: whole rows per copy, where every device
  // tier's blocks are whole numbers of its heads' strides (both usual layouts)
  bool by_lines = D == 128 && p.bt != nullptr && p.BS % kFine == 0 && mp.box_sh < 6;
  for (int t = 0; t < 3; ++t)
    if (p.nblk[t] > 0 && !(t < 2 && p.host[t]))
      by_lines = by_lines && p.head_sb[t] > 0 && p.blk_sb[t] >= p.head_sb[t] && p.blk_sb[t] % p.head_sb[t] == 0 &&
                 p.nblk[t] * (p.blk_sb[t] / p.head_sb[t]) < (1ll << 31);
  mp.group = by_lines ? 2048 : 1024;
  mp.panel = by_lines ? 1024 : kPanel;
  mp.q_tma = encode_rows(&mp.tmap_q, a->q, a->dtype, D, p.H, p.T, 1, p.q_sh, p.q_st, p.q_st * p.T, p.G, p.tq);
  for (int t = 0; t < 3; ++t) {
    if (p.nblk[t] == 0 || (t < 2 && p.host[t])) continue;
    const bool cross = p.bt == nullptr;
    if (cross && p.nblk[t] > 0x7fffffff) continue;  // rows by 16-byte loads
    if (!cross && p.BS % kFine != 0) continue;
    const int rows = cross ? (int)p.nblk[t] : p.BS;
    const int64_t blocks = cross ? 1 : p.nblk[t];
    const int64_t blk_sb = cross ? p.tok_sb[t] * rows : p.blk_sb[t];
    auto map = [&](CUtensorMap* m, const unsigned char* base, int keys) {
      return encode_rows(m, base, a->dtype, D, p.KVH, rows, blocks, p.head_sb[t], p.tok_sb[t], blk_sb, 1, keys);
    };
    if (by_lines) {
      mp.lines[t] = (int)(p.blk_sb[t] / p.head_sb[t]);
      auto lines = [&](CUtensorMap* m, const unsigned char* base) {
        return encode_lines(m, base, a->dtype, p.BS, (p.nblk[t] - 1) * mp.lines[t] + p.KVH, p.head_sb[t], p.tok_sb[t],
                            1 << mp.box_sh);
      };
      mp.kv_tma[t] = lines(&mp.tmap_k[t], p.k[t]) && (k_only || lines(&mp.tmap_v[t], p.v[t]));
    } else {
      mp.kv_tma[t] = map(&mp.tmap_k[t], p.k[t], 1 << mp.box_sh) && (k_only || map(&mp.tmap_v[t], p.v[t], 1 << mp.box_sh));
    }
    if (mp.box_sh > kFineSh && !k_only) mp.kv_tma[t] = mp.kv_tma[t] && map(&mp.tmap_vf[t], p.v[t], kFine);
  }
}

}  // namespace mm

bool mma_covers(const fd_attn_args* a) {
  return (a->dtype == FD_DTYPE_F16 || a->dtype == FD_DTYPE_BF16) && a->head_size >= 64 && a->head_size <= 128;
}

size_t mma_workspace(const fd_attn_args* a) {
  const size_t slots = 2 * (size_t)mm::kMaxCtas * mm::kItemRows;
  return mm::kMaxCtas * sizeof(Cut) + slots * 8 + slots * (size_t)a->head_size * 4;
}

int mma_launch(AttnParams& p, const fd_attn_args* a, cudaStream_t s) {
  // few query rows per request and kv head: the kernel made for them, which
  // spends no softmax on rows that are not there
  const int64_t rows = (int64_t)(a->max_q_len > 0 && a->max_q_len < p.T ? a->max_q_len : p.T) * p.G;
  if (rows <= kFewRows) return rows_launch(p, a, (int)rows, s);
  int dev = 0, sms = 0;
  int st = fdh::device_sms(&dev, &sms);
  if (st != FD_OK) return st;
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  p.cuts = reinterpret_cast<Cut*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + mm::kMaxCtas * sizeof(Cut));
  p.part_o = p.part_ml + 2 * 2 * (size_t)mm::kMaxCtas * mm::kItemRows;
  p.out32 = ((reinterpret_cast<uintptr_t>(p.out) | (uint64_t)p.o_st | (uint64_t)p.o_sh) & 31u) == 0 && p.D % 16 == 0;
  p.tq = mm::kM / p.G;
  p.ctas = sms < mm::kMaxCtas ? sms : mm::kMaxCtas;
  mm::MmaParams mp{};
  p.snap = whole_items(a, p.ctas, 2 * mm::kM, mm::kKT, mm::kWhole);
  mp.a = p;
  mm::encode_maps(mp, a);
  if (a->dtype == FD_DTYPE_BF16)
    st = p.D <= 64 ? mm::launch<__nv_bfloat16, 64>(mp, s) : mm::launch<__nv_bfloat16, 128>(mp, s);
  else
    st = p.D <= 64 ? mm::launch<__half, 64>(mp, s) : mm::launch<__half, 128>(mp, s);
  if (st != FD_OK || p.snap) return st;
  return combine_launch(p, a->dtype, mm::kItemRows, s);
}

}  // namespace at
}  // namespace fdk
