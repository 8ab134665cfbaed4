// Chunk and cross attention of few query rows (at most 32 per request and kv
// head: single tokens, draft tokens) on the tensor cores: fp16 and bf16, head
// sizes 64 to 128.
//
// Such calls are bound by the bytes of K and V, as long as the work per key
// tile stays below its load time (0.7 us for 32 KB at an SM's share of HBM).
// With the queries as the 128 rows of an MMA tile (fd_attn_mma.cu) it does
// not: a softmax thread has a row's 128 exponentials per tile however few rows
// are real.  So the products are turned over:
//   S^T [128 keys x N] = K . Q^T,  P = 2^(scale log2(e) S - m),  l = sum P,
//   O^T [dims x N] += V^T . P^T,   N = 16 or 32 query rows,
// a softmax thread has one KEY and an exponential per row, K and V are the MMA's A
// operands as they lie in shared memory, and the rows of O^T are dims, so a
// warp's output stores are whole lines.  The reference m of a column moves
// only when some score passes it by more than 2^8 (then, and on a segment's
// first tile, the 128 threads take the column's maximum together and rescale
// O); the sums l stay with their threads until the segment's end.
//
// A CTA walks its range of the schedule (fd_attn.cuh); eight warps: 0-3
// softmax, 4 schedule and Q tiles (segments ahead, so that the loads never
// wait for its arithmetic), 5 and 6 K and V tiles, 7 (one thread) the MMAs,
// q.K^T two tiles ahead of P.V over two S and two P buffers.  Heads of 64 dims
// take half of the shared memory, and two CTAs share an SM: one's loads run
// on while the other changes from one request to the next.
// Scores, sums and O are fp32; P is rounded to the input type (the tensor
// core's operand type), the result once.  Every wait is bounded; the four
// softmax warps agree at their barriers on going on.
//
// Measured: 32 requests of 1, 4 and 8 tokens of 32 heads over 4096 keys of 8
// heads x 128 in 87, 88 and 92 us (6.0 TB/s of cache read; fd_attn_mma 98 to
// 101); 24 of one token over 1500 keys of 20 heads x 64 in 47 us (fd_attn_mma
// 71); one request of 16384 keys, 1 and 8 tokens, in 25 and 28 us (31 and 31).

#include <type_traits>

#include "fd_attn_mma.cuh"

namespace fdk {
namespace at {
namespace rw {

using namespace mm;

constexpr int kWarpSched = 4, kWarpK = 5, kWarpV = 6, kWarpMma = 7;
constexpr int kThreads = 8 * 32;
constexpr int kSoft = 4 * 32;       // softmax threads
constexpr int kSegs = 4;            // segments in flight between the roles
constexpr int kSegReaders = 7;      // MMA thread, two producers, four softmax warps
constexpr int kMaxCtas = 320;
constexpr int kFixed = 2;           // an item's fixed cost in key tiles
// Least positions of a CTA: one request of 5 tokens over 1500 and 3500 keys of
// 8 heads x 128 17.3 and 20.2 us, 8192 keys of 8 x 64 22.5; with 2, 16.2, 20.7
// and 28.5; with 7, 18.4, 21.0 and 22.1.
constexpr int kMinPer = 4;
constexpr int kTmemCols = 128;      // S [0, 32), [32, 64), O [64, 96)
constexpr int kOcol = 64;
typedef Sched<kKT, false, kFixed> Walk;

template <int KD, int N>
struct Geo {
  static constexpr int kPanels = KD / 64;
  static constexpr int kTile = kPanels * kPanel;
  static constexpr int kRingK = KD == 64 && N == 32 ? 2 : 3;
  static constexpr int kRingV = 3;
  static constexpr int kQ = kPanels * N * 128;   // one Q buffer
  static constexpr int kP = 2 * N * 128;         // one P buffer: two panels of 64 keys
  static constexpr int kOffV = kRingK * kTile;
  static constexpr int kOffQ = kOffV + kRingV * kTile;
  static constexpr int kOffP = kOffQ + 2 * kQ;
  static constexpr int kOffBar = kOffP + 2 * kP;
  // k full/empty, v full/empty, q full/empty[2], s_full[2], p_full[2], pv_done, o_full, o_empty, seg full/empty, drain
  static constexpr int kNumBars = 2 * kRingK + 2 * kRingV + 4 + 2 + 2 + 3 + 2 * kSegs + 1;
  static constexpr int kOffSeg = (kOffBar + kNumBars * 8 + 15) / 16 * 16;
  static constexpr int kOffRed = kOffSeg + kSegs * 64;   // [4 warps][N] maxima, then sums (before that: Walk::Scratch)
  static constexpr int kOffM = kOffRed + 4 * N * 4 + 512;  // [N] m, then [N] factors of l and O
  static constexpr int kOffRow = kOffM + 2 * N * 4;      // [N] where the segment's rows go
  static constexpr int kOffMisc = kOffRow + N * 8;       // abort flag, TMEM address
  static constexpr int kSmem = kOffMisc + 16;
  static_assert(kSmem <= (KD == 64 ? 113 : 227) * 1024, "smem budget");
};

struct SegInfo {
  int live;    // 0: no more segments
  int j0, m;   // first key tile, key tiles
  int tok0;    // first query token of the item within the request
  int req, qst, qlen, klen, kbase, kh;
  int slot;    // -1: whole, else its slot of the partials
  int pad[5];
};
static_assert(sizeof(SegInfo) == 64, "segment record");

// Barrier of the softmax threads that also tells whether any / all of them say so.
__device__ __forceinline__ bool sync_or(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, 1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "n"(kSoft)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ bool sync_and(bool v) { return !sync_or(!v); }

// Maximum over the warp.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The N sums over the warp's lanes of v[0 .. N - 1]: lane c ends with the sum
// of column c % N.
template <int N>
__device__ __forceinline__ float column_sum(float (&v)[N], int lane) {
#pragma unroll
  for (int w = N / 2; w >= 1; w >>= 1) {
    const bool up = (lane & w) != 0;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float give = up ? v[i] : v[i + w], keep = up ? v[i + w] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
    }
  }
  float s = v[0];
#pragma unroll
  for (int w = N; w < 32; w <<= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
  return s;
}

// N consecutive TMEM columns of this warp's lanes.
__device__ __forceinline__ void tmem_load(uint32_t t, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(t));
}
__device__ __forceinline__ void tmem_load(uint32_t t, uint32_t (&r)[16]) { tmem_ld16_nowait(t, r); }
__device__ __forceinline__ void tmem_load(uint32_t t, uint32_t (&r)[32]) { tmem_ld32_nowait(t, r); }
__device__ __forceinline__ void tmem_store(uint32_t t, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(t), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t t, const uint32_t (&r)[16]) { tmem_st16(t, r); }
__device__ __forceinline__ void tmem_store(uint32_t t, const uint32_t (&r)[32]) { tmem_st32(t, r); }

// N: columns of the MMAs; NC: those that hold rows, the only ones that the
// softmax works on.  Items of at most 4 rows have NC = 4 (the least N of an MMA
// is 16): 64 single tokens of 32 heads over up to 2000 keys of 8 x 128 in 68.4
// us, with all 16 columns 76.5; 24 over 1500 keys of 20 x 64 in 47.6 and 49.3.
template <typename T, int KD, int N, int NC>
__global__ void __launch_bounds__(kThreads, KD == 64 ? 2 : 1) fd_attn_rows_kernel(const __grid_constant__ MmaParams mp) {
  typedef Geo<KD, N> Ge;
  constexpr int kTile = Ge::kTile, kRingK = Ge::kRingK, kRingV = Ge::kRingV;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdQK = instr_desc(kBF16, false, kKT, N);
  constexpr uint32_t kIdPV = instr_desc(kBF16, true, 128, N);  // V: MN-major A
  const AttnParams& p = mp.a;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + Ge::kOffBar);
  uint64_t* k_empty = k_full + kRingK;     // MMA commit after the q.K^T that read it
  uint64_t* v_full = k_empty + kRingK;
  uint64_t* v_empty = v_full + kRingV;     // MMA commit after the P.V that read it
  uint64_t* q_full = v_empty + kRingV;     // [2]
  uint64_t* q_empty = q_full + 2;          // [2] MMA commit after a segment's last q.K^T
  uint64_t* s_full = q_empty + 2;          // [2] MMA commit: S of a tile
  uint64_t* p_full = s_full + 2;           // [2] the four softmax warps wrote P
  uint64_t* pv_done = p_full + 2;          // MMA commit after each P.V
  uint64_t* o_full = pv_done + 1;          // MMA commit after a segment's last P.V
  // the four softmax warps are done with a segment that has keys.  One without
  // is left out: its softmax awaits nothing of the MMA thread's, which could
  // then find this barrier a phase past the one that it waits for
  uint64_t* o_empty = o_full + 1;
  uint64_t* seg_full = o_empty + 1;        // [kSegs]
  uint64_t* seg_empty = seg_full + kSegs;  // [kSegs]
  uint64_t* drain = seg_empty + kSegs;
  SegInfo* segs = reinterpret_cast<SegInfo*>(smem + Ge::kOffSeg);
  float* red = reinterpret_cast<float*>(smem + Ge::kOffRed);
  float* m_sh = reinterpret_cast<float*>(smem + Ge::kOffM);
  float* f_sh = m_sh + N;
  int64_t* row_sh = reinterpret_cast<int64_t*>(smem + Ge::kOffRow);
  volatile int* misc = reinterpret_cast<volatile int*>(smem + Ge::kOffMisc);  // [0] abort, [1] TMEM address

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  griddep_launch_dependents();  // the combine's CTAs may start, and wait for this grid's end
  prefetch_maps(mp, (int)threadIdx.x - 64);
  init_barriers(k_full, Ge::kNumBars, [&](int i) -> uint32_t {
    uint64_t* b = k_full + i;
    return (b >= p_full && b < pv_done) || b == o_empty ? 4 : b >= seg_empty && b < drain ? kSegReaders : 1;
  });
  if (threadIdx.x == 0) {
    p.cuts[cta].nparts = 0;
    misc[0] = 0;
  }
  // rows of the Q buffers that no load writes (behind the tile's tokens) stay 0
  for (int x = threadIdx.x; x < 2 * Ge::kQ / 16; x += kThreads) sts128(smem + Ge::kOffQ + 16 * x, make_uint4(0, 0, 0, 0));
  fence_proxy_async_smem();
  Walk walk(p);
  static_assert(sizeof(Walk::Scratch) <= 4 * N * 4 + 512, "scratch of the schedule");
  if (!walk.init<kThreads>(reinterpret_cast<Walk::Scratch*>(red), cta, kMinPer)) return;  // all threads alike
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(smem + Ge::kOffMisc + 4)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)misc[1];

  if (warp == kWarpSched) {
    // ------------------------------------------------ schedule and Q tiles
    int nseg = 0, nq = 0;
    bool ok = true;
    Walk::Seg g;
    while (ok) {
      const bool more = walk.next(g);
      const Req rq = walk.rq;
      const int ss = nseg % kSegs;
      if (nseg >= kSegs)
        ok = __all_sync(0xffffffffu, wait_or_abort(&seg_empty[ss], (uint32_t)(nseg / kSegs - 1) & 1u, misc, p.err));
      if (!ok) break;
      const int tok0 = g.tile0 * p.tq;
      if (lane == 0) {
        SegInfo& i = segs[ss];
        i.live = more;
        if (more) {
          i.j0 = g.j0;
          i.m = g.j1 - g.j0;
          i.tok0 = tok0;
          i.req = walk.r;
          i.qst = rq.qst;
          i.qlen = rq.qlen;
          i.klen = rq.klen;
          i.kbase = rq.kbase;
          i.kh = g.kh;
          i.slot = g.whole ? -1 : 2 * cta + (g.j0 > 0 ? 0 : 1);
        }
        mbar_arrive(&seg_full[ss]);
        if (more && g.nparts > 0) p.cuts[cta] = Cut{g.nparts, rq.qst + tok0, min(p.tq, rq.qlen - tok0) * p.G, g.kh};
      }
      __syncwarp();
      ++nseg;
      if (!more) break;
      if (g.j0 >= g.j1) continue;  // no key is seen: the softmax warps write zeros
      const int qb = nq & 1;
      if (nq >= 2 && !__all_sync(0xffffffffu, wait_or_abort(&q_empty[qb], (uint32_t)(nq / 2 - 1) & 1u, misc, p.err))) {
        ok = false;
        break;
      }
      ++nq;
      unsigned char* sq = smem + Ge::kOffQ + qb * Ge::kQ;
      if (mp.q_tma) {
        if (lane == 0) {
          mbar_expect_tx(&q_full[qb], (uint32_t)(Ge::kPanels * p.tq * p.G * 128));
          for (int c = 0; c < Ge::kPanels; ++c)
            tma_load_4d(sq + c * N * 128, &mp.tmap_q, 64 * c, g.kh * p.G, rq.qst + tok0, 0, &q_full[qb], 0ull);
          mbar_arrive(&q_full[qb]);
        }
      } else {
        load_q<KD>(p, sq, N * 128, g.kh, rq.qst + tok0, min(p.tq, rq.qlen - tok0), lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[qb]);
      }
    }
    if (!ok) misc[0] = 1;
    // no copy of this warp is in flight when the CTA ends
    for (int b = 0; b < 2 && b < nq; ++b) mbar_wait(&q_full[b], (uint32_t)((nq - 1 - b) / 2) & 1u, p.err);
  } else if (warp == kWarpK || warp == kWarpV) {
    // ------------------------------------------------ K or V tiles
    const bool is_v = warp == kWarpV;
    const int ring = is_v ? kRingV : kRingK;
    uint64_t* const full = is_v ? v_full : k_full;
    uint64_t* const empty = is_v ? v_empty : k_empty;
    unsigned char* const slots = smem + (is_v ? Ge::kOffV : 0);
    const uint64_t pol = l2_evict_first_policy();
    int st = 0, nseg = 0;
    uint32_t tiles = 0, ph = 0;
    // the next segment, and the block ids of its first tile on their way:
    // taken before the last tile of the one before is loaded
    SegInfo seg;
    int first_id = -1;
    auto take = [&]() {
      const int ss = nseg % kSegs;
      if (!__all_sync(0xffffffffu, wait_or_abort(&seg_full[ss], (uint32_t)(nseg / kSegs) & 1u, misc, p.err)))
        return false;
      seg = segs[ss];
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[ss]);
      ++nseg;
      first_id = seg.live && seg.m > 0 ? box_block(mp, is_v, seg.kbase, seg.klen, seg.j0, lane) : -1;
      return true;
    };
    bool ok = take();
    while (ok && seg.live) {
      const SegInfo i = seg;
      int id = first_id;
      if (i.m == 0) ok = take();
      for (int j = i.j0; j < i.j0 + i.m; ++j) {
        const bool last = j + 1 == i.j0 + i.m;
        const int id_next = last ? -1 : box_block(mp, is_v, i.kbase, i.klen, j + 1, lane);
        if (last) ok = take();
        if (ok && tiles >= (uint32_t)ring)
          ok = __all_sync(0xffffffffu, wait_or_abort(&empty[st], ph ^ 1u, misc, p.err));
        if (!ok) break;
        load_tile<KD>(mp, is_v, slots + st * kTile, &full[st], j, i.req, i.kbase, i.klen, i.kh, id, lane, pol);
        id = id_next;
        ++tiles;
        if (++st == ring) {
          st = 0;
          ph ^= 1u;
        }
      }
    }
    if (!ok) misc[0] = 1;
    // no copy of this warp is in flight when the CTA ends
    for (uint32_t s = 0; s < (uint32_t)ring && s < tiles; ++s) {
      const uint32_t last = s + ring * ((tiles - 1 - s) / ring);
      mbar_wait(&full[s], (last / ring) & 1u, p.err);
    }
  } else if (warp == kWarpMma) {
    // ------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t base = smem_u32(smem) >> 4;
      // 16-byte units: 16 keys of a K/V tile on, and from its first 64 dims to
      // the second; heads of 64 dims have V's twice (rows 64 .. 127 of O^T are not read)
      const uint32_t two = (uint32_t)mp.group * 2 >> 4, panel = (uint32_t)mp.panel >> 4;
      const uint32_t lbo = KD == 128 ? panel : 0u;
      const uint32_t q_hi = desc_hi(1024), kv_hi = desc_hi((uint32_t)mp.group);
      int ks_ = 0, vs_ = 0, nq = 0;  // nq: segments with keys
      uint32_t kp = 0, vp = 0, pp = 0;  // ring phases; parities of p_full's two buffers
      bool ok = true;
      for (int nseg = 0; ok; ++nseg) {
        const int ss = nseg % kSegs;
        ok = poll_or_abort(&seg_full[ss], (uint32_t)(nseg / kSegs) & 1u, misc, p.err);
        if (!ok) break;
        const int live = segs[ss].live, m = segs[ss].m;
        mbar_arrive(&seg_empty[ss]);
        if (!live) break;
        const int qb = nq & 1;
        const uint32_t q_lo = base + (uint32_t)((Ge::kOffQ + qb * Ge::kQ) >> 4) + (1u << 16);
        auto qk = [&](int t) {  // q.K^T of tile t
          if (!poll_or_abort(&k_full[ks_], kp, misc, p.err)) return false;
          tc_fence_after();
          const uint32_t k_lo = base + (uint32_t)((ks_ * kTile) >> 4) + (1u << 16);
#pragma unroll
          for (int ks = 0; ks < KD / 16; ++ks)
            umma_f16_lo(tmem + 32 * (t & 1), k_lo + (uint32_t)(ks >> 2) * panel + (uint32_t)((ks & 3) * 32 >> 4), kv_hi,
                        q_lo + (uint32_t)(((ks >> 2) * (N * 128) + (ks & 3) * 32) >> 4), q_hi, kIdQK, ks > 0 ? 1u : 0u);
          umma_commit(&s_full[t & 1]);
          umma_commit(&k_empty[ks_]);
          advance<kRingK>(ks_, kp);
          if (t == m - 1) umma_commit(&q_empty[qb]);
          return true;
        };
        if (m > 0) {
          ok = poll_or_abort(&q_full[qb], (uint32_t)(nq / 2) & 1u, misc, p.err);
          ++nq;
          ok = ok && qk(0) && (m < 2 || qk(1));
        }
        // the O of the segment with keys before has been read
        if (ok && m > 0 && nq > 1) ok = poll_or_abort(o_empty, (uint32_t)(nq - 2) & 1u, misc, p.err);
        for (int t = 0; ok && t < m; ++t) {
          const int h = t & 1;
          ok = poll_or_abort(&v_full[vs_], vp, misc, p.err) && poll_or_abort(&p_full[h], (pp >> h) & 1u, misc, p.err);
          if (!ok) break;
          pp ^= 1u << h;
          tc_fence_after();
          const uint32_t v_lo = base + (uint32_t)((Ge::kOffV + vs_ * kTile) >> 4) + (lbo << 16);
          const uint32_t p_lo = base + (uint32_t)((Ge::kOffP + h * Ge::kP) >> 4) + (1u << 16);
#pragma unroll
          for (int ks = 0; ks < kKT / 16; ++ks)
            umma_f16_lo(tmem + kOcol, v_lo + (uint32_t)ks * two, kv_hi,
                        p_lo + (uint32_t)(((ks >> 2) * (N * 128) + (ks & 3) * 32) >> 4), q_hi, kIdPV,
                        (t > 0 || ks > 0) ? 1u : 0u);
          umma_commit(pv_done);
          if (t + 2 < m) ok = qk(t + 2);
          umma_commit(&v_empty[vs_]);
          advance<kRingV>(vs_, vp);
        }
        if (ok && m > 0) umma_commit(o_full);
      }
      if (!ok) misc[0] = 1;
      umma_commit(drain);  // all MMAs complete before TMEM is released
      mbar_wait(drain, 0u, p.err);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ softmax: one key per thread, then one dim
    const int tid = threadIdx.x;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    uint32_t ph = 0;  // phase parities of s_full (bits 0, 1), o_full (2), pv_done of the tile at hand (3)
    bool ok = true;
    for (int nseg = 0;; ++nseg) {
      const int ss = nseg % kSegs;
      ok = sync_and(wait_or_abort(&seg_full[ss], (uint32_t)(nseg / kSegs) & 1u, misc, p.err));
      if (!ok) break;
      const SegInfo& seg = segs[ss];  // stays until this segment's end
      if (!seg.live) break;
      const int m_tiles = seg.m;
      // column n (token tok0 + n / G) sees key j: j <= first + n / G, so n >= (j - first) G
      const int first = p.bt != nullptr ? seg.klen - seg.qlen + seg.tok0 : seg.klen - 1;
      float l[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) l[n] = 0.f;
      for (int t = 0; t < m_tiles; ++t) {
        const int h = t & 1;
        ok = wait_or_abort(&s_full[h], (ph >> h) & 1u, misc, p.err);
        ph ^= 1u << h;
        __syncwarp();
        tc_fence_after();
        uint32_t s[NC];
        tmem_load(tmem + lanes + 32 * h, s);
        tmem_wait_ld();
        const int key0 = (seg.j0 + t) * kKT;
        if (key0 + kKT - 1 > first) {
          const int over = key0 + tid - first;
          const int from = over <= 0 ? 0 : p.bt != nullptr ? over * p.G : NC;
#pragma unroll
          for (int n = 0; n < NC; ++n)
            if (n < from) s[n] = __float_as_uint(-INFINITY);
        }
        // does some score pass its column's reference by more than 2^8?
        bool past = t == 0;
        if (t > 0) {
#pragma unroll
          for (int n = 0; n < NC; n += 4) {
            const float4 m = *reinterpret_cast<const float4*>(m_sh + n);
            past |= fmaf(__uint_as_float(s[n]), p.sl2, -m.x) > 8.f;
            past |= fmaf(__uint_as_float(s[n + 1]), p.sl2, -m.y) > 8.f;
            past |= fmaf(__uint_as_float(s[n + 2]), p.sl2, -m.z) > 8.f;
            past |= fmaf(__uint_as_float(s[n + 3]), p.sl2, -m.w) > 8.f;
          }
        }
        if (sync_or(past || !ok)) {
          // O takes the earlier tiles: P.V of the last one may still run (that
          // of the one before it is done: this S's q.K^T was issued behind it,
          // so the phase before the awaited one is known to have passed)
          ok = ok && (t == 0 || wait_or_abort(pv_done, ((ph >> 3) & 1u) ^ 1u, misc, p.err));
          __syncwarp();
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            const float mx = warp_max(__uint_as_float(s[n]));
            if (lane == 0) red[warp * NC + n] = mx;
          }
          if (!sync_and(ok)) {
            ok = false;
            break;
          }
          if (tid < NC) {
            const float mx = fmaxf(fmaxf(red[tid], red[NC + tid]), fmaxf(red[2 * NC + tid], red[3 * NC + tid])) * p.sl2;
            const float old = t == 0 ? -INFINITY : m_sh[tid];
            const bool set = old == -INFINITY, grow = !set && mx > old + 8.f;
            f_sh[tid] = grow ? exp2f(old - mx) : 1.f;
            m_sh[tid] = set || grow ? mx : old;
          }
          sync_or(false);
          if (t > 0) {
            tc_fence_after();
            uint32_t o[NC];
            tmem_load(tmem + lanes + kOcol, o);
            tmem_wait_ld();
#pragma unroll
            for (int n = 0; n < NC; ++n) {
              l[n] *= f_sh[n];
              o[n] = __float_as_uint(__uint_as_float(o[n]) * f_sh[n]);
            }
            tmem_store(tmem + lanes + kOcol, o);
            tmem_wait_st();
          }
        }
        // P: row n of the B operand, key `tid`
        unsigned char* pb = smem + Ge::kOffP + h * Ge::kP + (tid >> 6) * (N * 128) + (tid & 7) * 2;
        const int ch = (tid & 63) >> 3;
#pragma unroll
        for (int n = 0; n < NC; n += 4) {
          const float4 m4 = *reinterpret_cast<const float4*>(m_sh + n);
          const float m[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = ex2_approx(fmaf(__uint_as_float(s[n + i]), p.sl2, m[i] == -INFINITY ? 0.f : -m[i]));
            l[n + i] += e;
            *reinterpret_cast<T*>(pb + swz(n + i, ch)) = Dt<T>::narrow(e);
          }
        }
        fence_proxy_async_smem();  // P before the tensor cores read it
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[h]);
        ph ^= 8u;
      }
      if (!ok) break;
      // the segment's end: sums over the keys' threads, then rows
      if (m_tiles > 0) {
        ok = wait_or_abort(o_full, (ph >> 2) & 1u, misc, p.err);
        ph ^= 4u;
        __syncwarp();
      }
      const float sum = column_sum<NC>(l, lane);
      if (lane < NC) red[warp * NC + lane] = sum;
      if (!sync_and(ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int rows = min(p.tq, seg.qlen - seg.tok0) * p.G;
      const int slot = seg.slot;
      if (tid < NC) {
        const float lt = red[tid] + red[NC + tid] + red[2 * NC + tid] + red[3 * NC + tid];
        const float mt = m_tiles > 0 ? m_sh[tid] : -INFINITY;
        f_sh[tid] = slot >= 0 ? 1.f : row_inv(lt);
        const int t = tid / p.G, h = seg.kh * p.G + tid - t * p.G;
        const int64_t tok = seg.qst + seg.tok0 + t;
        row_sh[tid] = tok * p.o_st + h * p.o_sh;
        if (tid < rows) {
          if (slot >= 0)
            reinterpret_cast<float2*>(p.part_ml)[(int64_t)slot * NC + tid] = make_float2(mt, lt);
          else if (p.lse != nullptr)
            p.lse[h * p.lse_sh + tok * p.lse_st] = row_lse(mt, lt);
        }
      }
      uint32_t o[NC];
      if (m_tiles > 0) {
        tmem_load(tmem + lanes + kOcol, o);
        tmem_wait_ld();
      }
      tc_fence_before();
      sync_or(false);
      if (lane == 0) {  // O and the segment's record are read
        if (m_tiles > 0) mbar_arrive(o_empty);
        mbar_arrive(&seg_empty[ss]);
      }
      // thread `tid` has dim `tid` of every row
      if (tid < p.D && m_tiles > 0) {
        if (slot >= 0) {
          float* pp = p.part_o + (((int64_t)slot * (p.D / 4) + (tid >> 2)) * NC) * 4 + (tid & 3);
#pragma unroll
          for (int n = 0; n < NC; ++n)
            if (n < rows) pp[4 * n] = __uint_as_float(o[n]);
        } else {
          unsigned char* po = p.out + tid * 2;
#pragma unroll
          for (int n = 0; n < NC; n += 4) {
            const float4 f = *reinterpret_cast<const float4*>(f_sh + n);
            const float w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n + i < rows)
                *reinterpret_cast<T*>(po + row_sh[n + i]) = Dt<T>::narrow(__uint_as_float(o[n + i]) * w[i]);
          }
        }
      } else if (tid < p.D) {  // no key: zeros (never a partial)
#pragma unroll 1
        for (int n = 0; n < rows; ++n) *reinterpret_cast<T*>(p.out + tid * 2 + row_sh[n]) = Dt<T>::narrow(0.f);
      }
    }
    if (!ok) misc[0] = 1;
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpMma)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

template <typename T, int KD, int N, int NC>
int launch(const MmaParams& mp, cudaStream_t s) {
  const void* kern = reinterpret_cast<const void*>(fd_attn_rows_kernel<T, KD, N, NC>);
  static unsigned long long done = 0;
  const int st = fdh::ensure_smem(kern, Geo<KD, N>::kSmem, &done);
  if (st != FD_OK) return st;
  return fdh::launch_maybe_pdl(kern, dim3((unsigned)mp.a.ctas), dim3(kThreads), Geo<KD, N>::kSmem, s, false, mp,
                               "fd_attn_rows_kernel launch");
}

template <typename T>
int launch_for(const MmaParams& mp, int rows, cudaStream_t s) {
  if (mp.a.D <= 64)
    return rows == 4    ? launch<T, 64, 16, 4>(mp, s)
           : rows == 16 ? launch<T, 64, 16, 16>(mp, s)
                        : launch<T, 64, 32, 32>(mp, s);
  return rows == 4    ? launch<T, 128, 16, 4>(mp, s)
         : rows == 16 ? launch<T, 128, 16, 16>(mp, s)
                      : launch<T, 128, 32, 32>(mp, s);
}

}  // namespace rw

int rows_launch(AttnParams& p, const fd_attn_args* a, int rows, cudaStream_t s) {
  int dev = 0, sms = 0;
  int st = fdh::device_sms(&dev, &sms);
  if (st != FD_OK) return st;
  const int N = rows <= 4 ? 4 : rows <= 16 ? 16 : 32;  // rows of an item
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  p.ctas = sms * (p.D <= 64 ? 2 : 1);
  if (p.ctas > rw::kMaxCtas) p.ctas = rw::kMaxCtas;
  p.cuts = reinterpret_cast<Cut*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + rw::kMaxCtas * sizeof(Cut));
  p.part_o = p.part_ml + 2 * 2 * (size_t)rw::kMaxCtas * N;
  p.tq = N / p.G;
  p.snap = whole_items(a, p.ctas, N, mm::kKT, mm::kWhole);
  mm::MmaParams mp{};
  mp.a = p;
  mm::encode_maps(mp, a);
  st = a->dtype == FD_DTYPE_BF16 ? rw::launch_for<__nv_bfloat16>(mp, N, s) : rw::launch_for<__half>(mp, N, s);
  if (st != FD_OK || p.snap) return st;
  return combine_launch(p, a->dtype, N, s);
}

}  // namespace at
}  // namespace fdk
