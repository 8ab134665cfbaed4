// Attention weight per cached key on the 5th-generation tensor cores
// (tcgen05): fp16 and bf16, head sizes 64 to 128.
//
//   S^T [128 keys x N] = K . Q^T,   w[key] += sum_n 2^(scale log2(e) S - lse_n log2(e))
//
// K lies in shared memory as the MMA's A operand, the query rows (token x G +
// head) are its N columns, so a thread of the epilogue has one key and adds up
// what its columns give, over all chunks of queries, in registers.  An item is
// two such key tiles, each with its own four epilogue warps and TMEM buffers:
// a chunk of queries that is fetched once serves 256 keys.  With at most 32
// query rows (N = 16 or 32: single tokens, draft tokens) a call is bound by the
// bytes of K, and shared memory is a ring of K tiles; with more (N = 128) by
// the exponentials, and it is a ring of query chunks beside two items' K.
//
// Warps: the epilogue's first, four per key tile, and with N = 128 another four
// per tile, the two groups taking turns at the steps (two warps per scheduler
// leave the SFU idle while both wait; their sums are joined at the item's end);
// then one for the schedule, the query chunks and their lse (as many steps ahead
// as there are slots), one per key tile that loads K, and one per key tile (with
// N = 128 one for both) whose first thread issues the MMAs.  A STEP is one chunk against one item; its record goes
// through a ring to all roles.  Every wait is bounded, and a role
// that gives up raises the CTA's abort flag for the others.
//
// Measured: 32 single tokens of 32 heads over 512 to 8192 keys of 8 heads x 128
// in 56 us (342 MB, 6.1 TB/s; one warp that issues for both key tiles: 58, one
// that loads both: 100).  2 x 2048
// tokens over up to 12288 in 420 us (797 TFLOP/s): 1.3 G powers of two, of which
// the SFUs take 16 per SM and clock, 290 us at 1.9 GHz; they are busy for three
// quarters of the time.  Tried and slower: an eighth to three eighths of the powers by
// a polynomial on the FMA pipe (510 to 630 us: the warps wait for their own
// chains, not for the SFU), one group of warps with all 128 scores in registers
// (512), TMEM loads of 16 columns (556), both groups' step records read at once
// (503).

#include <type_traits>

#include "fd_attn_mma.cuh"
#include "fd_keyw.cuh"

namespace fdk {
namespace kw {
namespace mm {

using namespace at::mm;

constexpr int kTiles = 2;             // key tiles of an item
constexpr int kKeys = kTiles * kKT;
static_assert(kKeys == kMaxKeys, "partials per item");
constexpr int kFixed = 2;             // an item's fixed cost in chunks
constexpr int kMinPer = 3;            // least positions of a CTA

typedef Walk<kKeys, kFixed, false> MmaWalk;

struct KwMmaParams {
  at::mm::MmaParams m;  // m.a is k.a
  KwParams k;
};

template <int KD, int N>
struct Geo {
  static constexpr int kGroups = N <= 32 ? 1 : 2;        // epilogue warpgroups of a key tile
  static constexpr int kSumWarps = 4 * kTiles * kGroups;
  static constexpr int kWarpSched = kSumWarps, kWarpK = kSumWarps + 1, kWarpMma = kWarpK + kTiles;
  // one issuer of MMAs per key tile; with N = 128 one for both (21 warps leave a thread 80 registers: 607 us instead of
  // 420; one warp less for K instead: 412, but short calls take 16.7 instead of 13.6)
  static constexpr int kMmaWarps = N <= 32 ? kTiles : 1;
  static constexpr int kThreads = (kWarpMma + kMmaWarps) * 32;
  static constexpr int kSteps = N <= 32 ? 8 : 4;         // steps in flight between the roles
  static constexpr int kStepReaders = kSumWarps + kTiles + kMmaWarps;
  static constexpr int kPanels = KD / 64;
  static constexpr int kTile = kPanels * kPanel;
  static constexpr int kItem = kTiles * kTile;
  static constexpr int kRingK = (N <= 32 ? 3 : 2) * (KD == 64 ? 2 : 1);
  static constexpr int kRingQ = N <= 32 ? 4 : 3;
  static constexpr int kBufs = N <= 32 ? 4 : 2;          // TMEM buffers of a key tile
  static constexpr int kCols = N <= 32 ? 32 : N;         // columns of one
  static constexpr int kTmem = kTiles * kBufs * kCols;   // 256 or 512
  static constexpr int kQ = kPanels * N * 128;
  static constexpr int kOffQ = kRingK * kItem;
  static constexpr int kOffLse = kOffQ + kRingQ * kQ;    // [kRingQ][N] -lse log2(e)
  static constexpr int kOffStep = kOffLse + kRingQ * (N < 32 ? 32 : N) * 4;
  static constexpr int kOffJoin = kOffStep + kSteps * 48;  // [kTiles][kKT] the second groups' sums
  static constexpr int kOffBar = kOffJoin + (kGroups - 1) * kKeys * 4;
  // k full [ring][tiles], k empty, q full, q empty, s full [bufs][tiles], s empty [bufs][tiles], step full, step empty,
  // join full, empty [tiles], drain [MMA warps]
  static constexpr int kNumBars = kRingK * (kTiles + 1) + 2 * kRingQ + 2 * kBufs * kTiles + 2 * kSteps + 2 * kTiles + kMmaWarps;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;  // abort flag, TMEM address
  static constexpr int kSmem = kOffMisc + 16;
  static_assert(kSmem <= 227 * 1024, "smem budget");
  static_assert(sizeof(MmaWalk::Scratch) <= kRingQ * (N < 32 ? 32 : N) * 4, "scratch of the schedule");
};

// Whether a step is the first or last of its segment (K), and the first with a
// chunk of queries (Q: the slot of the chunk before is done with the steps
// before).  kMute: not every column of the chunk gives something (no row, or
// one whose lse is infinite).  Flags 0: no more steps.
enum StepFlag { kLive = 1, kNewK = 2, kLastK = 4, kNewQ = 8, kMute = 16 };
struct Step {
  int flags;
  int r, kh, kt, kbase;
  int first, last;   // the last key that the chunk's first, and its last token sees
  int rows;          // of the chunk
  int qlen, klen;
  int slot;          // -1: whole, else its slot of the partials
  int pad;
};
static_assert(sizeof(Step) == 48, "step record");

// Wait for this thread's TMEM loads.  The registers are operands, so that
// nothing that reads them is moved ahead of it.
__device__ __forceinline__ void wait_loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ void wait_loaded(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// What 32 scores of a key add up to; the e-th counts if see(e).  skip(c): none
// of scores c .. c + 3 counts for any key of the warp.
template <typename See, typename Skip>
__device__ __forceinline__ void add_up(const uint32_t (&s)[32], const float* neg, f2_t sl2, f2_t (&acc)[2], See see, Skip skip) {
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    if (skip(c)) break;
    const ulonglong2 ng = *reinterpret_cast<const ulonglong2*>(neg + c);
    const f2_t x0 = f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sl2, ng.x);
    const f2_t x1 = f2_fma(f2_pack(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), sl2, ng.y);
    float e[4];
    f2_unpack(x0, e[0], e[1]);
    f2_unpack(x1, e[2], e[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = at::ex2_approx(e[i]);
      if (!see(c + i)) e[i] = 0.f;
    }
    acc[0] = f2_add(acc[0], f2_pack(e[0], e[1]));
    acc[1] = f2_add(acc[1], f2_pack(e[2], e[3]));
  }
}

// Bits from .. to - 1 of a word.
__device__ __forceinline__ uint32_t bits_of(int from, int to) {
  const uint32_t below_to = to >= 32 ? ~0u : to > 0 ? (1u << to) - 1u : 0u;
  const uint32_t below_from = from >= 32 ? ~0u : from > 0 ? (1u << from) - 1u : 0u;
  return below_to & ~below_from;
}

template <typename T, int KD, int N>
__global__ void __launch_bounds__(Geo<KD, N>::kThreads, 1) fd_keyw_mma_kernel(const __grid_constant__ KwMmaParams kp) {
  typedef Geo<KD, N> Ge;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdQK = instr_desc(kBF16, false, kKT, N);
  constexpr int kTile = Ge::kTile, kRingK = Ge::kRingK, kRingQ = Ge::kRingQ, kBufs = Ge::kBufs, kSteps = Ge::kSteps;
  constexpr int kSumWarps = Ge::kSumWarps, kWarpK = Ge::kWarpK, kGroups = Ge::kGroups;
  constexpr int kLseRow = N < 32 ? 32 : N;
  const at::mm::MmaParams& mp = kp.m;
  const AttnParams& p = mp.a;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + Ge::kOffBar);  // [kRingK][kTiles]
  uint64_t* k_empty = k_full + kRingK * kTiles;  // [kRingK] MMA commits after the item's last step
  uint64_t* q_full = k_empty + kRingK;           // [kRingQ]
  uint64_t* q_empty = q_full + kRingQ;           // [kRingQ] MMA commits when the next chunk begins, and the epilogue warps
  uint64_t* s_full = q_empty + kRingQ;           // [kBufs][kTiles] MMA commit
  uint64_t* s_empty = s_full + kBufs * kTiles;   // [kBufs][kTiles] four epilogue warps have the scores
  uint64_t* step_full = s_empty + kBufs * kTiles;
  uint64_t* step_empty = step_full + kSteps;
  uint64_t* join_full = step_empty + kSteps;     // [kTiles] four warps of the second group wrote their sums
  uint64_t* join_empty = join_full + kTiles;     // [kTiles] four warps of the first have read them
  uint64_t* drain = join_empty + kTiles;         // [kMmaWarps]
  Step* steps = reinterpret_cast<Step*>(smem + Ge::kOffStep);
  float* lse_sh = reinterpret_cast<float*>(smem + Ge::kOffLse);
  volatile int* misc = reinterpret_cast<volatile int*>(smem + Ge::kOffMisc);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  griddep_launch_dependents();
  prefetch_maps(mp, (int)threadIdx.x - 64);
  init_barriers(k_full, Ge::kNumBars, [&](int i) -> uint32_t {
    uint64_t* b = k_full + i;
    if (b >= k_empty && b < q_full) return Ge::kMmaWarps;
    if (b >= q_empty && b < s_full) return Ge::kMmaWarps + kSumWarps;
    if (b >= s_empty && b < step_full) return 4;
    if (b >= join_full && b < drain) return 4;
    return b >= step_empty && b < join_full ? Ge::kStepReaders : 1;
  });
  if (threadIdx.x == 0) {
    if (kp.k.cuts != nullptr) kp.k.cuts[cta].nparts = 0;
    misc[0] = 0;
  }
  MmaWalk walk(p);
  if (!walk.init<Ge::kThreads>(reinterpret_cast<MmaWalk::Scratch*>(lse_sh), cta, kMinPer)) return;  // all threads alike
  if (warp == Ge::kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(smem + Ge::kOffMisc + 4)),
                 "r"(Ge::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)misc[1];

  if (warp == Ge::kWarpSched) {
    // ------------------------------------------------ schedule, query chunks and their lse
    constexpr int kPer = kLseRow / 32;  // columns per lane
    int col_t[kPer], col_h[kPer];       // token and head of each
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      col_t[i] = (32 * i + lane) / p.G;
      col_h[i] = 32 * i + lane - col_t[i] * p.G;
    }
    MmaWalk::Seg g;
    int left = 0, chunk = 0;            // chunks left of the segment, the next one
    int last_r = -1, last_kh = -1, last_chunk = -1;
    auto gen = [&](Step& s, Req& rq, float (&ls)[kPer]) {  // the next step, its lse on the way
      s.flags = kLive;
      if (left == 0) {
        if (!walk.next(g)) {
          s.flags = 0;
          return;
        }
        left = g.n;
        chunk = g.c0;
        s.flags |= kNewK;
        if (g.nparts > 0 && lane == 0) kp.k.cuts[cta] = Cut{g.nparts, g.r, g.kh, g.kt};
      }
      rq = walk.rq;
      if (--left == 0) s.flags |= kLastK;
      s.r = g.r;
      s.kh = g.kh;
      s.kt = g.kt;
      s.kbase = rq.kbase;
      const int tok0 = chunk * p.tq, ntok = min(p.tq, rq.qlen - tok0);
      rq.qst += tok0;  // the chunk's first row
      s.rows = ntok * p.G;
      s.first = rq.klen - rq.qlen + tok0;
      s.last = s.first + ntok - 1;
      s.qlen = rq.qlen;
      s.klen = rq.klen;
      s.slot = g.whole ? -1 : 2 * cta + (g.head ? 1 : 0);
      if (g.r != last_r || g.kh != last_kh || chunk != last_chunk) {
        s.flags |= kNewQ;
        const float* at = p.lse + (int64_t)(s.kh * p.G) * p.lse_sh + (int64_t)rq.qst * p.lse_st;
#pragma unroll
        for (int i = 0; i < kPer; ++i) ls[i] = 32 * i + lane < s.rows ? at[col_h[i] * p.lse_sh + col_t[i] * p.lse_st] : 0.f;
      }
      last_r = g.r;
      last_kh = g.kh;
      last_chunk = chunk++;
    };
    Step cur;
    Req rq = {0, 0, 0, 0};
    float ls[kPer];
    int qs = -1, mute = 0;
    uint32_t nq = 0;
    bool ok = true;
    for (uint32_t i = 0; ok; ++i) {
      gen(cur, rq, ls);
      const int ss = i % kSteps;
      if (i >= kSteps)
        ok = __all_sync(0xffffffffu, wait_or_abort(&step_empty[ss], (i / kSteps - 1) & 1u, misc, p.err));
      if (!ok) break;
      if ((cur.flags & kNewQ) != 0) {
        qs = (int)(nq % kRingQ);
        if (nq >= (uint32_t)kRingQ)
          ok = __all_sync(0xffffffffu, wait_or_abort(&q_empty[qs], (nq / kRingQ - 1) & 1u, misc, p.err));
        if (!ok) break;
        ++nq;
        mute = 0;
#pragma unroll
        for (int x = 0; x < kPer; ++x) {  // a row that saw nothing gives nothing
          const bool none = isinf(ls[x]);
          lse_sh[qs * kLseRow + 32 * x + lane] = none ? -INFINITY : -ls[x] * kLog2e;
          if (__any_sync(0xffffffffu, none)) mute = kMute;
        }
        unsigned char* sq = smem + Ge::kOffQ + qs * Ge::kQ;
        if (mp.q_tma) {
          if (lane == 0) {
            mbar_expect_tx(&q_full[qs], (uint32_t)(Ge::kPanels * p.tq * p.G * 128));
            for (int x = 0; x < Ge::kPanels; ++x)
              tma_load_4d(sq + x * N * 128, &mp.tmap_q, 64 * x, cur.kh * p.G, rq.qst, 0, &q_full[qs],
                          l2_evict_normal_policy());
            mbar_arrive(&q_full[qs]);
          }
        } else {
          at::mm::load_q<KD>(p, sq, N * 128, cur.kh, rq.qst, cur.rows / p.G, lane);
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[qs]);
        }
      }
      if (cur.flags != 0) cur.flags |= cur.rows < N ? kMute : mute;
      if (lane == 0) steps[ss] = cur;
      __syncwarp();
      if (lane == 0) mbar_arrive(&step_full[ss]);
      if (cur.flags == 0) break;
    }
    if (!ok) misc[0] = 1;
    // no copy of this warp is in flight when the CTA ends: the last chunk of each slot
    for (uint32_t s = 0; s < (uint32_t)kRingQ && s < nq; ++s) {
      const uint32_t last = s + kRingQ * ((nq - 1 - s) / kRingQ);
      mbar_wait(&q_full[s], (last / kRingQ) & 1u, p.err);
    }
  } else if (warp >= kWarpK && warp < kWarpK + kTiles) {
    // ------------------------------------------------ K, key tile t of every item
    const int t = warp - kWarpK;
    const uint64_t pol = l2_evict_first_policy();
    uint32_t i = 0, items = 0;
    Step item, ahead;    // the item to load, and the one after it where it is known already:
    int id = -1, id_ahead = -1;  // their block ids are on the way
    auto read = [&](Step& to, int& ids) {  // step i, which has been published; whether an item begins or all end with it
      const int ss = i % kSteps;
      to = steps[ss];
      __syncwarp();
      if (lane == 0) mbar_arrive(&step_empty[ss]);
      ++i;
      if (to.flags != 0 && (to.flags & kNewK) == 0) return false;
      if (to.flags != 0) ids = box_block(mp, false, to.kbase, to.klen, to.kt * kTiles + t, lane);
      return true;
    };
    auto take = [&]() {  // the next item; false: given up
      do {
        if (!__all_sync(0xffffffffu, wait_or_abort(&step_full[i % kSteps], (i / kSteps) & 1u, misc, p.err))) return false;
      } while (!read(item, id));
      return true;
    };
    bool ok = take();
    while (ok && item.flags != 0) {
      const int ks = (int)(items % kRingK);
      if (items >= (uint32_t)kRingK)
        ok = __all_sync(0xffffffffu, wait_or_abort(&k_empty[ks], (items / kRingK - 1) & 1u, misc, p.err));
      if (!ok) break;
      ++items;
      // (not awaited: the step may wait for this item's products)
      const bool known = __all_sync(0xffffffffu, mbar_test_wait(&step_full[i % kSteps], (i / kSteps) & 1u)) && read(ahead, id_ahead);
      load_tile<KD>(mp, false, smem + ks * Ge::kItem + t * kTile, &k_full[ks * kTiles + t], item.kt * kTiles + t, item.r,
                    item.kbase, item.klen, item.kh, id, lane, pol);
      if (known) {
        item = ahead;
        id = id_ahead;
      } else {
        ok = take();
      }
    }
    if (!ok) misc[0] = 1;
    for (uint32_t s = 0; s < (uint32_t)kRingK && s < items; ++s) {
      const uint32_t last = s + kRingK * ((items - 1 - s) / kRingK);
      mbar_wait(&k_full[s * kTiles + t], (last / kRingK) & 1u, p.err);
    }
  } else if (warp >= Ge::kWarpMma) {
    // ------------------------------------------------ MMA issuer of key tiles t0 .. t0 + kMine - 1
    constexpr int kMine = kTiles / Ge::kMmaWarps;
    const int t0 = (warp - Ge::kWarpMma) * kMine;
    if (lane == 0) {
      const uint32_t base = smem_u32(smem) >> 4;
      const uint32_t panel = (uint32_t)mp.panel >> 4;
      const uint32_t q_hi = desc_hi(1024), kv_hi = desc_hi((uint32_t)mp.group);
      uint32_t items = 0, nq = 0;
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        const int ss = i % kSteps;
        ok = poll_or_abort(&step_full[ss], (i / kSteps) & 1u, misc, p.err);
        if (!ok) break;
        const int flags = steps[ss].flags;
        mbar_arrive(&step_empty[ss]);
        if (flags == 0) break;
        const bool new_k = (flags & kNewK) != 0, new_q = (flags & kNewQ) != 0;
        if (new_q && nq > 0) umma_commit(&q_empty[(nq - 1) % kRingQ]);
        items += new_k;
        nq += new_q;
        const int ks = (int)((items - 1) % kRingK), qs = (int)((nq - 1) % kRingQ), b = (int)(i % kBufs);
        if (new_q) ok = poll_or_abort(&q_full[qs], ((nq - 1) / kRingQ) & 1u, misc, p.err);
        const uint32_t q_lo = base + (uint32_t)((Ge::kOffQ + qs * Ge::kQ) >> 4) + (1u << 16);
#pragma unroll
        for (int t = t0; t < t0 + kMine; ++t) {
          if (ok && new_k) ok = poll_or_abort(&k_full[ks * kTiles + t], ((items - 1) / kRingK) & 1u, misc, p.err);
          if (ok && i >= kBufs) ok = poll_or_abort(&s_empty[b * kTiles + t], (i / kBufs - 1) & 1u, misc, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint32_t k_lo = base + (uint32_t)((ks * Ge::kItem + t * kTile) >> 4) + (1u << 16);
#pragma unroll
          for (int x = 0; x < KD / 16; ++x)
            umma_f16_lo(tmem + (t * kBufs + b) * Ge::kCols, k_lo + (uint32_t)(x >> 2) * panel + (uint32_t)((x & 3) * 32 >> 4), kv_hi,
                        q_lo + (uint32_t)(((x >> 2) * (N * 128) + (x & 3) * 32) >> 4), q_hi, kIdQK, x > 0 ? 1u : 0u);
          umma_commit(&s_full[b * kTiles + t]);
        }
        if (ok && (flags & kLastK) != 0) umma_commit(&k_empty[ks]);
      }
      if (!ok) misc[0] = 1;
      umma_commit(drain + t0 / kMine);  // all MMAs complete before TMEM is released
      mbar_wait(drain + t0 / kMine, 0u, p.err);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ epilogue: one key per thread
    const int t = (warp >> 2) % kTiles, grp = (warp >> 2) / kTiles;  // key tile, group
    const int row = (warp & 3) * 32;                                 // first key of the warp in its tile
    const uint32_t lanes = (uint32_t)row << 16;
    const f2_t sl2 = f2_pack(p.sl2, p.sl2);
    float* const joined = reinterpret_cast<float*>(smem + Ge::kOffJoin) + t * kKT + row + lane;
    uint32_t nq = 0, items = 0;
    f2_t acc[2] = {0ull, 0ull};
    int64_t id = -1;
    bool ok = true;
    for (uint32_t i = 0;; ++i) {
      const int ss = i % kSteps, b = (int)(i % kBufs);
      ok = __all_sync(0xffffffffu, wait_or_abort(&step_full[ss], (i / kSteps) & 1u, misc, p.err));
      if (!ok) break;
      const Step s = steps[ss];
      __syncwarp();
      if (lane == 0) mbar_arrive(&step_empty[ss]);
      if (s.flags == 0) break;
      if ((s.flags & kNewQ) != 0) {
        if (nq > 0 && lane == 0) mbar_arrive(&q_empty[(nq - 1) % kRingQ]);
        ++nq;
      }
      const int qs = (int)((nq - 1) % kRingQ);
      const int key0 = s.kt * kKeys + t * kKT + row, key = key0 + lane;
      if ((s.flags & kNewK) != 0) {
        acc[0] = acc[1] = 0ull;
        // (of a cut item the combine looks it up)
        if (grp == 0 && key < s.klen && s.slot < 0) id = p.bt[(int64_t)s.kbase * p.bt_stride + (int)((unsigned)key / (unsigned)p.BS)];
      }
      if (kGroups == 1 || (int)(i & 1u) == grp) {
        ok = __all_sync(0xffffffffu, wait_or_abort(&s_full[b * kTiles + t], (i / kBufs) & 1u, misc, p.err));
        if (!ok) break;
        tc_fence_after();
        // column n sees keys up to first + n / G
        const bool any = key0 < s.klen && key0 <= s.last;  // the warp alike
        const uint32_t ts = tmem + lanes + (uint32_t)((t * kBufs + b) * Ge::kCols);
        const float* neg = lse_sh + qs * kLseRow;
        if (any) {
          const int over = key - s.first;
          const int from = over > 0 ? over * p.G : 0;
          const bool masked = key0 + 31 > s.first || (s.flags & kMute) != 0;
          // rows with an infinite lse, as bits (that 2^-inf is 0 would not do: an infinite or NaN score makes it a NaN)
          auto muted = [&](int c) { return (s.flags & kMute) != 0 ? __ballot_sync(0xffffffffu, neg[32 * c + lane] == -INFINITY) : 0u; };
          if constexpr (N <= 32) {
            uint32_t v[32];
            if constexpr (N == 16) {
              uint32_t w[16];
              tmem_ld16_nowait(ts, w);
              wait_loaded(w);
#pragma unroll
              for (int x = 0; x < 32; ++x) v[x] = x < 16 ? w[x] : 0u;
            } else {
              tmem_ld32_nowait(ts, v);
              wait_loaded(v);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_empty[b * kTiles + t]);
            const uint32_t seen = bits_of(from, s.rows) & ~muted(0);
            add_up(v, neg, sl2, acc, [&](int e) { return (seen >> e & 1u) != 0u; }, [&](int c) { return c >= s.rows; });
          } else {
            uint32_t v[2][32];
            tmem_ld32_nowait(ts, v[0]);
#pragma unroll
            for (int c = 0; c < N / 32; ++c) {
              wait_loaded(v[c & 1]);
              if (c + 1 < N / 32) {
                tmem_ld32_nowait(ts + 32 * (c + 1), v[(c + 1) & 1]);
              } else {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_empty[b * kTiles + t]);
              }
              const auto no_skip = [](int) { return false; };
              if (masked) {
                const uint32_t seen = bits_of(from - 32 * c, s.rows - 32 * c) & ~muted(c);
                add_up(v[c & 1], neg + 32 * c, sl2, acc, [&](int e) { return (seen >> e & 1u) != 0u; }, no_skip);
              } else {
                add_up(v[c & 1], neg + 32 * c, sl2, acc, [](int) { return true; }, no_skip);
              }
            }
          }
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[b * kTiles + t]);
        }
      }
      if ((s.flags & kLastK) != 0) {
        float a0, a1, a2, a3;
        f2_unpack(acc[0], a0, a1);
        f2_unpack(acc[1], a2, a3);
        float w = (a0 + a1) + (a2 + a3);
        if constexpr (kGroups > 1) {
          if (grp == 1) {
            if (items > 0) ok = __all_sync(0xffffffffu, wait_or_abort(&join_empty[t], (items - 1) & 1u, misc, p.err));
            if (!ok) break;
            *joined = w;
            __syncwarp();
            if (lane == 0) mbar_arrive(&join_full[t]);
            ++items;
            continue;
          }
          ok = __all_sync(0xffffffffu, wait_or_abort(&join_full[t], items & 1u, misc, p.err));
          if (!ok) break;
          w += *joined;
          __syncwarp();
          if (lane == 0) mbar_arrive(&join_empty[t]);
          ++items;
        }
        if (s.slot >= 0) {
          kp.k.parts[(int64_t)s.slot * kMaxKeys + t * kKT + row + lane] = w;
        } else if (key < s.klen) {
          const Req rq = {s.qlen, s.klen, 0, s.kbase};
          give(kp.k, rq, s.r, s.kh, key, id, w);
        }
      }
    }
    if (!ok) misc[0] = 1;
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == Ge::kWarpMma)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Ge::kTmem) : "memory");
}

template <typename T, int KD, int N>
int launch(const KwMmaParams& kp, cudaStream_t s) {
  const void* kern = reinterpret_cast<const void*>(fd_keyw_mma_kernel<T, KD, N>);
  static unsigned long long done = 0;
  const int st = fdh::ensure_smem(kern, Geo<KD, N>::kSmem, &done);
  if (st != FD_OK) return st;
  return fdh::launch_maybe_pdl(kern, dim3((unsigned)kp.k.a.ctas), dim3(Geo<KD, N>::kThreads), Geo<KD, N>::kSmem, s, false, kp,
                               "fd_keyw_mma_kernel launch");
}

template <typename T>
int launch_for(const KwMmaParams& kp, int n, cudaStream_t s) {
  if (kp.k.a.D <= 64)
    return n == 16 ? launch<T, 64, 16>(kp, s) : n == 32 ? launch<T, 64, 32>(kp, s) : launch<T, 64, 128>(kp, s);
  return n == 16 ? launch<T, 128, 16>(kp, s) : n == 32 ? launch<T, 128, 32>(kp, s) : launch<T, 128, 128>(kp, s);
}

}  // namespace mm

int mma_launch(KwParams& p, const fd_attn_args* a, const Plan& plan, cudaStream_t s) {
  p.a.tq = plan.cols / p.a.G;
  mm::KwMmaParams kp{};
  kp.k = p;
  kp.m.a = p.a;
  at::mm::encode_maps(kp.m, a, true);
  const int st = a->dtype == FD_DTYPE_BF16 ? mm::launch_for<__nv_bfloat16>(kp, plan.cols, s) : mm::launch_for<__half>(kp, plan.cols, s);
  if (st != FD_OK || plan.whole) return st;
  return combine_launch(p, mm::kKeys, s);
}

}  // namespace kw
}  // namespace fdk
