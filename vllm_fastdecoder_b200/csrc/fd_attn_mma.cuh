// What the two tensor-core kernels of chunk and cross attention
// (fd_attn_mma.cu: many query rows, fd_attn_rows.cu: few) share: tile shapes,
// the K/V and Q tile loads, bounded waits, and PTX forms.
#pragma once

#include "fd_attn.cuh"
#include "fd_decode.cuh"
#include "fd_tcgen05.cuh"

namespace fdk {
namespace at {
namespace mm {

constexpr int kKT = 128;            // keys per K/V tile
// Key tiles whose saving does not pay for a cut (whole_items): 5 tokens of one request
// and 100 of two, 32 heads, 512 keys 13.7 and 22.0 us, cut 16.4 and 25.3; 700
// keys 18.5 and 25.4, cut 18.6 and 25.7; 1024 keys 19.5 and 29.3, cut 16.3 and
// 26.5.
constexpr int kWhole = 5;
constexpr int kFine = 8;            // keys per TMA box at a request's end, and per box of plain loads
constexpr int kFines = kKT / kFine;
constexpr int kFineSh = 5;          // log2 of the box whose cut rows plain loads fetch as fast as boxes of kFine
constexpr int kPanel = 128 * 128;   // 128 rows x 64 dims of 16 bits

struct MmaParams {
  CUtensorMap tmap_q;       // {D, H, T, 1}, box {64, G, tq, 1}
  // per tier {D, KVH, BS, blocks} (cross: {D, KVH, rows, 1}): boxes {64, 1,
  // 2^box_sh, 1} of whole tiles, and of kFine keys for the tile that holds the end of V
  CUtensorMap tmap_k[3];
  CUtensorMap tmap_v[3];
  CUtensorMap tmap_vf[3];
  AttnParams a;
  int box_sh;               // log2 of the keys per box: the largest power of two (8 to 128) that divides a block
  // Layout of a K/V tile in shared memory: groups of 8 keys `group` bytes
  // apart, the second 64 dims `panel` bytes behind the first.  One TMA copy
  // takes one 64-dim panel of a box (1024, kPanel), or, of heads of 128 dims,
  // whole rows (2048, 1024: the maps are encode_lines'; a block
  // of tier t having lines[t] lines): an SM's copies come at ~80 cycles apiece
  // whatever their size, and small boxes leave no slack (32 requests of 4
  // tokens over 4096 keys: blocks of 8 keys 104 us, by panels 135; of 16, 92
  // and 104; of 32, 91 and 91).
  int group, panel;
  int lines[3];
  int q_tma, kv_tma[3];     // the view has a tensor map
};

__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 0) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        set_error(err, FD_DEVERR_TIMEOUT);
        return false;
      }
    }
  }
}

// The same without suspending, for the MMA issuer.
__device__ __forceinline__ bool poll_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
  if (mbar_test_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_test_wait(bar, parity)) return true;
    if ((it & 255u) == 0) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        set_error(err, FD_DEVERR_TIMEOUT);
        return false;
      }
    }
  }
}

// L2 policy for data that other CTAs read too.
__device__ __forceinline__ uint64_t l2_evict_normal_policy() {
  uint64_t pol;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(pol));
  return pol;
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Scores from the nv-th on are not seen.
__device__ __forceinline__ void hide(uint32_t (&r)[32], int nv) {
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (e >= nv) r[e] = __float_as_uint(-INFINITY);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// One thread per barrier: bars[i] counts `count(i)` arrivals.
template <typename F>
__device__ __forceinline__ void init_barriers(uint64_t* bars, int num, F count) {
  if ((int)threadIdx.x < num) {
    mbar_init(bars + threadIdx.x, count((int)threadIdx.x));
    fence_barrier_init();
  }
}

// The next slot of a ring, and its phase's parity.
template <int R>
__device__ __forceinline__ void advance(int& slot, uint32_t& phase) {
  if (++slot == R) {
    slot = 0;
    phase ^= 1u;
  }
}

// The products with 128-byte swizzled operands, descriptors by their low
// words (address and leading offset, 16-byte units) and high words (stride of
// the 8-row groups, version, swizzle).
__device__ __forceinline__ uint32_t desc_hi(uint32_t group) { return (group >> 4) | (1u << 14) | (2u << 29); }
__device__ __forceinline__ void umma_f16_lo(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                            uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts_lo(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi,
                                               uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc), "r"(b_hi)
      : "memory");
}

// Tiled TMA load of a 5-D box (see tma_load_4d).
__device__ __forceinline__ void tma_load_5d(void* smem_dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            int c4, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7], %8;" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar)),
      "l"(policy)
      : "memory");
}

// 32 bytes in one store (both 32-byte aligned).
__device__ __forceinline__ void stg256(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Fetch the tensor maps that the call's loads use (one thread per map).
__device__ __forceinline__ void prefetch_maps(const MmaParams& mp, int x) {
  const CUtensorMap* map = nullptr;
  if (x >= 0 && x < 9) {
    const int t = x / 3;
    if (mp.kv_tma[t] && (x % 3 < 2 || mp.box_sh > kFineSh))
      map = x % 3 == 0 ? &mp.tmap_k[t] : x % 3 == 1 ? &mp.tmap_v[t] : &mp.tmap_vf[t];
  } else if (x == 9 && mp.q_tma) {
    map = &mp.tmap_q;
  }
  if (map != nullptr) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// The box of key tile j that lane `lane` loads: its first key (of the tile)
// and its keys.  Lanes below 16 have the boxes of 2^box_sh keys; for V, whose
// rows behind the request's end must be 0, lanes 16 .. have the kFine-key
// pieces of a large box that the end cuts (of a box of up to 32 keys, plain
// loads fetch them as fast).
struct Box {
  int at, keys;  // keys = 0: none
};
__device__ __forceinline__ Box box_of(const MmaParams& mp, bool is_v, int left, int lane) {  // left: klen - 128 j
  const int sh = mp.box_sh;
  if (lane < 16) return {lane << sh, (lane << sh) < kKT ? 1 << sh : 0};
  const int cut = left >> sh, at = (cut << sh) + (lane - 16) * kFine;  // the box that is cut, if any
  return {at, is_v && left < kKT && at + kFine <= left && sh > kFineSh ? kFine : 0};
}

// Block id of this lane's box where boxes lie within blocks, -1 where there
// is none.  Read one tile ahead of its use.
__device__ __forceinline__ int box_block(const MmaParams& mp, bool is_v, int kbase, int klen, int j, int lane) {
  const AttnParams& p = mp.a;
  const Box box = box_of(mp, is_v, klen - j * kKT, lane);
  const int t = j * kKT + box.at;
  if (p.bt == nullptr || p.BS % kFine != 0 || box.keys == 0 || t >= klen) return -1;
  return p.bt[(int64_t)kbase * p.bt_stride + t / p.BS];
}

// One warp: K or V of key tile j into `dst`, completion on `bar` (bytes of
// the TMA boxes, and lane 0's arrival once what TMA does not load is stored).
template <int KD>
__device__ __forceinline__ void load_tile(const MmaParams& mp, bool is_v, unsigned char* dst, uint64_t* bar, int j,
                                          int r, int kbase, int klen, int kh, int id, int lane, uint64_t pol) {
  const AttnParams& p = mp.a;
  const int sh = mp.box_sh, left = klen - j * kKT;
  const Box box = box_of(mp, is_v, left, lane);
  const int t = j * kKT + box.at;
  const bool boxed = p.bt == nullptr || p.BS % kFine == 0;
  bool in = box.keys > 0 && t < klen;  // the box holds a key
  int tier = 0, blk = 0, r0 = 0;
  bool tma = false;
  if (in && boxed) {
    if (p.bt == nullptr) {
      r0 = kbase + t;
    } else {
      int64_t b = id;
      const int page = t / p.BS;
      r0 = t - page * p.BS;
      tier = locate(p, r, page, b);
      if (tier < 0) {
        in = false;
        tier = 0;
      }
      blk = (int)b;
    }
    tma = in && mp.kv_tma[tier] && (!is_v || box.at + box.keys <= left);
  }
  const unsigned tmask = __ballot_sync(0xffffffffu, tma);
  if (lane == 0)
    mbar_expect_tx(bar, (uint32_t)(KD / 64 * 128) * (((uint32_t)__popc(tmask & 0xffffu) << sh) +
                                                     (uint32_t)__popc(tmask >> 16) * (uint32_t)kFine));
  __syncwarp();
  unsigned char* const to = dst + (box.at >> 3) * mp.group;
  if (tma && lane < 16) {
    const CUtensorMap* map = is_v ? &mp.tmap_v[tier] : &mp.tmap_k[tier];
    if (KD == 128 && mp.group == 2048) {
      tma_load_5d(to, map, 0, 0, 0, r0 >> 3, blk * mp.lines[tier] + kh, bar, pol);
    } else {
#pragma unroll
      for (int x = 0; x < KD / 64; ++x) tma_load_4d(to + x * mp.panel, map, 64 * x, kh, r0, blk, bar, pol);
    }
  }
  if (tmask >> 16 != 0u && tma && lane >= 16) {
#pragma unroll
    for (int x = 0; x < KD / 64; ++x)
      tma_load_4d(to + x * mp.panel, &mp.tmap_vf[tier], 64 * x, kh, r0, blk, bar, pol);
  }
  // kFine-key pieces that no TMA box covers: K's without a key need nothing
  // (the mask replaces their scores), V's are zeros
  const unsigned imask = __ballot_sync(0xffffffffu, in);
  const int owner = lane >> (sh - 3);  // the box that piece `lane` lies in
  const int fine = 16 + lane - ((left >> sh) << (sh - 3));
  const bool covered = ((tmask >> owner) & 1u) || (fine >= 16 && fine < 32 && ((tmask >> fine) & 1u));
  unsigned need = __ballot_sync(0xffffffffu, lane < kFines && !covered && (is_v || lane * kFine < left));
  if (need != 0u) {
    constexpr int kCh = KD / 8;             // 16-byte chunks per row
    constexpr int kPer = kFine * kCh / 32;  // chunks of a piece per lane
    constexpr int kPair = 2;                // pieces in flight
#pragma unroll 1
    while (need != 0u) {
      uint4 v[kPair][kPer];
      int piece[kPair];
#pragma unroll
      for (int w = 0; w < kPair; ++w) {
        piece[w] = __ffs(need) - 1;  // -1: none
        need &= need - 1u;
        const int own = max(piece[w], 0) >> (sh - 3);
        const bool have = piece[w] >= 0 && ((imask >> own) & 1u);
        const int box_tier = __shfl_sync(0xffffffffu, tier, own);
        const int box_blk = __shfl_sync(0xffffffffu, blk, own);
        const int box_r0 = __shfl_sync(0xffffffffu, r0, own) + piece[w] * kFine - (own << sh);
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
          const int idx = c * 32 + lane, row = idx / kCh, ch = idx % kCh;
          const int key = j * kKT + piece[w] * kFine + row;
          v[w][c] = make_uint4(0u, 0u, 0u, 0u);
          if (!have || key >= klen || ch * 8 >= p.D) continue;
          int tr = box_tier, rr = box_r0 + row;
          int64_t b = box_blk;
          if (!boxed) {
            const int page = key / p.BS;
            b = p.bt[(int64_t)kbase * p.bt_stride + page];
            rr = key - page * p.BS;
            tr = locate(p, r, page, b);
            if (tr < 0) continue;
          }
          const unsigned char* base = is_v ? p.v[tr] : p.k[tr];
          v[w][c] = *reinterpret_cast<const uint4*>(base + b * p.blk_sb[tr] + kh * p.head_sb[tr] +
                                                    (int64_t)rr * p.tok_sb[tr] + ch * 16);
        }
      }
#pragma unroll
      for (int w = 0; w < kPair; ++w) {
        if (piece[w] < 0) continue;
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
          const int idx = c * 32 + lane, row = idx / kCh, ch = idx % kCh;
          sts128(dst + piece[w] * mp.group + (ch >> 3) * mp.panel + swz(row, ch & 7), v[w][c]);
        }
      }
    }
    fence_proxy_async_smem();  // the stores before the tensor cores read the slot
  }
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// One warp: the query rows of one tile into `dst` (64-dim panels `panel`
// bytes apart) without TMA.
template <int KD>
__device__ __forceinline__ void load_q(const AttnParams& p, unsigned char* dst, int panel, int kh, int tok, int ntok,
                                       int lane) {
  constexpr int kCh = KD / 8;
  for (int idx = lane; idx < ntok * p.G * kCh; idx += 32) {
    const int row = idx / kCh, ch = idx % kCh;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (ch * 8 < p.D)
      v = *reinterpret_cast<const uint4*>(p.q + (int64_t)(tok + row / p.G) * p.q_st +
                                          (int64_t)(kh * p.G + row % p.G) * p.q_sh + ch * 16);
    sts128(dst + (ch >> 3) * panel + swz(row, ch & 7), v);
  }
  fence_proxy_async_smem();
}

// The tensor maps of a call's q (tiles of p.tq tokens) and K/V views (K's alone
// with k_only); views that have none are read by 16-byte loads.
void encode_maps(MmaParams& mp, const fd_attn_args* a, bool k_only = false);

}  // namespace mm
}  // namespace at
}  // namespace fdk
