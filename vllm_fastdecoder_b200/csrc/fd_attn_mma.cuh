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
constexpr int kWhole = 8;           // key tiles up to which no item is cut (whole_items)
constexpr int kSub = 16;            // keys per TMA box
constexpr int kSubs = kKT / kSub;
constexpr int kPanel = 128 * 128;   // 128 rows x 64 dims of 16 bits

struct MmaParams {
  CUtensorMap tmap_q;       // {D, H, T, 1}, box {64, G, tq, 1}
  CUtensorMap tmap_k[3];    // per tier {D, KVH, BS, blocks} (cross: {D, KVH, rows, 1}), box {64, 1, 16, 1}
  CUtensorMap tmap_v[3];
  AttnParams a;
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

// A ring position moved on by `by` slots.
template <int R>
__device__ __forceinline__ void advance(int& slot, uint32_t& phase, int by) {
  if (by > R) {
    phase ^= (uint32_t)(by / R) & 1u;
    by %= R;
  }
  slot += by;
  if (slot >= R) {
    slot -= R;
    phase ^= 1u;
  }
}

// The products with 128-byte swizzled operands, descriptors by their low
// words (address and leading offset, 16-byte units); the high word (stride
// 1024 bytes, version, swizzle) is the same for all of them.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void umma_f16_lo(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts_lo(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc,
                                               uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}

// 32 bytes in one store (both 32-byte aligned).
__device__ __forceinline__ void stg256(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Block id of box `lane` (keys 128 j + 16 lane ..) where boxes lie within
// blocks, -1 where there is none.  Read one tile ahead of its use.
__device__ __forceinline__ int box_block(const AttnParams& p, int kbase, int klen, int j, int lane) {
  const int t = j * kKT + lane * kSub;
  if (p.bt == nullptr || p.BS % kSub != 0 || lane >= kSubs || t >= klen) return -1;
  return p.bt[(int64_t)kbase * p.bt_stride + t / p.BS];
}

// One warp: K or V of key tile j into `dst`, completion on `bar` (bytes of
// the TMA boxes, and lane 0's arrival once the other boxes are stored).
template <int KD>
__device__ __forceinline__ void load_tile(const MmaParams& mp, bool is_v, unsigned char* dst, uint64_t* bar, int j,
                                          int r, int kbase, int klen, int kh, int id, int lane, uint64_t pol) {
  const AttnParams& p = mp.a;
  const int t = j * kKT + lane * kSub;
  const bool boxed = p.bt == nullptr || p.BS % kSub == 0;
  bool in = lane < kSubs && t < klen;  // the box holds a key
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
    tma = in && mp.kv_tma[tier] && (!is_v || t + kSub <= klen);
  }
  const unsigned tmask = __ballot_sync(0xffffffffu, tma);
  const unsigned all = (1u << kSubs) - 1u;
  // K boxes without a key need nothing (the mask replaces their scores)
  unsigned rest = is_v ? all & ~tmask : __ballot_sync(0xffffffffu, in) & ~tmask;
  if (lane == 0) mbar_expect_tx(bar, (uint32_t)__popc(tmask) * (uint32_t)(KD / 64 * kSub * 128));
  __syncwarp();
  if (tma) {
    const CUtensorMap* map = is_v ? &mp.tmap_v[tier] : &mp.tmap_k[tier];
#pragma unroll
    for (int x = 0; x < KD / 64; ++x)
      tma_load_4d(dst + x * kPanel + lane * kSub * 128, map, 64 * x, kh, r0, blk, bar, pol);
  }
  if (rest != 0u) {
    constexpr int kCh = KD / 8;                   // 16-byte chunks per row
    constexpr int kPer = kSub * kCh / 32;         // chunks of a box per lane
    while (rest != 0u) {
      const int s = __ffs(rest) - 1;
      rest &= rest - 1u;
      const bool box_in = __shfl_sync(0xffffffffu, (int)in, s) != 0;
      const int box_tier = __shfl_sync(0xffffffffu, tier, s);
      const int box_blk = __shfl_sync(0xffffffffu, blk, s);
      const int box_r0 = __shfl_sync(0xffffffffu, r0, s);
      uint4 v[kPer];
#pragma unroll
      for (int c = 0; c < kPer; ++c) {
        const int idx = c * 32 + lane, row = idx / kCh, ch = idx % kCh;
        const int key = j * kKT + s * kSub + row;
        v[c] = make_uint4(0u, 0u, 0u, 0u);
        if (!box_in || key >= klen || ch * 8 >= p.D) continue;
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
        v[c] = *reinterpret_cast<const uint4*>(base + b * p.blk_sb[tr] + kh * p.head_sb[tr] +
                                               (int64_t)rr * p.tok_sb[tr] + ch * 16);
      }
#pragma unroll
      for (int c = 0; c < kPer; ++c) {
        const int idx = c * 32 + lane, row = idx / kCh, ch = idx % kCh;
        sts128(dst + (ch >> 3) * kPanel + swz(s * kSub + row, ch & 7), v[c]);
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

// The tensor maps of a call's q (tiles of p.tq tokens) and K/V views; views
// that have none are read by 16-byte loads.
void encode_maps(MmaParams& mp, const fd_attn_args* a);

}  // namespace mm
}  // namespace at
}  // namespace fdk
