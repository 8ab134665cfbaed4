// Rotary positions of one to four axes, fused with the tier-aware KV write.
//
//   pair i of a head of token t:  c = cos_sin[p, i], s = cos_sin[p, R/2 + i],
//   p = positions[axis_of_pair[i], t];  (x1, x2) -> (x1 c - x2 s, x2 c + x1 s)
//
// One pass over q, k and v: three flops per element, so bytes bound it (HBM
// for prompts, launch and three dependent loads for a decode step).  A CTA
// takes up to kMaxTok tokens: it gathers their cos / sin rows once into shared memory
// (every head of a token turns by the same angles, each axis by its own row
// of the table) and then walks the tokens' vectors: two vectors of VE elements
// that hold VE whole pairs (one of either half, or two neighbours) of every
// head, then plain vectors of v and of the dims behind rot_dim.  A thread
// loads kBatch of them before it stores the first, so enough loads are in
// flight and q_out = q (in place) stays safe: every element is read and
// written by one thread, in that order.
//
// Measured: 16384 tokens of 32 + 8 heads x 128 in 80 us, 5.1 TB/s read and
// written; 128 tokens in 4.7 us.

#include <type_traits>

#include "fd_common.cuh"
#include "fd_internal.h"

namespace fdk {
namespace rp {

struct RopeParams {
  const unsigned char *q, *k, *v;
  unsigned char *q_out, *k_out;
  int64_t q_st, q_sh, qo_st, qo_sh, k_st, k_sh, v_st, v_sh, ko_st, ko_sh;  // bytes
  const int64_t* pos;
  int64_t pos_stride;
  const float* cs;
  int64_t max_pos;
  const int64_t* slots;
  unsigned char *tk[2], *tv[2];
  int64_t blk_sb[2], head_sb[2], tok_sb[2], nblk[2];
  int64_t split;
  int T, H, KVH, D, rot, BS;
  int pairs;    // 1: neighbouring dims form a pair
  int upr;      // units per head: rot / 2 / VE
  int rest;     // vectors per head behind rot_dim: (D - rot) / VE
  int vch;      // vectors per head of v: D / VE (0: no KV write)
  int tok;      // tokens per CTA
  unsigned char axis[FD_ROPE_MAX_PAIRS];
  int32_t* err;
};

constexpr int kThreads = 256;
constexpr int kCtasPerSm = 4;
constexpr int kBatch = 4;
constexpr int kMaxTok = 8;

template <int BYTES>
struct VecOf;
template <>
struct VecOf<16> {
  typedef uint4 type;
};
template <>
struct VecOf<8> {
  typedef uint2 type;
};
template <>
struct VecOf<4> {
  typedef uint32_t type;
};
template <>
struct VecOf<2> {
  typedef unsigned short type;
};

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(float x) { return x; }

template <typename T, int VE>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) fd_rope_kernel(const __grid_constant__ RopeParams p) {
  typedef typename VecOf<VE * sizeof(T)>::type V;
  union Vec {
    V v;
    T e[VE];
  };
  constexpr int VB = VE * (int)sizeof(T);
  extern __shared__ float cs[];  // [tok][rot]: cos of the pairs, then sin
  __shared__ int64_t k_at[kMaxTok];  // byte offset of the token's K/V row in its tier, -1: none
  __shared__ int tier_of[kMaxTok];
  __shared__ int live[kMaxTok];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * p.tok;
  const int nt = min(p.tok, p.T - t0);
  const int half = p.rot / 2;

  if (tid < nt) {
    live[tid] = 1;
    int64_t at = -1;
    int tr = 0;
    if (p.slots != nullptr) {
      const int64_t s = p.slots[t0 + tid];
      if (s >= 0) {
        int64_t b = s / p.BS;
        const int64_t off = s - b * p.BS;
        if (b >= p.split) {
          tr = 1;
          b -= p.split;
        }
        if (b < p.nblk[tr])
          at = b * p.blk_sb[tr] + off * p.tok_sb[tr];
        else
          set_error(p.err, FD_DEVERR_SLOT);
      }
    }
    k_at[tid] = at;
    tier_of[tid] = tr;
  }
  __syncthreads();
  for (int x = tid; x < nt * half; x += kThreads) {
    const int t = x / half, i = x - t * half;
    const int64_t pos = p.pos[(int64_t)p.axis[i] * p.pos_stride + t0 + t];
    if (pos < 0 || pos >= p.max_pos) {
      live[t] = 0;  // every writer writes the same value
      set_error(p.err, FD_DEVERR_POSITION);
    } else {
      cs[t * p.rot + i] = p.cs[pos * p.rot + i];
      cs[t * p.rot + half + i] = p.cs[pos * p.rot + half + i];
    }
  }

  // v: its first loads are under way while the angles arrive.  A row has a
  // thread per vector, as far as there are threads
  const int v_lanes = min(p.vch, kThreads);
  const int v_lane = v_lanes > 0 ? tid % v_lanes : 0, v_row = v_lanes > 0 ? tid / v_lanes : 0;
  const int v_step = v_lanes > 0 ? kThreads / v_lanes : 1;
  const int v_rows = v_lanes > 0 && v_row < v_step ? nt * p.KVH : 0;
  for (int f0 = v_row;; f0 += v_step * kBatch) {
    const bool first = f0 == v_row;
    if (f0 >= v_rows && !first) break;
    V a[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int f = f0 + u * v_step;
      if (f >= v_rows) continue;
      const int t = f / p.KVH, h = f - t * p.KVH;
      a[u] = *reinterpret_cast<const V*>(p.v + (int64_t)(t0 + t) * p.v_st + h * p.v_sh + v_lane * VB);
    }
    if (first) __syncthreads();  // angles, slots and live tokens (every thread comes here once)
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int f = f0 + u * v_step;
      if (f >= v_rows) continue;
      const int t = f / p.KVH, h = f - t * p.KVH;
      const int tr = tier_of[t];
      if (live[t] && k_at[t] >= 0)
        *reinterpret_cast<V*>(p.tv[tr] + k_at[t] + h * p.head_sb[tr] + v_lane * VB) = a[u];
    }
  }
  // the vectors of a row behind the first kThreads
  if (const int tail = p.vch - v_lanes; tail > 0) {
    for (int x = tid; x < nt * p.KVH * tail; x += kThreads) {
      const int f = x / tail, t = f / p.KVH, h = f - t * p.KVH, tr = tier_of[t];
      const int off = (kThreads + x - f * tail) * VB;
      if (live[t] && k_at[t] >= 0)
        *reinterpret_cast<V*>(p.tv[tr] + k_at[t] + h * p.head_sb[tr] + off) =
            *reinterpret_cast<const V*>(p.v + (int64_t)(t0 + t) * p.v_st + h * p.v_sh + off);
    }
  }

  // Where vector `off` of head h (q's, then k's) of token t is read.
  auto source = [&](int t, int h, int off) -> const unsigned char* {
    return h < p.H ? p.q + (int64_t)(t0 + t) * p.q_st + h * p.q_sh + off
                   : p.k + (int64_t)(t0 + t) * p.k_st + (h - p.H) * p.k_sh + off;
  };
  // The destinations of it: q_out, or the cache row and k_out.
  auto put = [&](int t, int h, int off, const V& x) {
    if (h < p.H) {
      *reinterpret_cast<V*>(p.q_out + (int64_t)(t0 + t) * p.qo_st + h * p.qo_sh + off) = x;
      return;
    }
    const int kh = h - p.H, tr = tier_of[t];
    if (k_at[t] >= 0) *reinterpret_cast<V*>(p.tk[tr] + k_at[t] + kh * p.head_sb[tr] + off) = x;
    if (p.k_out != nullptr)
      *reinterpret_cast<V*>(p.k_out + (int64_t)(t0 + t) * p.ko_st + kh * p.ko_sh + off) = x;
  };
  const int heads = p.H + p.KVH, rows = nt * heads;

  // the rotated dims: thread `lane` of a head's upr takes pairs lane * VE ..
  {
    const int lane = tid % p.upr, row = tid / p.upr, step = kThreads / p.upr;
    const int off = (p.pairs ? 2 * lane : lane) * VB, gap = p.pairs ? VB : half * (int)sizeof(T);
    for (int f0 = row; row < step && f0 < rows; f0 += step * kBatch) {
      Vec a[kBatch], b[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int f = f0 + u * step;
        if (f >= rows) continue;
        const int t = f / heads, h = f - t * heads;
        const unsigned char* src = source(t, h, off);
        a[u].v = *reinterpret_cast<const V*>(src);
        b[u].v = *reinterpret_cast<const V*>(src + gap);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int f = f0 + u * step;
        if (f >= rows) continue;
        const int t = f / heads, h = f - t * heads;
        if (!live[t]) continue;
        const float* c = cs + t * p.rot + lane * VE;
        Vec ra, rb;
        if (p.pairs) {  // the two vectors hold pairs (2 i, 2 i + 1) in turn
          T in[2 * VE], out[2 * VE];
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            in[e] = a[u].e[e];
            in[VE + e] = b[u].e[e];
          }
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float x1 = to_f(in[2 * e]), x2 = to_f(in[2 * e + 1]);
            out[2 * e] = Dt<T>::narrow(x1 * c[e] - x2 * c[half + e]);
            out[2 * e + 1] = Dt<T>::narrow(x2 * c[e] + x1 * c[half + e]);
          }
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            ra.e[e] = out[e];
            rb.e[e] = out[VE + e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float x1 = to_f(a[u].e[e]), x2 = to_f(b[u].e[e]);
            ra.e[e] = Dt<T>::narrow(x1 * c[e] - x2 * c[half + e]);
            rb.e[e] = Dt<T>::narrow(x2 * c[e] + x1 * c[half + e]);
          }
        }
        put(t, h, off, ra.v);
        put(t, h, off + gap, rb.v);
      }
    }
  }

  // the dims behind rot_dim
  if (p.rest > 0) {
    for (int x = tid; x < rows * p.rest; x += kThreads) {
      const int f = x / p.rest, t = f / heads, h = f - t * heads;
      if (!live[t]) continue;
      const int off = p.rot * (int)sizeof(T) + (x - f * p.rest) * VB;
      put(t, h, off, *reinterpret_cast<const V*>(source(t, h, off)));
    }
  }
}

template <typename T, int VE>
int launch(RopeParams& p, cudaStream_t s) {
  p.upr = p.rot / 2 / VE;
  p.rest = (p.D - p.rot) / VE;
  p.vch = p.slots != nullptr ? p.D / VE : 0;
  int dev = 0, sms = 0;
  const int st = fdh::device_sms(&dev, &sms);
  if (st != FD_OK) return st;
  // tokens per CTA: as few as keep the grid to one wave (a decode step: one),
  // so the cos / sin gather and the slots are under way at once, and the
  // vectors behind them cover the latency.  1024 tokens: 8.3 us; with grids up
  // to two waves 10.1, one token per CTA 10.0.  16384: 80 us, one token per
  // CTA 161.
  p.tok = 1;
  while (p.tok < kMaxTok && (int64_t)p.T > (int64_t)p.tok * sms * kCtasPerSm) p.tok *= 2;
  const unsigned grid = (unsigned)((p.T + p.tok - 1) / p.tok);
  fd_rope_kernel<T, VE><<<grid, kThreads, (size_t)p.tok * p.rot * 4, s>>>(p);
  return fdh::cuda_status(cudaGetLastError(), "fd_rope_kernel launch");
}

// The widest vector that every pointer, stride, half and rest is a multiple of.
template <typename T>
int dispatch(RopeParams& p, cudaStream_t s) {
  constexpr int kFull = 16 / (int)sizeof(T);
  auto fits = [&](int ve) { return (p.rot / 2) % ve == 0 && (p.D - p.rot) % ve == 0; };
  if (fits(kFull)) return launch<T, kFull>(p, s);
  if (fits(kFull / 2)) return launch<T, kFull / 2>(p, s);
  return launch<T, 1>(p, s);
}

}  // namespace rp
}  // namespace fdk

extern "C" int fd_rope_store_kv(const fd_rope_args* a, void* stream) {
  if (a == nullptr) return fdh::fail(FD_ERR_INVALID, "fd_rope_store_kv: null args");
  const int es = fdh::elem_size(a->dtype);
  if (es == 0) return fdh::fail(FD_ERR_UNSUPPORTED, "fd_rope_store_kv: unsupported dtype %d", a->dtype);
  if (a->num_tokens < 0 || a->num_heads <= 0 || a->num_kv_heads <= 0 || a->head_size <= 0)
    return fdh::fail(FD_ERR_INVALID, "fd_rope_store_kv: bad shape");
  if (a->rot_dim <= 0 || a->rot_dim % 2 != 0 || a->rot_dim > a->head_size)
    return fdh::fail(FD_ERR_INVALID, "fd_rope_store_kv: rot_dim must be even, positive and at most head_size");
  if (a->rot_dim / 2 > FD_ROPE_MAX_PAIRS)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_rope_store_kv: rot_dim at most %d", 2 * FD_ROPE_MAX_PAIRS);
  if (a->num_axes < 1 || a->num_axes > FD_ROPE_MAX_AXES)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_rope_store_kv: 1 to %d axes", FD_ROPE_MAX_AXES);
  for (int i = 0; i < a->rot_dim / 2; ++i)
    if (a->axis_of_pair[i] >= a->num_axes)
      return fdh::fail(FD_ERR_INVALID, "fd_rope_store_kv: pair %d has axis %d of %d", i, a->axis_of_pair[i],
                       a->num_axes);
  if (a->num_tokens == 0) return FD_OK;
  if (a->q == nullptr || a->q_out == nullptr || a->k == nullptr || a->v == nullptr || a->positions == nullptr ||
      a->cos_sin == nullptr || a->max_pos <= 0)
    return fdh::fail(FD_ERR_INVALID, "fd_rope_store_kv: q, q_out, k, v, positions and cos_sin are required");
  if (((int64_t)a->head_size * es) % 16 != 0)
    return fdh::fail(FD_ERR_ALIGN, "fd_rope_store_kv: head_size*elem_size must be a multiple of 16");
  const int64_t strides[] = {a->q_stride_t, a->q_stride_h, a->qo_stride_t, a->qo_stride_h, a->k_stride_t,
                             a->k_stride_h, a->v_stride_t, a->v_stride_h,
                             a->k_out != nullptr ? a->ko_stride_t : 0, a->k_out != nullptr ? a->ko_stride_h : 0};
  for (const int64_t x : strides)
    if ((x * es) % 16 != 0)
      return fdh::fail(FD_ERR_ALIGN, "fd_rope_store_kv: strides must be multiples of 16 bytes");
  if (!fdh::aligned16(a->q) || !fdh::aligned16(a->q_out) || !fdh::aligned16(a->k) || !fdh::aligned16(a->v) ||
      !fdh::aligned16(a->k_out) || !fdh::aligned16(a->cos_sin))
    return fdh::fail(FD_ERR_ALIGN, "fd_rope_store_kv: pointers must be 16-byte aligned");
  fdk::rp::RopeParams p{};
  p.q = static_cast<const unsigned char*>(a->q);
  p.k = static_cast<const unsigned char*>(a->k);
  p.v = static_cast<const unsigned char*>(a->v);
  p.q_out = static_cast<unsigned char*>(a->q_out);
  p.k_out = static_cast<unsigned char*>(a->k_out);
  p.q_st = a->q_stride_t * es;
  p.q_sh = a->q_stride_h * es;
  p.qo_st = a->qo_stride_t * es;
  p.qo_sh = a->qo_stride_h * es;
  p.k_st = a->k_stride_t * es;
  p.k_sh = a->k_stride_h * es;
  p.v_st = a->v_stride_t * es;
  p.v_sh = a->v_stride_h * es;
  p.ko_st = a->ko_stride_t * es;
  p.ko_sh = a->ko_stride_h * es;
  p.pos = a->positions;
  p.pos_stride = a->pos_stride;
  p.cs = a->cos_sin;
  p.max_pos = a->max_pos;
  p.slots = a->slots;
  p.split = a->tier_split;
  if (a->slots != nullptr) {
    if (a->block_size <= 0) return fdh::fail(FD_ERR_INVALID, "fd_rope_store_kv: block_size must be positive");
    for (int t = 0; t < 2; ++t) {
      const fd_kv_tier& tr = a->tier[t];
      p.tk[t] = static_cast<unsigned char*>(tr.k);
      p.tv[t] = static_cast<unsigned char*>(tr.v);
      p.blk_sb[t] = tr.blk_stride * es;
      p.head_sb[t] = tr.head_stride * es;
      p.tok_sb[t] = tr.tok_stride * es;
      p.nblk[t] = tr.num_blocks > 0 ? tr.num_blocks : 0;
      if (p.nblk[t] == 0) continue;
      if (p.tk[t] == nullptr || p.tv[t] == nullptr)
        return fdh::fail(FD_ERR_INVALID, "fd_rope_store_kv: tier %d has blocks but no K/V pointer", t);
      if (!fdh::aligned16(p.tk[t]) || !fdh::aligned16(p.tv[t]) || p.blk_sb[t] % 16 || p.head_sb[t] % 16 ||
          p.tok_sb[t] % 16)
        return fdh::fail(FD_ERR_ALIGN, "fd_rope_store_kv: tier %d pointers/strides must be 16-byte aligned", t);
    }
  }
  p.T = a->num_tokens;
  p.H = a->num_heads;
  p.KVH = a->num_kv_heads;
  p.D = a->head_size;
  p.rot = a->rot_dim;
  p.BS = a->block_size > 0 ? a->block_size : 1;
  p.pairs = (a->flags & FD_ROPE_PAIRS) ? 1 : 0;
  for (int i = 0; i < a->rot_dim / 2; ++i) p.axis[i] = a->axis_of_pair[i];
  p.err = a->error;
  // a CTA's vectors are counted in 32 bits (eight tokens of at least two elements a vector)
  if (((int64_t)p.H + 2 * (int64_t)p.KVH) * p.D * fdk::rp::kMaxTok >= (int64_t)1 << 30)
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_rope_store_kv: a token's heads are too many");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case FD_DTYPE_F16:
      return fdk::rp::dispatch<__half>(p, s);
    case FD_DTYPE_BF16:
      return fdk::rp::dispatch<__nv_bfloat16>(p, s);
    default:
      return fdk::rp::dispatch<float>(p, s);
  }
}

extern "C" size_t fd_rope_args_bytes(void) { return sizeof(fd_rope_args); }
