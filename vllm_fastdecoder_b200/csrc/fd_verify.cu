// Verification of drafted tokens against the target's probabilities.
//
//   a = the first draft d without u_d q_d(x_d) < p_d(x_d)
//   w = max(p_a - q_a, 0) (p where all were accepted)
//   next token = the first i with w_0 + .. + w_i > u (w_0 + .. + w_{V-1})
//
// A cluster of CTAs per request.  Every CTA finds a by itself (a few values
// of a few rows), then takes an equal part of the vocabulary: one pass over
// its part of p_a and q_a gives the parts' sums, each CTA learns all of them
// through distributed shared memory, and the one that holds u times the whole
// goes through its winning warp's few hundred values again for the place.  No
// workspace, no second launch, no atomics: every sum has a fixed order.
// The sums are fp64: a running sum over 100,000 probabilities in fp32 is off by
// more than the smaller of them, so the drawn token would depend on the order.
// A difference of two fp32 (or 16-bit) values is nearly always exact in fp64,
// the comparison u q < p always (48 bits).
//
// Bound by the bytes of one target row and one draft row per request, and for
// a few requests by the chain of loads that leads to them (lengths, tokens,
// two probabilities, the rows).
// Measured: 1 request of 4 drafts over 32,000 fp32 values in 6.4 us; 64 of 5 over
// 131,072 fp32 values in 21.4, most of it the stream of 67 MB (256 CTAs, of which
// 108 SMs have two and the others one), the rest the chain of loads before it, the
// exchange and the search; 19.2 without draft probabilities; of 16 bits 18.8 and
// 16.8.  With one vector of each row in flight per thread 23.4, with 3, 6 and 8
// 22.3, 26.2 and 29.8 (a warp's span ends inside its last round, whose loads are
// then few).  With 8 CTAs per request, in several waves, 55.

#include <cooperative_groups.h>

#include <type_traits>

#include "fd_common.cuh"
#include "fd_internal.h"

namespace fdk {
namespace vf {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

struct VerifyParams {
  fd_verify_args a;
  int wide;  // rows are 16-byte aligned
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// A probability, or 0 where it is negative, infinite or a NaN.
__device__ __forceinline__ float prob(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The weights of a request's rows, a vector of kV values at a time.  Where x <=
// y the weight is 0, which fp32 tells exactly; only the others become fp64.
template <typename T, int kV>
struct Rows {
  const T* p;
  const T* q;        // null: none
  long long struck;  // the element that counts as 0, or -1
  typedef typename std::conditional<kV == 1, T, uint4>::type Vec;
  __device__ __forceinline__ static Vec get(const T* at, long long i) {
    if constexpr (kV == 1)
      return __ldg(at + i);
    else
      return __ldg(reinterpret_cast<const uint4*>(at + i));
  }
  __device__ __forceinline__ static void values(const Vec& v, float (&x)[kV]) {
    if constexpr (kV == 1)
      x[0] = as_float(v);
    else
      Dt<T>::widen(v, x);
  }
  __device__ __forceinline__ static double over(float x, float y) {
    x = prob(x);
    y = prob(y);
    return x > y ? (double)x - (double)y : 0.0;
  }
  // of the vector from element i on
  __device__ __forceinline__ void weights(const Vec& vp, const Vec& vq, long long i, double (&w)[kV]) const {
    float x[kV];
    values(vp, x);
    if (q != nullptr) {
      float y[kV];
      values(vq, y);
#pragma unroll
      for (int e = 0; e < kV; ++e) w[e] = over(x[e], y[e]);
    } else {
#pragma unroll
      for (int e = 0; e < kV; ++e) w[e] = i + e == struck ? 0.0 : (double)prob(x[e]);
    }
  }
  // of element i alone
  __device__ __forceinline__ double weight(long long i) const {
    return i == struck ? 0.0 : over(as_float(p[i]), q != nullptr ? as_float(q[i]) : 0.f);
  }
};

template <typename T, int kV>
__global__ void __launch_bounds__(kThreads, 2) fd_verify_kernel(const __grid_constant__ VerifyParams vp) {
  constexpr int kUnroll = kV > 1 ? 2 : 4;  // pieces of each row that a thread has in flight
  const fd_verify_args& a = vp.a;
  __shared__ int s_accepted;  // -1: no tokens
  __shared__ double part[2][kMaxCluster];  // the CTAs' sums, of either attempt
  __shared__ double warps[kWarps];
  __shared__ double scan[kWarps];
  __shared__ unsigned s_found[kWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const int nct = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int r = blockIdx.x / nct;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int K = a.num_drafts;
  if (nct > 1) cluster.barrier_arrive();  // this CTA has started; awaited before the first write to another's memory
  const int qlen = a.q_len[r], qst = a.q_start[r];

  if (warp == 0) {  // the first draft that is not accepted
    int acc = qlen - 1;
    const bool ok = qlen >= 1 && qlen <= K + 1 && qst >= 0 && (long long)qst + qlen <= a.num_rows;
    if (!ok) {
      acc = -1;
      if (qlen != 0 && lane == 0 && rank == 0) set_error(a.error, FD_DEVERR_LEN);
    }
    for (int base = 0; base < K; base += 32) {  // (the first tokens and numbers are fetched beside the lengths)
      const int d = base + lane;
      bool good = true;
      long long x = 0;
      float u = 0.f;
      if (d < K) {
        x = a.draft_tokens[(int64_t)r * a.tokens_stride + d];
        u = a.accept_u[(int64_t)r * a.accept_stride + d];
      }
      if (d < acc) {
        good = x >= 0 && x < a.vocab;
        if (good) {
          const float p = prob(as_float(static_cast<const T*>(a.target)[(int64_t)(qst + d) * a.target_stride + x]));
          const float q = a.draft_probs == nullptr
                              ? 1.f
                              : prob(as_float(static_cast<const T*>(a.draft_probs)[(int64_t)r * a.draft_stride_r +
                                                                                   (int64_t)d * a.draft_stride_k + x]));
          good = (double)u * (double)q < (double)p;
        } else if (rank == 0) {
          set_error(a.error, FD_DEVERR_TOKEN);
        }
      }
      const unsigned bad = __ballot_sync(0xffffffffu, !good);
      if (bad != 0u) acc = base + __ffs(bad) - 1;
      if (bad != 0u || base + 32 >= acc) break;
    }
    if (lane == 0) s_accepted = acc;
  }
  __syncthreads();
  const int acc = s_accepted;
  const bool none = acc < 0;  // the whole cluster alike
  if (rank == 0) {
    // the drawn token is written by the CTA that finds it
    for (int c = tid; c <= K; c += kThreads)
      if (none || c != acc)
        a.tokens[(int64_t)r * (K + 1) + c] = c < acc ? a.draft_tokens[(int64_t)r * a.tokens_stride + c] : -1;
    if (tid == 0) {
      a.accepted[r] = none ? 0 : acc;
      if (a.lens != nullptr) a.keep_lens[r] = none ? a.lens[r] : a.lens[r] - (qlen - 1 - acc);
    }
  }
  if (none) {
    if (nct > 1) cluster.barrier_wait();
    return;
  }

  const bool rejected = acc < qlen - 1;
  const long long V = a.vocab;
  Rows<T, kV> rows;
  rows.p = static_cast<const T*>(a.target) + (int64_t)(qst + acc) * a.target_stride;
  rows.q = rejected && a.draft_probs != nullptr
               ? static_cast<const T*>(a.draft_probs) + (int64_t)r * a.draft_stride_r + (int64_t)acc * a.draft_stride_k
               : nullptr;
  rows.struck = rejected && a.draft_probs == nullptr ? a.draft_tokens[(int64_t)r * a.tokens_stride + acc] : -1;
  typedef typename Rows<T, kV>::Vec Vec;
  // whole vectors of the row, cut into equal spans over the CTAs, then over
  // their warps; the elements behind the last whole vector (fewer than kV)
  // follow the last warp's of the last CTA
  const long long nvec = V / kV;
  const long long cta_lo = nvec * rank / nct, cta_n = nvec * (rank + 1) / nct - cta_lo;
  const bool last_cta = rank == nct - 1;
  const int ntail = last_cta ? (int)(V - nvec * kV) : 0;

  double total = 0.0;
  int attempt = 0;
  for (;; ++attempt) {
    const long long lo = cta_lo + cta_n * warp / kWarps, hi = cta_lo + cta_n * (warp + 1) / kWarps;
    double s = 0.0;
    for (long long base = lo; base < hi; base += 32 * kUnroll) {
      Vec x[kUnroll], y[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const long long i = base + 32 * u + lane;
        if (i < hi) {
          x[u] = Rows<T, kV>::get(rows.p, i * kV);
          if (rows.q != nullptr) y[u] = Rows<T, kV>::get(rows.q, i * kV);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const long long i = base + 32 * u + lane;
        if (i >= hi) continue;
        double w[kV];
        rows.weights(x[u], y[u], i * kV, w);
#pragma unroll
        for (int e = 0; e < kV; ++e) s += w[e];
      }
    }
    if (warp == kWarps - 1 && lane < ntail) s += rows.weight(nvec * kV + lane);
    s = warp_sum(s);
    if (lane == 0) warps[warp] = s;
    __syncthreads();
    if (nct > 1 && attempt == 0) cluster.barrier_wait();
    if (tid < nct) {
      s = 0.0;
      for (int w = 0; w < kWarps; ++w) s += warps[w];
      cluster.map_shared_rank(&part[attempt][0], tid)[rank] = s;
    }
    if (nct > 1)
      cluster.sync();
    else
      __syncthreads();
    // all CTAs from the same numbers in the same order
    total = 0.0;
    for (int c = 0; c < nct; ++c) total += part[attempt][c];
    if (total > 0.0 || attempt == 1) break;
    rows.q = nullptr;  // nothing is left of p less q: p itself
    rows.struck = -1;
  }
  if (!(total > 0.0)) {
    if (rank == 0 && tid == 0) {
      a.tokens[(int64_t)r * (K + 1) + acc] = -1;
      set_error(a.error, FD_DEVERR_PROBS);
    }
    return;
  }
  // The CTA that holds u times the sum: it has a prefix <= target < prefix + its
  // part, so its part is positive.
  const double target = (double)fminf(fmaxf(a.sample_u[r], 0.f), 0x1.fffffep-1f) * total;
  double before = 0.0;
  int owner = 0;
  while (owner < nct - 1 && !(target < before + part[attempt][owner])) before += part[attempt][owner++];
  if (owner != rank) return;
  // the warp's span: the first that passes the target, or, where rounding leaves
  // none, the last one with any weight (every warp by itself)
  const double own = lane < kWarps ? warps[lane] : 0.0;
  double upto = before;
  {
    double incl = own;
#pragma unroll
    for (int off = 1; off < kWarps; off <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    upto += incl;
  }
  const unsigned some = __ballot_sync(0xffffffffu, own > 0.0), beyond = __ballot_sync(0xffffffffu, own > 0.0 && target < upto);
  const int ws = beyond != 0u ? __ffs(beyond) - 1 : 31 - __clz(some);  // (some: the CTA's part is positive)
  const double at_ws = __shfl_sync(0xffffffffu, upto - own, ws);
  // that span again, a vector per thread
  const long long from = cta_lo + cta_n * ws / kWarps;
  const long long to = cta_lo + cta_n * (ws + 1) / kWarps + (ws == kWarps - 1 && ntail > 0 ? 1 : 0);  // (the tail as a vector)
  double run = at_ws;
  for (long long base = from; base < to; base += kThreads) {
    const long long i = base + tid;
    double w[kV], s = 0.0;
#pragma unroll
    for (int e = 0; e < kV; ++e) w[e] = 0.0;
    if (i < to && i < nvec) {
      const Vec x = Rows<T, kV>::get(rows.p, i * kV);
      Vec y{};
      if (rows.q != nullptr) y = Rows<T, kV>::get(rows.q, i * kV);
      rows.weights(x, y, i * kV, w);
    } else if (i < to) {
#pragma unroll
      for (int e = 0; e < kV; ++e)
        if (e < ntail) w[e] = rows.weight(nvec * kV + e);
    }
#pragma unroll
    for (int e = 0; e < kV; ++e) s += w[e];
    double incl = s;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    double sums = lane < kWarps ? scan[lane] : 0.0;
#pragma unroll
    for (int off = 1; off < kWarps; off <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, sums, off);
      if (lane >= off) sums += o;
    }
    const double to_here = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0));
    const double ahead = warp > 0 ? run + to_here : run;
    run += __shfl_sync(0xffffffffu, sums, kWarps - 1);
    // threads with weight, of those the ones that pass the target
    const unsigned any = __ballot_sync(0xffffffffu, s > 0.0);
    const unsigned past = __ballot_sync(0xffffffffu, s > 0.0 && target < ahead + incl);
    if (lane == 0) s_found[warp] = past != 0u ? 64u + (unsigned)(__ffs(past) - 1) : any != 0u ? 32u + (31 - __clz(any)) : 0u;
    __syncthreads();
    const unsigned f = lane < kWarps ? s_found[lane] : 0u;
    const unsigned hits = __ballot_sync(0xffffffffu, f >= 64u), full = __ballot_sync(0xffffffffu, f != 0u);
    const bool done = hits != 0u;
    const int w_at = done ? __ffs(hits) - 1 : 31 - __clz(full);  // -1: no weight in this pass
    const int pick = w_at < 0 ? -1 : 32 * w_at + (int)(__shfl_sync(0xffffffffu, f, max(w_at, 0)) & 31u);
    if (pick == tid) {  // the vector's first element past the target, or its last one with weight
      double b = ahead + (incl - s);
      bool hit = false;
      long long at = -1;
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        b += w[e];
        if (!hit && w[e] > 0.0) {
          at = i * kV + e;
          hit = target < b;
        }
      }
      a.tokens[(int64_t)r * (K + 1) + acc] = at;  // (a later pass with weight writes over it)
    }
    if (done) return;
    __syncthreads();  // scan and s_found have been read; the write above is ordered before the next one
  }
}

template <typename T, int kV>
int launch(const VerifyParams& vp, int ctas, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(vp.a.num_reqs * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[1] = {const_cast<VerifyParams*>(&vp)};
  return fdh::cuda_status(cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(fd_verify_kernel<T, kV>), args),
                          "fd_verify_kernel launch");
}

template <typename T>
int launch_for(const VerifyParams& vp, int ctas, cudaStream_t s) {
  return vp.wide ? launch<T, 16 / (int)sizeof(T)>(vp, ctas, s) : launch<T, 1>(vp, ctas, s);
}

}  // namespace vf
}  // namespace fdk

extern "C" int fd_verify_drafts(const fd_verify_args* a, void* stream) {
  using namespace fdk::vf;
  if (a == nullptr) return fdh::fail(FD_ERR_INVALID, "fd_verify_drafts: null args");
  const int es = fdh::elem_size(a->dtype);
  if (es == 0) return fdh::fail(FD_ERR_UNSUPPORTED, "fd_verify_drafts: unsupported dtype %d", a->dtype);
  if (a->num_reqs < 0 || a->num_drafts < 0 || a->vocab <= 0 || a->num_rows < 0)
    return fdh::fail(FD_ERR_INVALID, "fd_verify_drafts: bad num_reqs, num_drafts, vocab or num_rows");
  if (a->num_drafts > FD_VERIFY_MAX_DRAFTS || a->num_reqs > (1 << 24))
    return fdh::fail(FD_ERR_UNSUPPORTED, "fd_verify_drafts: %d drafts (at most %d) of %d requests", a->num_drafts,
                     FD_VERIFY_MAX_DRAFTS, a->num_reqs);
  if (a->num_reqs == 0) return FD_OK;
  if (a->q_start == nullptr || a->q_len == nullptr || a->sample_u == nullptr || a->tokens == nullptr ||
      a->accepted == nullptr || (a->num_rows > 0 && a->target == nullptr) ||
      (a->num_drafts > 0 && (a->draft_tokens == nullptr || a->accept_u == nullptr)) ||
      (a->lens != nullptr && a->keep_lens == nullptr))
    return fdh::fail(FD_ERR_INVALID, "fd_verify_drafts: null buffer");
  if (a->num_rows > 1 && a->target_stride < a->vocab)
    return fdh::fail(FD_ERR_INVALID, "fd_verify_drafts: target rows must not overlap");
  VerifyParams vp;
  vp.a = *a;
  if (a->num_drafts == 0) vp.a.draft_probs = nullptr;
  auto aligned = [&](const void* p, int64_t stride) { return fdh::aligned16(p) && (stride * es) % 16 == 0; };
  vp.wide = aligned(a->target, a->target_stride) &&
            (vp.a.draft_probs == nullptr || (aligned(a->draft_probs, a->draft_stride_r) && (a->draft_stride_k * es) % 16 == 0));
  // CTAs per request: no more than run at once (two per SM), each with 4096 values at least
  int dev = 0, sms = 0;
  const int st = fdh::device_sms(&dev, &sms);
  if (st != FD_OK) return st;
  int ctas = 1;
  while (ctas < kMaxCluster && 2 * (int64_t)ctas * a->num_reqs <= 2 * sms && (int64_t)a->vocab > (int64_t)ctas * 4096) ctas *= 2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case FD_DTYPE_F16:
      return launch_for<__half>(vp, ctas, s);
    case FD_DTYPE_BF16:
      return launch_for<__nv_bfloat16>(vp, ctas, s);
    default:
      return launch_for<float>(vp, ctas, s);
  }
}

extern "C" size_t fd_verify_args_bytes(void) { return sizeof(fd_verify_args); }
