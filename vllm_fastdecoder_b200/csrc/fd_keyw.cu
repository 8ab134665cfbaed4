// Attention weight per cached key on the CUDA cores, the combine of cut items,
// and the host side of fd_key_weights.
//
// fd_keyw_kernel takes what the tensor-core kernel (fd_keyw_mma.cu) does not:
// fp32, and 16-bit heads of fewer than 64 or more than 128 dims.  A CTA of 16 x
// 16 threads holds 64 keys of its item in shared memory as fp32 and takes the
// queries 64 rows (tokens x heads) at a time; thread (y, x) has rows 4 y .. 4 y
// + 3 and keys x, x + 16, x + 32, x + 48: 16 scores, of which it keeps four
// sums, one per key.  The 16 threads that share a key add theirs up at the
// item's end.  The next rows are fetched into registers during the products.
// Bound by the fp32 pipe, or, with few rows, by the loads of K.
// Measured: 8 requests of up to 77 tokens over up to 512 keys, 8 heads x 64 of
// fp32, in 10.2 us (13.8 where each CTA looks for its work, 14.8 with the combine
// as well); 2048 tokens of 32 heads over 4096 keys of 8 heads x 256 of bf16 in 3.2
// ms (33 TFLOP/s), 32 single tokens over 4096 such keys in 0.92 ms.

#include "fd_keyw.cuh"

namespace fdk {
namespace kw {

constexpr int kKeys = 64;
constexpr int kRows = 64;
constexpr int kThreads = 256;
constexpr int kFixed = 1;
constexpr int kMinPer = 1;

constexpr int ctas_of(int DP) { return DP <= 64 ? 3 : DP <= 128 ? 2 : 1; }
constexpr int smem_bytes(int DP) { return (kRows + kKeys) * (DP + 4) * 4; }

template <typename T, int DP, bool kDirect>
__global__ void __launch_bounds__(kThreads, ctas_of(DP)) fd_keyw_kernel(const __grid_constant__ KwParams kp) {
  constexpr int VE = 16 / (int)sizeof(T);     // elements per 16-byte load
  constexpr int NV = DP / VE;                 // loads per row
  constexpr int LD = DP + 4;                  // row stride of the tiles (floats)
  constexpr int kVecs = kRows * NV / kThreads;  // loads per thread and tile
  constexpr int KN = kKeys / 16;
  typedef Walk<kKeys, kFixed, kDirect> CoreWalk;
  const AttnParams& p = kp.a;
  extern __shared__ float4 smem4[];
  float* sq = reinterpret_cast<float*>(smem4);
  float* sk = sq + kRows * LD;
  __shared__ typename CoreWalk::Scratch scratch;
  __shared__ const unsigned char* k_row[kKeys];
  __shared__ float neg[kRows];          // -lse log2(e) of the rows
  __shared__ float sums[kThreads / 32][kKeys];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int cta = blockIdx.x;  // (of a grid of items not used)
  const int nvec = p.D / VE;

  griddep_launch_dependents();
  if (tid == 0 && kp.cuts != nullptr) kp.cuts[cta].nparts = 0;
  CoreWalk walk(p);
  if (!walk.template init<kThreads>(&scratch, cta, kMinPer)) return;

  auto put = [&](float* dst, int x, const uint4& v) {
    float f[VE];
    Dt<T>::widen(v, f);
#pragma unroll
    for (int e = 0; e < VE; e += 4)
      *reinterpret_cast<float4*>(dst + x / NV * LD + x % NV * VE + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
  };
  typename CoreWalk::Seg g;
  while (walk.next(g)) {
    const Req rq = walk.rq;
    const int key0 = g.kt * kKeys, base = rq.klen - rq.qlen;
    float acc[KN];
#pragma unroll
    for (int c = 0; c < KN; ++c) acc[c] = 0.f;
    uint4 qr[kVecs];
    float next_neg = 0.f;
    auto fetch = [&](int chunk) {  // the chunk's rows into registers (zeros behind them)
      const int tok0 = chunk * p.tq, rows = min(p.tq, rq.qlen - tok0) * p.G;
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const int x = tid + u * kThreads, row = x / NV, c = x % NV, t = row / p.G;
        qr[u] = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows && c < nvec)
          qr[u] = *reinterpret_cast<const uint4*>(p.q + (int64_t)(rq.qst + tok0 + t) * p.q_st +
                                                  (int64_t)(g.kh * p.G + row - t * p.G) * p.q_sh + c * 16);
      }
      if (tid < kRows && tid < rows) {
        const int t = tid / p.G;
        next_neg = -p.lse[(int64_t)(g.kh * p.G + tid - t * p.G) * p.lse_sh + (int64_t)(rq.qst + tok0 + t) * p.lse_st] * kLog2e;
      }
    };
    fetch(g.c0);
    __syncthreads();  // the last segment's reads of shared memory are done
    if (tid < kKeys) {
      const int j = key0 + tid;
      const unsigned char* row = nullptr;
      if (j < rq.klen) {
        int64_t id = p.bt[(int64_t)rq.kbase * p.bt_stride + j / p.BS];
        const int t = at::locate(p, g.r, j / p.BS, id);
        if (t >= 0) row = p.k[t] + id * p.blk_sb[t] + g.kh * p.head_sb[t] + (int64_t)(j % p.BS) * p.tok_sb[t];
      }
      k_row[tid] = row;
    }
    __syncthreads();
    {
      uint4 kr[kVecs];
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const int x = tid + u * kThreads, row = x / NV, c = x % NV;
        kr[u] = c < nvec && k_row[row] != nullptr ? *reinterpret_cast<const uint4*>(k_row[row] + c * 16)
                                                  : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < kVecs; ++u) put(sk, tid + u * kThreads, kr[u]);
    }
    for (int ch = g.c0; ch < g.c0 + g.n; ++ch) {
      const int tok0 = ch * p.tq, rows = min(p.tq, rq.qlen - tok0) * p.G;
      if (ch > g.c0) __syncthreads();  // the last chunk's reads are done
#pragma unroll
      for (int u = 0; u < kVecs; ++u) put(sq, tid + u * kThreads, qr[u]);
      if (tid < kRows) neg[tid] = next_neg;
      __syncthreads();
      if (ch + 1 < g.c0 + g.n) fetch(ch + 1);
      if ((ty & ~1) * 4 >= rows) continue;  // no row of this warp is real
      float s[4][KN];
      f2_t s2[4][KN];  // even and odd dims' sums in the two halves of a packed FMA
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < KN; ++c) s2[i][c] = 0ull;
#pragma unroll 2
      for (int d = 0; d < p.D; d += 4) {
        ulonglong2 b[KN];
#pragma unroll
        for (int c = 0; c < KN; ++c) b[c] = *reinterpret_cast<const ulonglong2*>(sk + (tx + 16 * c) * LD + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(sq + (4 * ty + i) * LD + d);
#pragma unroll
          for (int c = 0; c < KN; ++c) s2[i][c] = f2_fma(a.y, b[c].y, f2_fma(a.x, b[c].x, s2[i][c]));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 4 * ty + i;
        // the last key that the row sees, relative to the tile
        const int lim = row < rows ? base + tok0 + row / p.G - key0 : -1;
        const float ng = neg[row];
#pragma unroll
        for (int c = 0; c < KN; ++c) {
          float even, odd;
          f2_unpack(s2[i][c], even, odd);
          // a row that saw nothing (lse infinite) gives nothing
          const bool seen = tx + 16 * c <= lim && !isinf(ng);
          s[i][c] = seen ? at::ex2_approx(fmaf(even + odd, p.sl2, ng)) : 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < KN; ++c) acc[c] += (s[0][c] + s[1][c]) + (s[2][c] + s[3][c]);
    }
    // the 16 threads of a key: two in a warp, then the warps
#pragma unroll
    for (int c = 0; c < KN; ++c) {
      const float v = acc[c] + __shfl_xor_sync(0xffffffffu, acc[c], 16);
      if ((tid & 16) == 0) sums[tid >> 5][tx + 16 * c] = v;
    }
    __syncthreads();
    if (tid < kKeys) {
      float w = 0.f;
#pragma unroll
      for (int x = 0; x < kThreads / 32; ++x) w += sums[x][tid];
      const int j = key0 + tid;
      if (!g.whole)
        kp.parts[(int64_t)(2 * cta + (g.head ? 1 : 0)) * kMaxKeys + tid] = w;
      else if (j < rq.klen)
        give(kp, rq, g.r, g.kh, j, p.bt[(int64_t)rq.kbase * p.bt_stride + j / p.BS], w);
    }
    if (g.nparts > 0 && tid == 0) kp.cuts[cta] = Cut{g.nparts, g.r, g.kh, g.kt};
  }
}

// The cut items' partials added up, in ascending order of the CTAs: part 0 is
// slot 1 of the CTA that wrote the record, part i slot 0 of the i-th after it.
__global__ void __launch_bounds__(kMaxKeys) fd_keyw_combine_kernel(const __grid_constant__ KwParams kp, int kt) {
  griddep_wait();
  const AttnParams& p = kp.a;
  const int c = blockIdx.x, tid = threadIdx.x;
  const Cut cut = kp.cuts[c];
  if (cut.nparts == 0) return;
  const Req rq = at::load_req(p, cut.r);
  const int j = cut.kt * kt + tid;
  if (tid >= kt || j >= rq.klen) return;
  const int64_t id = p.bt[(int64_t)rq.kbase * p.bt_stride + j / p.BS];
  float w = 0.f;
#pragma unroll 4
  for (int i = 0; i < cut.nparts; ++i) w += kp.parts[(int64_t)(2 * (c + i) + (i == 0 ? 1 : 0)) * kMaxKeys + tid];
  give(kp, rq, cut.r, cut.kh, j, id, w);
}

int combine_launch(const KwParams& p, int kt, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.a.ctas);
  cfg.blockDim = dim3(kMaxKeys);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[2] = {const_cast<KwParams*>(&p), &kt};
  return fdh::cuda_status(cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(fd_keyw_combine_kernel), args),
                          "fd_keyw_combine_kernel launch");
}

namespace {

size_t base_workspace(const Plan& plan) { return plan.whole ? 0 : (workspace_bytes() + 255) / 256 * 256; }

template <typename T, int DP, bool kDirect>
int core_launch_dp(KwParams& p, const Plan& plan, cudaStream_t s) {
  const void* kern = reinterpret_cast<const void*>(fd_keyw_kernel<T, DP, kDirect>);
  static unsigned long long done = 0;
  int st = fdh::ensure_smem(kern, smem_bytes(DP), &done);
  if (st != FD_OK) return st;
  const dim3 grid = kDirect ? dim3((unsigned)plan.tiles, (unsigned)p.a.KVH, (unsigned)p.a.n) : dim3((unsigned)p.a.ctas);
  st = fdh::launch_maybe_pdl(kern, grid, dim3(kThreads), smem_bytes(DP), s, false, p, "fd_keyw_kernel launch");
  if (st != FD_OK || plan.whole) return st;
  return combine_launch(p, kKeys, s);
}

template <typename T>
int core_launch(KwParams& p, const Plan& plan, cudaStream_t s) {
  const bool direct = plan.tiles > 0;
  if (p.a.D <= 64) return direct ? core_launch_dp<T, 64, true>(p, plan, s) : core_launch_dp<T, 64, false>(p, plan, s);
  if (p.a.D <= 128) return direct ? core_launch_dp<T, 128, true>(p, plan, s) : core_launch_dp<T, 128, false>(p, plan, s);
  return direct ? core_launch_dp<T, 256, true>(p, plan, s) : core_launch_dp<T, 256, false>(p, plan, s);
}

}  // namespace

// Chunks of an item from which on cutting pays: what it evens out is at most
// one item's time per CTA (or, with fewer items than CTAs, the idle ones'
// share of it), what it costs the partials and the combine's launch.  Tensor
// cores (a chunk 1.2 us): 48 items of 10 chunks 18.8 us, whole 23.3; 96 of 10
// 27.3 and 24.5; 512 of 4 51.2 and 45.7; 64 of 32 31.9 and 55.4.  CUDA cores:
// 40 of 5 15.3 and 23.0; 256 of 5 40.8 and 32.0; 80 of 3 18.3 and 14.1; 1024 of 3
// 88.8 and 94.1.
constexpr int cut_from(bool mma) { return mma ? 5 : 3; }

Plan plan_of(const fd_attn_args* a) {
  Plan p;
  int dev = 0, sms = 0;
  if (fdh::device_sms(&dev, &sms) != FD_OK) sms = 148;
  const int G = a->num_heads / a->num_kv_heads;
  const int64_t q = a->max_q_len > 0 && a->max_q_len < a->num_tokens ? a->max_q_len : a->num_tokens;
  const bool mma = at::mma_covers(a);
  // as many columns as there are rows, if the caller is right.  32 requests of
  // tokens x 4 heads over 4096 keys, with 16, 32 and 128 columns: 1 token 46, 46 and
  // 83 us; 4 47, 47 and 84; 8 64, 49 and 84; 16 111, 74 and 84; 32 205, 129 and 86.
  // (33 to 64 rows would take 32 columns by these; 8 requests over 2048 keys gain
  // 1.7 of 18.1)
  p.cols = !mma ? 0 : q * G <= 16 ? 16 : q * G <= 32 ? 32 : 128;
  p.ctas = mma ? sms : sms * ctas_of(a->head_size <= 64 ? 64 : a->head_size <= 128 ? 128 : 256);
  if (p.ctas > kMaxCtas) p.ctas = kMaxCtas;
  const int tq = (mma ? p.cols : kRows) / G, keys = mma ? kMaxKeys : kKeys;
  const int64_t chunks = (q + tq - 1) / tq;
  p.whole = p.cols == 16 || p.cols == 32 || chunks < cut_from(mma);
  if (!p.whole && a->max_k_len > 0) {
    const int64_t items = ((int64_t)a->max_k_len + keys - 1) / keys * a->n * a->num_kv_heads;
    p.whole = items <= p.ctas && chunks * (p.ctas - items) < cut_from(mma) * (int64_t)p.ctas;
  }
  // a grid of items: whole ones, at most two for each CTA that runs at once (where lengths differ most are not there).
  // 320 items of one chunk 12.1 us, looked for 16.1; 80 6.3 and 10.1
  p.tiles = 0;
  if (!mma && p.whole && a->max_k_len > 0 && a->n <= 65535 && a->num_kv_heads <= 65535) {
    const int64_t tiles = ((int64_t)a->max_k_len + keys - 1) / keys;
    if (tiles * a->n * a->num_kv_heads <= 2 * p.ctas) p.tiles = (int)tiles;
  }
  return p;
}

}  // namespace kw
}  // namespace fdk

extern "C" size_t fd_key_weights_workspace_size(const fd_key_weights_args* a) {
  if (a == nullptr || a->attn.head_size <= 0 || a->attn.head_size > 256) return 0;
  if (a->attn.n <= 0 || a->attn.num_tokens <= 0) return 0;  // nothing to do
  if (a->attn.num_kv_heads <= 0 || a->attn.num_heads < a->attn.num_kv_heads ||
      a->attn.num_heads / a->attn.num_kv_heads > fdk::kw::kRows)
    return 0;
  return fdk::kw::base_workspace(fdk::kw::plan_of(&a->attn)) + fdk::at::stage_bytes(&a->attn);
}

extern "C" int fd_key_weights(const fd_key_weights_args* args, void* stream) {
  using namespace fdk;
  const char* what = "fd_key_weights";
  if (args == nullptr) return fdh::fail(FD_ERR_INVALID, "%s: null args", what);
  const fd_attn_args* a = &args->attn;
  kw::KwParams p{};
  bool empty = false;
  int st = at::fill_params(a, at::kWeights, what, p.a, &empty);
  if (st != FD_OK || empty) return st;
  if (args->stats.num_blocks < 0 ||
      (args->stats.num_blocks > 0 && (args->stats.weights == nullptr || args->stats.positions == nullptr)))
    return fdh::fail(FD_ERR_INVALID, "%s: stats need weights and positions", what);
  const size_t need = fd_key_weights_workspace_size(args);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need || !fdh::aligned16(a->workspace)))
    return fdh::fail(FD_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  p.weights = args->stats.weights;
  p.positions = args->stats.positions;
  p.nstat = args->stats.num_blocks;
  p.evicted = args->evicted;
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  const kw::Plan plan = kw::plan_of(a);
  if (!plan.whole) {
    p.cuts = reinterpret_cast<kw::Cut*>(ws);
    p.parts = reinterpret_cast<float*>(ws + kw::cut_bytes());
  }
  st = at::stage_launch(p.a, a, kw::base_workspace(plan), true, s);
  if (st != FD_OK) return st;
  p.a.ctas = plan.ctas;
  p.a.snap = plan.whole;
  if (plan.cols > 0) return kw::mma_launch(p, a, plan, s);
  p.a.tq = kw::kRows / p.a.G;
  switch (a->dtype) {
    case FD_DTYPE_F16:
      return kw::core_launch<__half>(p, plan, s);
    case FD_DTYPE_BF16:
      return kw::core_launch<__nv_bfloat16>(p, plan, s);
    default:
      return kw::core_launch<float>(p, plan, s);
  }
}

extern "C" size_t fd_key_weights_args_bytes(void) { return sizeof(fd_key_weights_args); }
