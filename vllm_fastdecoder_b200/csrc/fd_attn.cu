// Chunk and cross attention on the CUDA cores, the combine of cut items, and
// the host side of both entry points.
//
// fd_attn_kernel takes what the tensor-core kernels (fd_attn_mma.cu,
// fd_attn_rows.cu) do not: fp32, and 16-bit heads of fewer than 64 or more
// than 128 dims.  With q the tile's rows and j
// its keys, for every key tile
//   s = scale log2(e) q.K^T,  m' = max(m, max_j s),  p = 2^(s - m'),
//   l = l 2^(m - m') + sum_j p,  O = O 2^(m - m') + p V
// and o = O / l, lse = ln 2 (m + log2 l), all in fp32.  A CTA of 16 x 16
// threads holds 64 rows and 64 keys (32 for heads of more than 64 dims) in
// shared memory as fp32; thread (y, x) owns rows 4 y .. 4 y + 3: the scores of
// keys x, x + 16, .. and D / 16 dims of O in registers.  A float4 of K or V
// then feeds 4 rows, one of Q or P 4 keys or dims (64 FMAs per 12
// shared-memory wavefronts of a warp), which keeps the fp32 pipe the bound,
// and four warps per scheduler hide each other's latencies (8 x 4 scores in
// half the threads took 2.1 cycles per FMA).  The next tile's K/V are fetched
// into registers during this one's products.

#include "fd_attn.cuh"

namespace fdk {
namespace at {

constexpr int kRows = 64;   // rows per tile
constexpr int kThreads = 256;
constexpr int kFixed = 1;   // an item's fixed cost in key tiles
constexpr int kMinPer = 1;  // least positions of a CTA (9 tokens of 32 heads over 300 keys: 15.6 us; with 2, 20.3)
// Key tiles whose saving does not pay for a cut (whole_items): 9 tokens of 2
// requests and 8 kv heads, 64 keys 12.0 us, cut 12.8; 128 keys 17.4 and 14.6.
constexpr int kWhole = 1;
constexpr int kMaxCtas = 320;

// Keys per tile (heads of up to 64 dims, 8 x 256 tokens of 32 heads over 1024
// keys: 570 us, with 32 keys 604; larger heads have shared memory for 32).
constexpr int keys_of(int DP) { return DP <= 64 ? 64 : 32; }
constexpr int ctas_of(int DP) { return DP <= 128 ? 2 : 1; }  // CTAs per SM
constexpr int smem_bytes(int DP) {
  return ((kRows + 2 * keys_of(DP)) * (DP + 4) + kRows * (keys_of(DP) + 4)) * 4;
}

// Byte offset of K (and V) row j of the request for kv head kh within its tier,
// -1 when there is none (behind klen, or a block id outside both tiers).
__device__ __forceinline__ int64_t key_offset(const AttnParams& p, const Req& q, int r, int kh, int j, int* tier) {
  *tier = 0;
  if (j >= q.klen) return -1;
  if (p.bt == nullptr) return ((int64_t)q.kbase + j) * p.tok_sb[0] + kh * p.head_sb[0];
  int64_t id = p.bt[(int64_t)q.kbase * p.bt_stride + j / p.BS];
  const int t = locate(p, r, j / p.BS, id);
  if (t < 0) return -1;
  *tier = t;
  return id * p.blk_sb[t] + kh * p.head_sb[t] + (int64_t)(j % p.BS) * p.tok_sb[t];
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, ctas_of(DP)) fd_attn_kernel(const __grid_constant__ AttnParams p) {
  constexpr int VE = 16 / (int)sizeof(T);      // elements per 16-byte load
  constexpr int NV = DP / VE;                  // loads per row
  constexpr int kKeys = keys_of(DP);
  constexpr int KN = kKeys / 16;               // keys of a thread
  constexpr int LD = DP + 4;                   // row stride of the tiles (floats)
  constexpr int LP = kKeys + 4;                // row stride of P
  constexpr int kDim4 = DP / 64;               // float4 of O per row and thread
  constexpr int kVecs = kKeys * NV / kThreads;  // loads of K (and of V) per thread and tile
  typedef Sched<kKeys, false, kFixed> Walk;
  extern __shared__ float4 smem4[];
  float* sq = reinterpret_cast<float*>(smem4);
  float* sk = sq + kRows * LD;
  float* sv = sk + kKeys * LD;
  float* sp = sv + kKeys * LD;  // [kRows][LP]
  __shared__ typename Walk::Scratch scratch;
  __shared__ const unsigned char* k_row[kKeys];
  __shared__ const unsigned char* v_row[kKeys];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int cta = blockIdx.x;
  const int D = p.D, nvec = D / VE;

  griddep_launch_dependents();  // the combine's CTAs may start, and wait for this grid's end
  if (tid == 0) p.cuts[cta].nparts = 0;
  Walk walk(p);
  if (!walk.template init<kThreads>(&scratch, cta, kMinPer)) return;

  // 16 bytes of a tile's row as fp32
  auto put = [&](float* dst, int x, const uint4& v) {
    float f[VE];
    Dt<T>::widen(v, f);
#pragma unroll
    for (int e = 0; e < VE; e += 4)
      *reinterpret_cast<float4*>(dst + x / NV * LD + x % NV * VE + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
  };
  typename Walk::Seg g;
  while (walk.next(g)) {
    const Req rq = walk.rq;
    const int tok0 = g.tile0 * p.tq;
    const int rows = min(p.tq, rq.qlen - tok0) * p.G;
    const bool active = (ty & ~1) * 4 < rows;  // some row of this warp is real
    const int lim0 = p.bt != nullptr ? rq.klen - rq.qlen + tok0 : rq.klen - 1;  // last key that the first token sees
    float m[4], l[4];
    ulonglong2 o[4][kDim4];  // four dims, packed in pairs
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < kDim4; ++d) o[i][d] = make_ulonglong2(0ull, 0ull);
    }
    uint4 kr[kVecs], vr[kVecs];
    auto fetch = [&](int j) {  // all threads: key tile j into registers (zeros where there is no key or dim)
      if (tid < kKeys) {
        int t;
        const int64_t at = key_offset(p, rq, walk.r, g.kh, j * kKeys + tid, &t);
        k_row[tid] = at < 0 ? nullptr : p.k[t] + at;
        v_row[tid] = at < 0 ? nullptr : p.v[t] + at;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const int x = tid + u * kThreads, row = x / NV, c = x % NV;
        const bool real = c < nvec && k_row[row] != nullptr;
        kr[u] = real ? *reinterpret_cast<const uint4*>(k_row[row] + c * 16) : make_uint4(0u, 0u, 0u, 0u);
        vr[u] = real ? *reinterpret_cast<const uint4*>(v_row[row] + c * 16) : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    __syncthreads();  // the last segment's reads of shared memory are done
    if (g.j0 < g.j1) {
      fetch(g.j0);
#pragma unroll 4
      for (int x = tid; x < kRows * NV; x += kThreads) {  // the query rows, zeros behind them
        const int row = x / NV, c = x % NV, t = row / p.G;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows && c < nvec)
          v = *reinterpret_cast<const uint4*>(p.q + (int64_t)(rq.qst + tok0 + t) * p.q_st +
                                              (int64_t)(g.kh * p.G + row - t * p.G) * p.q_sh + c * 16);
        put(sq, x, v);
      }
    }
    for (int j = g.j0; j < g.j1; ++j) {
      __syncthreads();  // the last tile's reads are done
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        put(sk, tid + u * kThreads, kr[u]);
        put(sv, tid + u * kThreads, vr[u]);
      }
      __syncthreads();
      if (j + 1 < g.j1) fetch(j + 1);
      if (!active) continue;
      // even and odd dims' sums in the two halves of a packed FMA
      float s[4][KN];
      f2_t s2[4][KN];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < KN; ++c) s2[i][c] = 0ull;
#pragma unroll 2
      for (int d = 0; d < D; d += 4) {
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
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < KN; ++c) {
          float even, odd;
          f2_unpack(s2[i][c], even, odd);
          s[i][c] = even + odd;
        }
      const bool cut = j * kKeys + kKeys - 1 > lim0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 4 * ty + i;
        const int lim = row >= rows ? -1 : p.bt != nullptr ? lim0 + row / p.G : lim0;
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < KN; ++c) {
          s[i][c] = cut && j * kKeys + tx + 16 * c > lim ? -INFINITY : s[i][c] * p.sl2;
          mx = fmaxf(mx, s[i][c]);
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float mn = fmaxf(m[i], mx);
        const float base = mn == -INFINITY ? 0.f : mn;  // no key seen so far: every p is 2^-inf = 0
        const float alpha = ex2_approx(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < KN; ++c) {
          const float e = ex2_approx(s[i][c] - base);
          sp[row * LP + tx + 16 * c] = e;
          sum += e;
        }
        l[i] = l[i] * alpha + sum;  // this thread's keys; the row's threads are added up at the end
        m[i] = mn;
        const f2_t alpha2 = f2_pack(alpha, alpha);
#pragma unroll
        for (int d = 0; d < kDim4; ++d) {
          o[i][d].x = f2_mul(o[i][d].x, alpha2);
          o[i][d].y = f2_mul(o[i][d].y, alpha2);
        }
      }
      __syncwarp();  // a row's P is written and read by one half-warp
#pragma unroll 1
      for (int c = 0; c < kKeys; c += 4) {
        float4 a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(sp + (4 * ty + i) * LP + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int d = 0; d < kDim4; ++d) {
            const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(sv + (c + e) * LD + 64 * d + 4 * tx);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float w = e == 0 ? a[i].x : e == 1 ? a[i].y : e == 2 ? a[i].z : a[i].w;
              const f2_t w2 = f2_pack(w, w);
              o[i][d].x = f2_fma(w2, b.x, o[i][d].x);
              o[i][d].y = f2_fma(w2, b.y, o[i][d].y);
            }
          }
        }
      }
    }
    // the rows' results, or this segment's partials
    const int slot = 2 * cta + (g.j0 > 0 ? 0 : 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float li = l[i];
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) li += __shfl_xor_sync(0xffffffffu, li, off);
      const int row = 4 * ty + i;
      if (row >= rows) continue;
      const int t = row / p.G;
      const int64_t tok = rq.qst + tok0 + t;
      const int h = g.kh * p.G + row - t * p.G;
      if (!g.whole) {
        float4* po = reinterpret_cast<float4*>(p.part_o) + (int64_t)slot * (D / 4) * kRows + row;
        if (tx == 0)
          reinterpret_cast<float2*>(p.part_ml)[(int64_t)slot * kRows + row] = make_float2(m[i], li);
#pragma unroll
        for (int d = 0; d < kDim4; ++d)
          if (64 * d + 4 * tx < D) po[(16 * d + tx) * kRows] = *reinterpret_cast<const float4*>(&o[i][d]);
        continue;
      }
      const float inv = row_inv(li);
      if (tx == 0 && p.lse != nullptr)
        p.lse[h * p.lse_sh + tok * p.lse_st] = row_lse(m[i], li);
      T* po = reinterpret_cast<T*>(p.out + tok * p.o_st + h * p.o_sh);
#pragma unroll
      for (int d = 0; d < kDim4; ++d) {
        const int c = 64 * d + 4 * tx;
        if (c >= D) continue;
        float f[4];
        f2_unpack(o[i][d].x, f[0], f[1]);
        f2_unpack(o[i][d].y, f[2], f[3]);
        T t4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t4[e] = Dt<T>::narrow(f[e] * inv);
        if (sizeof(T) == 4)
          *reinterpret_cast<uint4*>(po + c) = *reinterpret_cast<const uint4*>(t4);
        else
          *reinterpret_cast<uint2*>(po + c) = *reinterpret_cast<const uint2*>(t4);
      }
    }
    if (g.nparts > 0 && tid == 0) p.cuts[cta] = Cut{g.nparts, rq.qst + tok0, rows, g.kh};
  }
}

// The cut items' partials joined: o = sum_i O_i 2^(m_i - m) / sum_i l_i 2^(m_i - m),
// every sum in a fixed order of the parts.  CTA (c, y, z) takes rows 32 y ..
// and dims 64 z .. of the item whose first part CTA c wrote, so a long item's
// parts are read by many SMs at once.  An item of few rows and many keys has
// dozens of parts, and a thread that walked them one load after another would
// wait longer than the products took (8 items of 36 rows and 4096 keys of fp32
// heads x 64: 38.6 us in all, walked 47.8; 5 tokens over 8192 keys x 128: 22.5
// and 36): the parts' weights are taken by eight threads per row at once, and
// 16 loads of O are in flight per thread.  A warp's lanes are 8 rows times 4
// groups of 4 dims: the partials lie row by row within a group of dims (whole
// lines), and the 4 groups are 32 bytes of an output row.  A programmatic dependent of the attention kernel: its CTAs start
// while that one's last ones run (5 KB of shared memory fit beside two of the
// row kernel's), and await its end.
constexpr int kCombineRows = 32, kCombineThreads = 256, kCombineDims = 64;
constexpr int kCombineLanes = kCombineThreads / kCombineRows;  // threads per row that take weights
constexpr int kCombineParts = 32;                              // parts per round
template <typename T>
__global__ void __launch_bounds__(kCombineThreads) fd_attn_combine_kernel(const __grid_constant__ AttnParams p,
                                                                          int item_rows) {
  __shared__ float weight[kCombineParts][kCombineRows];
  __shared__ float red[kCombineLanes][kCombineRows];
  griddep_wait();
  const int c = blockIdx.x;
  const Cut cut = p.cuts[c];
  const int row0 = blockIdx.y * kCombineRows;
  if (row0 >= cut.rows || cut.nparts == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // part 0 is slot 1 of CTA c, part i slot 0 of CTA c + i
  auto slot = [&](int i) { return (int64_t)(2 * (c + i) + (i == 0 ? 1 : 0)); };
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  // warp w takes the weights of parts w, w + 8, ..: lane = row
  const bool mine = row0 + lane < cut.rows;
  float m = -INFINITY, l = 0.f;
  if (mine) {
#pragma unroll 4
    for (int i = warp; i < cut.nparts; i += kCombineLanes) m = fmaxf(m, ml[slot(i) * item_rows + row0 + lane].x);
  }
  red[warp][lane] = m;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < kCombineLanes; ++x) m = fmaxf(m, red[x][lane]);
  const float base = m == -INFINITY ? 0.f : m;
  // and adds up the O of 8 rows, two groups of dims per lane
  const int sub = (warp & 3) * 8 + (lane & 7), row = row0 + sub;
  const int groups = p.D / 4, d0 = blockIdx.z * (kCombineDims / 4) + (warp >> 2) * 4 + (lane >> 3);
  const bool ok[2] = {row < cut.rows && d0 < groups, row < cut.rows && d0 + 8 < groups};
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int i0 = 0; i0 < cut.nparts; i0 += kCombineParts) {
    const int n = min(kCombineParts, cut.nparts - i0);
    if (i0 > 0) __syncthreads();  // the last round's weights have been read
    if (mine) {
#pragma unroll
      for (int x = 0; x < kCombineParts / kCombineLanes; ++x) {
        const int i = warp + x * kCombineLanes;
        if (i >= n) break;
        const float2 v = ml[slot(i0 + i) * item_rows + row0 + lane];
        const float w = exp2f(v.x - base);
        weight[i][lane] = w;
        l += v.y * w;
      }
    }
    __syncthreads();
    if (ok[0]) {
      const float4* po = reinterpret_cast<const float4*>(p.part_o) + row;
      const int second = ok[1] ? 8 * item_rows : 0;
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float4* at = po + (slot(i0 + i) * groups + d0) * item_rows;
        const float w = weight[i][sub];
        const float4 x = at[0], y = at[second];
        acc[0].x = fmaf(w, x.x, acc[0].x);
        acc[0].y = fmaf(w, x.y, acc[0].y);
        acc[0].z = fmaf(w, x.z, acc[0].z);
        acc[0].w = fmaf(w, x.w, acc[0].w);
        acc[1].x = fmaf(w, y.x, acc[1].x);
        acc[1].y = fmaf(w, y.y, acc[1].y);
        acc[1].z = fmaf(w, y.z, acc[1].z);
        acc[1].w = fmaf(w, y.w, acc[1].w);
      }
    }
  }
  __syncthreads();  // m has been read
  red[warp][lane] = l;
  __syncthreads();
  if (warp == 0 && blockIdx.z == 0 && mine && p.lse != nullptr) {
    l = 0.f;
    for (int x = 0; x < kCombineLanes; ++x) l += red[x][lane];
    const int at = row0 + lane;
    p.lse[(cut.kh * p.G + at % p.G) * p.lse_sh + (int64_t)(cut.row0 + at / p.G) * p.lse_st] = row_lse(m, l);
  }
  if (!ok[0]) return;
  l = 0.f;
#pragma unroll
  for (int x = 0; x < kCombineLanes; ++x) l += red[x][sub];
  const float inv = row_inv(l);
  const int64_t tok = cut.row0 + row / p.G;
  T* po = reinterpret_cast<T*>(p.out + tok * p.o_st + (cut.kh * p.G + row % p.G) * p.o_sh);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (!ok[e]) continue;
    const float f[4] = {acc[e].x * inv, acc[e].y * inv, acc[e].z * inv, acc[e].w * inv};
    T t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) t[u] = Dt<T>::narrow(f[u]);
    T* const to = po + 4 * (d0 + 8 * e);
    if (sizeof(T) == 4)
      *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(t);
    else
      *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(t);
  }
}

bool whole_items(const fd_attn_args* a, int ctas, int item_rows, int keys, int most) {
  if (a->max_k_len <= 0) return false;
  const int G = a->num_heads / a->num_kv_heads;
  const int64_t q = a->max_q_len > 0 && a->max_q_len < a->num_tokens ? a->max_q_len : a->num_tokens;
  const int64_t items = (q + item_rows / G - 1) / (item_rows / G) * a->n * a->num_kv_heads;
  const int64_t tiles = ((int64_t)a->max_k_len + keys - 1) / keys;
  return items <= ctas && tiles * (ctas - items) <= (int64_t)most * ctas;
}

int combine_launch(const AttnParams& p, int dtype, int rows, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.ctas, (unsigned)((rows + kCombineRows - 1) / kCombineRows),
                     (unsigned)((p.D + kCombineDims - 1) / kCombineDims));
  cfg.blockDim = dim3(kCombineThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const void* kern = dtype == FD_DTYPE_F16    ? reinterpret_cast<const void*>(fd_attn_combine_kernel<__half>)
                     : dtype == FD_DTYPE_BF16 ? reinterpret_cast<const void*>(fd_attn_combine_kernel<__nv_bfloat16>)
                                              : reinterpret_cast<const void*>(fd_attn_combine_kernel<float>);
  void* args[2] = {const_cast<AttnParams*>(&p), &rows};
  return fdh::cuda_status(cudaLaunchKernelExC(&cfg, kern, args), "fd_attn_combine_kernel launch");
}

// Host blocks are copied to device memory first, by all SMs: read in place
// they would cross PCIe once per item that sees them (an SM's loads do not
// keep them in L2), and a few CTAs, those whose requests have spilled, would
// wait for it one tile after another.  (64 requests of up to 8 tokens and 4000
// keys, a twentieth in host memory: 678 us, in place 1190; 8 of 200 tokens and
// 2000 keys, a fifth: 365 and 1125; of one token: 286 and 279.  PCIe at ~55
// GB/s bounds it.)  CTA (j, r) copies block j of request
// r, when it lies in the host tier, to block r * stage_w + j of the copies.
constexpr int kStageThreads = 256, kStageBatch = 8;
__global__ void __launch_bounds__(kStageThreads) fd_attn_stage_kernel(const __grid_constant__ AttnParams p, int vec) {
  const int j = blockIdx.x, r = blockIdx.y;
  const Req q = load_req(p, r);
  if (q.qlen <= 0 || j * (long long)p.BS >= q.klen) return;
  const int64_t id = p.bt[(int64_t)q.kbase * p.bt_stride + j];
  if (id < p.split || id - p.split >= p.nblk[1]) return;
  const int rows = p.KVH * p.BS, total = 2 * rows * vec;  // K, then V
  const int64_t src = (id - p.split) * p.blk_sb[1], dst = ((int64_t)r * p.stage_w + j) * p.blk_sb[2];
  for (int x0 = threadIdx.x; x0 < total; x0 += kStageThreads * kStageBatch) {
    uint4 v[kStageBatch];
    int64_t to[kStageBatch];
#pragma unroll
    for (int u = 0; u < kStageBatch; ++u) {
      const int x = x0 + u * kStageThreads;
      to[u] = -1;
      if (x >= total) continue;
      const int row = x / vec % rows, c = x % vec, h = row / p.BS, t = row - h * p.BS;
      const unsigned char* base = x < rows * vec ? p.k[1] : p.v[1];
      v[u] = *reinterpret_cast<const uint4*>(base + src + h * p.head_sb[1] + t * p.tok_sb[1] + c * 16);
      to[u] = dst + h * p.head_sb[2] + t * p.tok_sb[2] + c * 16;
    }
#pragma unroll
    for (int u = 0; u < kStageBatch; ++u) {
      if (to[u] < 0) continue;
      const int x = x0 + u * kStageThreads;
      *reinterpret_cast<uint4*>(const_cast<unsigned char*>(x < rows * vec ? p.k[2] : p.v[2]) + to[u]) = v[u];
    }
  }
}

namespace {

// Blocks per request whose host-tier ones are copied (0: read in place, where
// the copies could take more than kStageBytes), and the bytes of K (and of V)
// of one.
constexpr int64_t kStageBytes = (int64_t)1 << 30;
int stage_blocks(const fd_attn_args* a, int64_t* block_bytes) {
  *block_bytes = (int64_t)a->num_kv_heads * a->block_size * a->head_size * fdh::elem_size(a->dtype);
  if (a->block_table == nullptr || !a->tier[1].host_mapped || a->tier[1].num_blocks <= 0 || a->block_size <= 0 ||
      a->num_kv_heads <= 0 || a->n <= 0)
    return 0;
  int64_t w = a->max_k_len > 0 ? ((int64_t)a->max_k_len + a->block_size - 1) / a->block_size : a->bt_width;
  if (w > a->bt_width) w = a->bt_width;
  return w * a->n * 2 * *block_bytes <= kStageBytes ? (int)w : 0;
}

size_t core_workspace(const fd_attn_args* a) {
  const size_t slots = 2 * (size_t)kMaxCtas * kRows;
  return kMaxCtas * sizeof(Cut) + slots * 2 * 4 + slots * (size_t)a->head_size * 4;
}

size_t base_workspace(const fd_attn_args* a) {
  const size_t b = mma_covers(a) ? mma_workspace(a) : core_workspace(a);
  return (b + 255) / 256 * 256;
}

template <typename T, int DP>
int core_launch_dp(AttnParams& p, const fd_attn_args* a, cudaStream_t s) {
  const int dtype = a->dtype;
  const void* kern = reinterpret_cast<const void*>(fd_attn_kernel<T, DP>);
  static unsigned long long done = 0;
  int st = fdh::ensure_smem(kern, smem_bytes(DP), &done);
  if (st != FD_OK) return st;
  int dev = 0, sms = 0;
  st = fdh::device_sms(&dev, &sms);
  if (st != FD_OK) return st;
  p.ctas = sms * ctas_of(DP);
  if (p.ctas > kMaxCtas) p.ctas = kMaxCtas;
  const dim3 grid((unsigned)p.ctas);
  p.snap = whole_items(a, p.ctas, kRows, keys_of(DP), kWhole);
  st = fdh::launch_maybe_pdl(kern, grid, dim3(kThreads), smem_bytes(DP), s, false, p, "fd_attn_kernel launch");
  if (st != FD_OK || p.snap) return st;
  return combine_launch(p, dtype, kRows, s);
}

template <typename T>
int core_launch(AttnParams& p, const fd_attn_args* a, cudaStream_t s) {
  if (p.D <= 64) return core_launch_dp<T, 64>(p, a, s);
  if (p.D <= 128) return core_launch_dp<T, 128>(p, a, s);
  return core_launch_dp<T, 256>(p, a, s);
}

// Shared checks and parameters; `what` names the entry point in messages.
int attn_impl(const fd_attn_args* a, bool chunk, const char* what, void* stream) {
  if (a == nullptr) return fdh::fail(FD_ERR_INVALID, "%s: null args", what);
  const int es = fdh::elem_size(a->dtype);
  if (es == 0) return fdh::fail(FD_ERR_UNSUPPORTED, "%s: unsupported dtype %d", what, a->dtype);
  if (a->n < 0 || a->num_tokens < 0) return fdh::fail(FD_ERR_INVALID, "%s: negative n or num_tokens", what);
  if (a->n > 65535) return fdh::fail(FD_ERR_UNSUPPORTED, "%s: %d requests (at most 65535)", what, a->n);
  if (a->num_kv_heads <= 0 || a->num_heads <= 0 || a->num_heads % a->num_kv_heads != 0)
    return fdh::fail(FD_ERR_INVALID, "%s: num_heads must be a multiple of num_kv_heads", what);
  const int G = a->num_heads / a->num_kv_heads;
  if (G > kRows) return fdh::fail(FD_ERR_UNSUPPORTED, "%s: query group %d (at most %d)", what, G, kRows);
  if (a->head_size <= 0 || a->head_size > 256)
    return fdh::fail(FD_ERR_UNSUPPORTED, "%s: head_size must be 1 to 256", what);
  if (((int64_t)a->head_size * es) % 16 != 0)
    return fdh::fail(FD_ERR_ALIGN, "%s: head_size*elem_size must be a multiple of 16", what);
  if (!(a->scale > 0.f) || !(a->scale < 3.0e38f))
    return fdh::fail(FD_ERR_INVALID, "%s: scale must be positive and finite", what);
  if (a->n == 0 || a->num_tokens == 0) return FD_OK;
  if (a->q == nullptr || a->out == nullptr || a->q_start == nullptr || a->q_len == nullptr || a->k_len == nullptr)
    return fdh::fail(FD_ERR_INVALID, "%s: q, out, q_start, q_len and k_len are required", what);
  if (chunk && (a->block_table == nullptr || a->bt_width <= 0 || a->bt_stride < 0 || a->block_size <= 0))
    return fdh::fail(FD_ERR_INVALID, "%s: block_table, bt_width and block_size are required", what);
  if (chunk && a->bt_rows < 0) return fdh::fail(FD_ERR_INVALID, "%s: bt_rows must not be negative", what);
  // no state rows at all: no pointers either, and no request has keys
  if (!chunk && (a->k_start == nullptr ||
                 (a->tier[0].num_blocks > 0 && (a->tier[0].k == nullptr || a->tier[0].v == nullptr))))
    return fdh::fail(FD_ERR_INVALID, "%s: states and k_start are required", what);
  if (!chunk && a->tier[0].host_mapped)
    return fdh::fail(FD_ERR_UNSUPPORTED, "%s: states must be device memory", what);
  if (!fdh::aligned16(a->q) || !fdh::aligned16(a->out) || (a->q_stride_t * es) % 16 != 0 ||
      (a->q_stride_h * es) % 16 != 0 || (a->out_stride_t * es) % 16 != 0 || (a->out_stride_h * es) % 16 != 0)
    return fdh::fail(FD_ERR_ALIGN, "%s: q / out pointers and strides must be 16-byte aligned", what);
  AttnParams p{};
  for (int t = 0; t < (chunk ? 2 : 1); ++t) {
    const fd_kv_tier& tr = a->tier[t];
    p.nblk[t] = tr.num_blocks > 0 ? tr.num_blocks : 0;
    if (p.nblk[t] == 0) continue;
    if (tr.k == nullptr || tr.v == nullptr)
      return fdh::fail(FD_ERR_INVALID, "%s: tier %d has blocks but no K/V pointer", what, t);
    if (!fdh::aligned16(tr.k) || !fdh::aligned16(tr.v) || (tr.blk_stride * es) % 16 != 0 ||
        (tr.head_stride * es) % 16 != 0 || (tr.tok_stride * es) % 16 != 0)
      return fdh::fail(FD_ERR_ALIGN, "%s: tier %d pointers/strides must be 16-byte aligned", what, t);
    p.k[t] = static_cast<const unsigned char*>(tr.k);
    p.v[t] = static_cast<const unsigned char*>(tr.v);
    p.blk_sb[t] = tr.blk_stride * es;
    p.head_sb[t] = tr.head_stride * es;
    p.tok_sb[t] = tr.tok_stride * es;
    p.host[t] = tr.host_mapped ? 1 : 0;
  }
  p.split = chunk ? a->tier_split : 0;
  p.q = static_cast<const unsigned char*>(a->q);
  p.out = static_cast<unsigned char*>(a->out);
  p.lse = a->lse;
  p.q_st = a->q_stride_t * es;
  p.q_sh = a->q_stride_h * es;
  p.o_st = a->out_stride_t * es;
  p.o_sh = a->out_stride_h * es;
  p.lse_sh = a->lse_stride_h;
  p.lse_st = a->lse_stride_t;
  p.bt = chunk ? a->block_table : nullptr;
  p.bt_stride = a->bt_stride;
  p.bt_row = a->bt_row;
  p.k_start = a->k_start;
  p.q_start = a->q_start;
  p.q_len = a->q_len;
  p.k_len = a->k_len;
  p.bt_width = a->bt_width;
  p.bt_rows = a->bt_rows;
  p.n = a->n;
  p.T = a->num_tokens;
  p.H = a->num_heads;
  p.KVH = a->num_kv_heads;
  p.G = G;
  p.D = a->head_size;
  p.BS = chunk ? a->block_size : 1;
  p.sl2 = a->scale * kLog2e;
  p.err = a->error;
  const size_t need = fd_attn_workspace_size(a);
  if (a->workspace == nullptr || a->workspace_bytes < need || !fdh::aligned16(a->workspace))
    return fdh::fail(FD_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int64_t block_bytes = 0;
  p.stage_w = chunk ? stage_blocks(a, &block_bytes) : 0;
  if (p.stage_w > 0) {
    const int64_t blocks = (int64_t)p.stage_w * p.n;
    const unsigned char* at = static_cast<const unsigned char*>(a->workspace) + base_workspace(a);
    p.k[2] = at;
    p.v[2] = at + blocks * block_bytes;
    p.tok_sb[2] = (int64_t)p.D * es;
    p.head_sb[2] = p.tok_sb[2] * p.BS;
    p.blk_sb[2] = block_bytes;
    p.nblk[2] = blocks;
    fd_attn_stage_kernel<<<dim3((unsigned)p.stage_w, (unsigned)p.n), kStageThreads, 0, s>>>(p, p.D * es / 16);
    const int st = fdh::cuda_status(cudaGetLastError(), "fd_attn_stage_kernel launch");
    if (st != FD_OK) return st;
  }
  if (mma_covers(a)) return mma_launch(p, a, s);
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  p.cuts = reinterpret_cast<Cut*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + kMaxCtas * sizeof(Cut));
  p.part_o = p.part_ml + 2 * (size_t)kMaxCtas * kRows * 2;
  p.tq = kRows / G;
  switch (a->dtype) {
    case FD_DTYPE_F16:
      return core_launch<__half>(p, a, s);
    case FD_DTYPE_BF16:
      return core_launch<__nv_bfloat16>(p, a, s);
    default:
      return core_launch<float>(p, a, s);
  }
}

}  // namespace
}  // namespace at
}  // namespace fdk

extern "C" size_t fd_attn_workspace_size(const fd_attn_args* a) {
  if (a == nullptr || a->head_size <= 0 || a->head_size > 256) return 0;
  int64_t block_bytes = 0;
  const int w = fdk::at::stage_blocks(a, &block_bytes);
  return fdk::at::base_workspace(a) + (size_t)(2 * (int64_t)w * a->n * block_bytes);
}

extern "C" int fd_chunk_attn(const fd_attn_args* a, void* stream) {
  return fdk::at::attn_impl(a, true, "fd_chunk_attn", stream);
}

extern "C" int fd_cross_attn(const fd_attn_args* a, void* stream) {
  return fdk::at::attn_impl(a, false, "fd_cross_attn", stream);
}

extern "C" size_t fd_attn_args_bytes(void) { return sizeof(fd_attn_args); }
