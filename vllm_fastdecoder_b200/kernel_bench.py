"""Per-kernel timings of the engine's smaller kernels (one JSON line per case).

    python -m vllm_fastdecoder_b200.kernel_bench [case ...] [--launches N]

The decode kernels and their combine are timed by bench.py on the benchmark
workloads; this covers the rest, each on inputs sized like the workload it
serves (and larger than the 126 MB L2 where the kernel streams data):

  store_kv_prefill  fd_store_kv_kernel: 16384 new tokens x 32 kv heads x D128
                    fp16 into the HBM tier (a prefill-sized write)
  store_kv_decode   fd_store_kv_kernel: 128 new tokens, half of them into the
                    mapped host tier (a decode step of config 4)
  merge2            fd_merge2_kernel: two fp16 partials of 4096 rows x 32
                    heads x D128 merged into one (the two-tier merge)
  merge_partials    fd_mergeP_kernel: 8 fp32 partials of 8 rows x 32 heads x
                    D128 (config 3's merge at 8 GPUs)
  split_merge       fd_split_merge_kernel: the split-grid combine of config 2
                    (tiles_per_split 16)
  combine           fd_persistent_combine_kernel: the persistent schedule's
                    merge of cut segments, config 2
  host_mapped       fd_decode_kernel reading only the host tier in place over
                    PCIe (pinned, device-mapped): 16 rows x 4096 tokens, 32/32
                    heads, D128, fp16 (1.07 GB in host memory)
  prefill           fd_prefill_kernel: 8 requests of 1024 new queries over
                    1024 cached + 1024 new keys (causal), 32/8 heads, D128,
                    bf16, paged HBM tier (achieved TFLOP/s against the
                    measured dense bf16 peak)
  prefill_fa        the same prefill through FlashAttention, the library the
                    reference calls for these rows: vLLM's
                    flash_attn_varlen_func over the paged cache when its
                    extension loads, else flash-attn 2.8 over the gathered
                    K/V (a baseline timing, not this engine's path)
  plan              fd_plan_kernel: the device planner on a 128-request
                    decode step of the config-4 trace
  exchange1         fd_exchange_merge_kernel with one rank (push, flags, merge
                    of config 3's partial)
  weights_few       fd_keyw_mma_kernel: weights that 32 requests of 4 new tokens
                    give to 4096 keys each, 32/8 heads, D128, bf16
  weights_many      the same kernel: 2 requests of 2048 tokens over 8192 keys
  select_keys       fd_select_kernel: 32 requests x 8 heads, 2048 of 2080 keys
  move_keys         fd_move_kernel: 4 requests x 8 heads cut from 16384 to 2048
                    keys of D128 bf16
  trim_tables       fd_trim_kernel: 100 requests from 8192 to 2048 tokens
  verify_drafts     fd_verify_kernel: 64 requests of 4 drafts over 131072 fp32
                    probabilities
  extend_tables     fd_tables_kernel: block tables, slots and positions of 601
                    requests with 0 to 400 new tokens over up to 1000 cached
  rope_store_kv     fd_rope_kernel: 16384 tokens x 32/8 heads x D128 bf16, three
                    position axes, q in place, k and v to the HBM tier
  chunk_few         fd_attn_rows_kernel: 32 requests of 4 new tokens over 4096
                    keys, 32/8 heads, D128, bf16 (bytes of the cache)
  chunk_many        fd_attn_mma_kernel: 2 requests of 2048 new tokens over 8192
                    keys, same heads (achieved TFLOP/s)
  cross_few         fd_attn_rows_kernel: 24 requests of one token over 1500
                    encoder states, 20 heads, D64, fp16
  cross_fp32        fd_attn_kernel: 4 requests of 64 tokens over 1500 encoder
                    states, 8 heads, D64, fp32 (achieved TFLOP/s)

Each line: the kernel, the mean device time per launch (CUDA events around
`--launches` back-to-back launches after warm-up), the algorithmic bytes per
launch, and achieved GB/s against the measured HBM copy rate (for
host_mapped: against a pinned host-to-device cudaMemcpyAsync of the same
bytes timed in the same run, and against PCIe Gen5 x16's nominal 63 GB/s).
"""

from __future__ import annotations

import argparse
import json
import math
from pathlib import Path

import torch

from vllm_fastdecoder_b200 import gpu_ops, workloads
from vllm_fastdecoder_b200.gpu_ops import KVTier

ROOT = Path(__file__).resolve().parents[1]
PCIE5_X16_GBS = 63.0  # PCIe Gen5 x16, per direction, nominal (32 GT/s x 16 lanes, 128b/130b)


def _hbm_peak() -> float:
    p = ROOT / "MEASURED_PEAKS.json"
    return float(json.loads(p.read_text())["hbm_gbs"]) if p.exists() else 6650.0


def _bf16_peak() -> float:
    p = ROOT / "MEASURED_PEAKS.json"
    return float(json.loads(p.read_text())["bf16_tflops"]) if p.exists() else 1590.0


def _time(fn, launches: int, warmup: int = 3) -> float:
    for _ in range(warmup):
        fn()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(launches):
        fn()
    e1.record()
    torch.cuda.synchronize()
    return e0.elapsed_time(e1) * 1e-3 / launches


def case_store_kv(dev, host_half: bool):
    m, KVH, D, BS, dt = (16384, 32, 128, 16, torch.float16) if not host_half else (128, 32, 128, 16, torch.float16)
    G = 8192 if not host_half else 2048
    phys = torch.zeros(G, BS, KVH, 2 * D, dtype=dt, device=dev)  # vLLM NHD [B, BS, KVH, 2D]
    cache = phys.permute(0, 2, 1, 3)
    tiers = [KVTier(cache[..., :D], cache[..., D:]), None]
    C = 0
    if host_half:
        C = 512
        hk = torch.zeros(C, KVH, BS, D, dtype=dt, pin_memory=True)
        hv = torch.zeros(C, KVH, BS, D, dtype=dt, pin_memory=True)
        tiers[1] = KVTier(hk, hv)
    g = torch.Generator().manual_seed(0)
    slots = torch.randperm((G + C) * BS, generator=g)[:m].to(torch.int64)
    if host_half:  # half the rows to the host tier, half to HBM
        slots[: m // 2] = torch.randperm(C * BS, generator=g)[: m // 2] + G * BS
        slots[m // 2:] = torch.randperm(G * BS, generator=g)[: m - m // 2]
    slots = slots.to(dev)
    k = torch.randn(m, KVH, D, dtype=dt, device=dev)
    v = torch.randn(m, KVH, D, dtype=dt, device=dev)
    nbytes = 2 * m * KVH * D * 2 * 2 + m * 8  # K and V read and written, slots read
    return (lambda: gpu_ops.store_kv_tiered(k, v, slots, tuple(tiers), G)), nbytes, "fd_store_kv_kernel"


def case_merge2(dev):
    n, H, D, dt = 4096, 32, 128, torch.float16
    o_a = torch.randn(n, H, D, dtype=dt, device=dev)
    o_b = torch.randn(n, H, D, dtype=dt, device=dev)
    la = torch.randn(H, n, device=dev)
    lb = torch.randn(H, n, device=dev)
    out = torch.empty(n, H, D, dtype=dt, device=dev)
    out_lse = torch.empty(H, n, device=dev)
    nbytes = 3 * n * H * D * 2 + 3 * H * n * 4
    return (lambda: gpu_ops.merge_attn_states(out, o_a, la, o_b, lb, out_lse)), nbytes, "fd_merge2_kernel"


def case_merge_partials(dev):
    P, n, H, D = 8, 8, 32, 128
    stride = n * H * D + H * n
    parts = torch.randn(P, stride, device=dev)
    out = torch.empty(n, H, D, dtype=torch.bfloat16, device=dev)
    out_lse = torch.empty(H, n, device=dev)
    nbytes = P * stride * 4 + n * H * D * 2 + H * n * 4
    return (lambda: gpu_ops.merge_partials(parts, P, n, H, D, out, out_lse)), nbytes, "fd_mergeP_kernel"


def case_split_merge(dev):
    b = workloads.config2()
    res = workloads.materialize(b, dev)
    out = torch.empty(b.n, b.H, b.D, dtype=b.dtype, device=dev)
    lse = torch.empty(b.H, b.n, dtype=torch.float32, device=dev)
    a = gpu_ops.decode_args(res.q, res.tiers, b.G, res.block_table, res.lens, b.scale, out, lse,
                            max_len=int(b.lens.max()), tiles_per_split=16)
    gpu_ops.launch_decode(a, dev, "partials")
    torch.cuda.synchronize()
    # the merge reads every split's fp32 partial (o and lse) of every row-head
    tiles = [(int(L) + 15) // 16 for L in b.lens]
    splits = sum((t + 15) // 16 for t in tiles if (t + 15) // 16 > 1)
    rows_split = sum(1 for t in tiles if (t + 15) // 16 > 1)
    nbytes = splits * b.H * (b.D + 1) * 4 + rows_split * b.H * (b.D * 2 + 4)
    return (lambda: gpu_ops.launch_decode(a, dev, "combine")), nbytes, "fd_split_merge_kernel"


def case_combine(dev):
    b = workloads.config2()
    res = workloads.materialize(b, dev)
    out = torch.empty(b.n, b.H, b.D, dtype=b.dtype, device=dev)
    lse = torch.empty(b.H, b.n, dtype=torch.float32, device=dev)
    a = gpu_ops.decode_args(res.q, res.tiers, b.G, res.block_table, res.lens, b.scale, out, lse,
                            max_len=int(b.lens.max()))
    gpu_ops.launch_decode(a, dev, "partials")
    torch.cuda.synchronize()
    # every decode CTA's two fp32 partial slots (GQ heads of D + 1 floats)
    # are read at most once, and one merged segment (GQ heads of D outputs
    # and an lse) is written per CTA at most: an upper bound of the bytes the
    # kernel must move.  The tensor-core decode runs one CTA per SM.
    ctas = torch.cuda.get_device_properties(dev).multi_processor_count
    gq = b.H // b.KVH
    nbytes = ctas * 2 * gq * (b.D + 1) * 4 + ctas * gq * (b.D * 2 + 4)
    return (lambda: gpu_ops.launch_decode(a, dev, "combine")), nbytes, "fd_persistent_combine_kernel"


def case_host_mapped(dev):
    n, H, D, BS, L, dt = 16, 32, 128, 16, 4096, torch.float16
    nb = L // BS
    C = n * nb
    g = torch.Generator().manual_seed(3)
    hk = torch.empty(C, H, BS, D, dtype=dt, pin_memory=True)
    hv = torch.empty(C, H, BS, D, dtype=dt, pin_memory=True)
    tmp = torch.empty(nb, H, BS, D, dtype=dt, device=dev)
    for dst in (hk, hv):
        for r in range(n):
            tmp.normal_()
            dst[r * nb:(r + 1) * nb].copy_(tmp)
    del tmp
    bt = torch.randperm(C, generator=g).to(torch.int32).view(n, nb).to(dev)  # host ids from tier_split 0
    lens = torch.full((n,), L, dtype=torch.int32, device=dev)
    q = torch.randn(n, H, D, dtype=dt, device=dev)
    out = torch.empty(n, H, D, dtype=dt, device=dev)
    lse = torch.empty(H, n, dtype=torch.float32, device=dev)
    tiers = (None, KVTier(hk, hv))
    torch.cuda.synchronize()
    nbytes = 2 * n * L * H * D * 2 + n * H * (2 * D * 2 + 4) + n * nb * 4
    return (lambda: gpu_ops.decode_tiered(q, tiers, 0, bt, lens, 1.0 / math.sqrt(D), out, lse)), nbytes, \
        "fd_decode_kernel"


def pinned_copy_gbs(dev, nbytes: int = 1 << 30) -> float:
    """Pinned host-to-device cudaMemcpyAsync rate (GB/s), the PCIe reference."""
    src = torch.empty(nbytes, dtype=torch.uint8, pin_memory=True)
    dst = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    t = _time(lambda: dst.copy_(src, non_blocking=True), 5, warmup=2)
    return nbytes / t / 1e9


def case_prefill(dev):
    n, ql, kl, H, KVH, D, BS, dt = 8, 1024, 2048, 32, 8, 128, 16, torch.bfloat16
    nb = kl // BS
    g = torch.Generator().manual_seed(4)
    phys = torch.empty(n * nb + 8, BS, KVH, 2 * D, dtype=dt, device=dev).normal_()
    cache = phys.permute(0, 2, 1, 3)
    kv = KVTier(cache[..., :D], cache[..., D:])
    bt = torch.randperm(n * nb + 8, generator=g)[: n * nb].to(torch.int32).view(n, nb).to(dev)
    q = torch.randn(n * ql, H, D, dtype=dt, device=dev)
    out = torch.empty_like(q)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    qs, qls, kls = i32([i * ql for i in range(n)]), i32([ql] * n), i32([kl] * n)
    # causal: query i sees kl - ql + i + 1 keys; 4 flops per (query, key, dim, head)
    keys_seen = sum(kl - ql + i + 1 for i in range(ql)) * n
    flops = 4 * keys_seen * H * D
    return (lambda: gpu_ops.prefill_attn(q, out, qs, qls, kls, 1.0 / math.sqrt(D), kv=kv, block_table=bt,
                                         total_q=n * ql)), flops, "fd_prefill_kernel"


def case_prefill_fa(dev):
    n, ql, kl, H, KVH, D, BS, dt = 8, 1024, 2048, 32, 8, 128, 16, torch.bfloat16
    nb = kl // BS
    g = torch.Generator().manual_seed(4)
    phys = torch.empty(n * nb + 8, BS, KVH, 2 * D, dtype=dt, device=dev).normal_()
    bt = torch.randperm(n * nb + 8, generator=g)[: n * nb].to(torch.int32).view(n, nb).to(dev)
    q = torch.randn(n * ql, H, D, dtype=dt, device=dev)
    cu_q = torch.arange(0, (n + 1) * ql, ql, dtype=torch.int32, device=dev)
    keys_seen = sum(kl - ql + i + 1 for i in range(ql)) * n
    flops = 4 * keys_seen * H * D
    scale = 1.0 / math.sqrt(D)
    try:  # the reference's own call (fastdecode/backend.py:317-329)
        from vllm.vllm_flash_attn import flash_attn_varlen_func as fa

        k_cache, v_cache = phys[..., :D], phys[..., D:]  # [B, BS, KVH, D] views
        seqused = torch.full((n,), kl, dtype=torch.int32, device=dev)
        fn = lambda: fa(q=q, k=k_cache, v=v_cache, cu_seqlens_q=cu_q, max_seqlen_q=ql, seqused_k=seqused,  # noqa: E731
                        max_seqlen_k=kl, softmax_scale=scale, causal=True, block_table=bt, fa_version=2)
        fn()
        return fn, flops, "vllm_flash_attn (fa2, paged)"
    except Exception:
        from flash_attn import flash_attn_varlen_func as fa

        k = phys[bt.long().flatten()].reshape(n * kl, KVH, 2 * D)
        kc, vc = k[..., :D].contiguous(), k[..., D:].contiguous()
        cu_k = torch.arange(0, (n + 1) * kl, kl, dtype=torch.int32, device=dev)
        fn = lambda: fa(q, kc, vc, cu_q, cu_k, ql, kl, softmax_scale=scale, causal=True)  # noqa: E731
        fn()
        return fn, flops, "flash_attn 2.8 (gathered K/V)"


def case_plan(dev):
    from vllm_fastdecoder_b200 import plan

    tr = workloads.trace4(seed=0, steps=1)
    st = tr.steps[0]
    R = st.rows
    qsl = torch.arange(R + 1, dtype=torch.int32, device=dev)
    lens, bt, slots = st.lens.to(dev), st.block_table.to(dev), st.slots.to(dev)
    out = plan.DeviceStepPlan(R, R, bt.shape[1], dev)

    def run():
        plan.plan_on_device(qsl, lens, bt, slots, tr.G, tr.host_blocks, tr.BS, out=out, max_tokens=R)

    nbytes = bt.numel() * 4 * 3 + R * (4 * 4 + 8 * 8)  # table read, two compacted tables written, lists
    return run, nbytes, "fd_plan_kernel"


def case_exchange1(dev):
    from vllm_fastdecoder_b200 import sharded

    n, H, D = 8, 32, 128
    ex = sharded.PeerExchange(n, H, D, 1, dev)
    ex.o_view.normal_()
    ex.lse_view.normal_()
    final = torch.empty(n, H, D, dtype=torch.bfloat16, device=dev)
    nbytes = 2 * ex.slot * 4 + ex.slot * 4 + n * H * D * 2  # read send, write + read the slot, write out
    return (lambda: ex.exchange_and_merge(None, None, final)), nbytes, "fd_exchange_merge_kernel"


def case_extend_tables(dev):
    R, bs, T = 601, 16, 131072
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 401, (R,), generator=g, dtype=torch.int32)
    prior = torch.randint(0, 1001, (R,), generator=g, dtype=torch.int32)
    held, after = -(-prior // bs), -(-(prior + new) // bs)
    W, need, n_held = 96, int((after - held).sum()), int(held.sum())
    table = torch.full((R, W), -1, dtype=torch.int32)
    table[torch.arange(W) < held[:, None]] = torch.arange(n_held, dtype=torch.int32)
    free = gpu_ops.FreeBlocks(torch.arange(n_held, n_held + need, dtype=torch.int32, device=dev), None,
                              torch.tensor([need, 0], dtype=torch.int32, device=dev))
    new, prior, table = new.to(dev), prior.to(dev), table.to(dev)
    out = gpu_ops.StepTables(R, T, dev)
    nbytes = 16 * R + 8 * need + 16 * T
    return lambda: gpu_ops.extend_tables(new, prior, table, free, n_held + need, 0, bs, out), nbytes, "fd_tables_kernel"


def case_rope_store_kv(dev):
    T, H, KVH, D, bs, max_pos = 16384, 32, 8, 128, 16, 16384
    q, k, v = (torch.randn(T, h, D, device=dev, dtype=torch.bfloat16) for h in (H, KVH, KVH))
    pos = torch.randint(0, max_pos, (3, T), device=dev)
    ang = torch.rand(max_pos, D // 2, device=dev)
    cs = torch.cat((ang.cos(), ang.sin()), 1)
    kc, vc = (torch.empty(T // bs, KVH, bs, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
    slots = torch.randperm(T, device=dev)
    # a token's cosines and sines: one of each per pair, from the pair's own axis
    nbytes = 2 * D * T * (2 * H + 4 * KVH) + T * (D * 4 + 32)
    return (lambda: gpu_ops.rope_store_kv(q, k, v, pos, cs, slots, (KVTier(kc, vc), None), T // bs, sections=(24, 20, 20)),
            nbytes, "fd_rope_kernel")


def _chunk(dev, R, ql, kl, flops: bool):
    H, KVH, D, bs = 32, 8, 128, 16
    W = kl // bs
    kc, vc = (torch.randn(R * W, KVH, bs, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
    table = torch.randperm(R * W, device=dev).to(torch.int32).view(R, W)
    q = torch.randn(R * ql, H, D, device=dev, dtype=torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(H, R * ql, device=dev)
    start = torch.arange(R, device=dev, dtype=torch.int32) * ql
    qlen, klen = (torch.full((R,), n, device=dev, dtype=torch.int32) for n in (ql, kl))
    work = 4 * R * H * D * (ql * kl - ql * (ql - 1) // 2) if flops else R * (4 * KVH * D * kl + 4 * ql * H * D)
    return (lambda: gpu_ops.chunk_attn(q, (KVTier(kc, vc), None), R * W, table, start, qlen, klen, D ** -0.5, out, lse,
                                       max_q_len=ql, max_k_len=kl),
            work, "fd_attn_mma_kernel" if flops else "fd_attn_rows_kernel")


def case_chunk_few(dev):
    return _chunk(dev, 32, 4, 4096, False)


def case_chunk_many(dev):
    return _chunk(dev, 2, 2048, 8192, True)


def _cross(dev, dtype, R, H, D, ql, kl):
    q = torch.randn(R * ql, H, D, device=dev, dtype=dtype)
    k, v = (torch.randn(R * kl, H, D, device=dev, dtype=dtype) for _ in range(2))
    out, lse = torch.empty_like(q), torch.empty(H, R * ql, device=dev)
    start, k_start = (torch.arange(R, device=dev, dtype=torch.int32) * n for n in (ql, kl))
    qlen, klen = (torch.full((R,), n, device=dev, dtype=torch.int32) for n in (ql, kl))
    return lambda: gpu_ops.cross_attn(q, k, v, start, qlen, k_start, klen, D ** -0.5, out, lse, max_q_len=ql, max_k_len=kl)


def case_cross_few(dev):
    return _cross(dev, torch.float16, 24, 20, 64, 1, 1500), 2 * 24 * 20 * 64 * (2 * 1500 + 2), "fd_attn_rows_kernel"


def case_cross_fp32(dev):
    return _cross(dev, torch.float32, 4, 8, 64, 64, 1500), 4 * 4 * 8 * 64 * 64 * 1500, "fd_attn_kernel"


def _stats(blocks, KVH, bs, dev):
    g = torch.Generator(device=dev).manual_seed(3)
    return gpu_ops.KeyStats(torch.rand(blocks, KVH, bs, generator=g, device=dev),
                            torch.randint(0, 1000, (blocks, KVH, bs), generator=g, device=dev, dtype=torch.int32))


def _weights(dev, R, ql, kl, flops: bool):
    H, KVH, D, bs = 32, 8, 128, 16
    W = kl // bs
    kc = torch.randn(R * W, KVH, bs, D, device=dev, dtype=torch.bfloat16)
    table = torch.randperm(R * W, device=dev).to(torch.int32).view(R, W)
    q = torch.randn(R * ql, H, D, device=dev, dtype=torch.bfloat16)
    lse = torch.full((H, R * ql), math.log(kl) + 0.5, device=dev)
    start = torch.arange(R, device=dev, dtype=torch.int32) * ql
    qlen, klen = (torch.full((R,), n, device=dev, dtype=torch.int32) for n in (ql, kl))
    stats = _stats(R * W, KVH, bs, dev)
    pairs = R * (ql * kl - ql * (ql - 1) // 2)
    work = 2 * pairs * H * D if flops else R * kl * KVH * (2 * D + 8) + 2 * R * ql * H * D
    return (lambda: gpu_ops.key_weights(q, (KVTier(kc, kc), None), R * W, table, start, qlen, klen, D ** -0.5, lse, stats,
                                        max_q_len=ql, max_k_len=kl), work, "fd_keyw_mma_kernel")


def case_weights_few(dev):
    return _weights(dev, 32, 4, 4096, False)


def case_weights_many(dev):
    return _weights(dev, 2, 2048, 8192, True)


def _cut(dev, R, n, keep):
    KVH, bs = 8, 16
    W = -(-n // bs)
    stats = _stats(R * W, KVH, bs, dev)
    table = torch.randperm(R * W, device=dev).to(torch.int32).view(R, W)
    lens, kept = (torch.full((R,), x, device=dev, dtype=torch.int32) for x in (n, keep))
    moves = gpu_ops.KeyMoves(R, KVH, min(keep, n - keep), dev)
    return stats, table, lens, kept, moves, lambda: gpu_ops.select_keys(stats, table, lens, kept, moves, max_k_len=n)


def case_select_keys(dev):
    R, n = 32, 2080
    *_, run = _cut(dev, R, n, 2048)
    return run, R * 8 * n * 8, "fd_select_kernel"


def case_move_keys(dev):
    R, n, keep, KVH, bs, D = 4, 16384, 2048, 8, 16, 128
    stats, table, lens, kept, moves, select = _cut(dev, R, n, keep)
    select()
    k, v = (torch.randn(table.numel(), KVH, bs, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
    nbytes = int(moves.counts.sum()) * (2 * (4 * D + 8) + 8)
    return lambda: gpu_ops.move_keys(moves, (KVTier(k, v), None), table.numel(), table, stats), nbytes, "fd_move_kernel"


def case_trim_tables(dev):
    R, n, bs = 100, 8192, 16
    W = n // bs
    table = torch.randperm(R * W, device=dev).to(torch.int32).view(R, W)
    lens, kept = (torch.full((R,), x, device=dev, dtype=torch.int32) for x in (n, 2048))
    free = gpu_ops.FreeBlocks(torch.empty(R * W, dtype=torch.int32, device=dev), None, torch.zeros(2, dtype=torch.int32, device=dev))
    out = gpu_ops.TrimTables(R, dev)
    return (lambda: gpu_ops.trim_tables(kept, lens, table, free, R * W, 0, bs, out), 12 * R + 8 * R * (n - 2048) // bs,
            "fd_trim_kernel")


def case_verify_drafts(dev):
    R, K, V = 64, 4, 131072
    target, draft = (torch.rand(*n, V, device=dev) for n in ((R * (K + 1),), (R, K)))
    tokens = torch.randint(0, V, (R, K), device=dev)
    start = torch.arange(R, device=dev, dtype=torch.int32) * (K + 1)
    qlen = torch.full((R,), K + 1, device=dev, dtype=torch.int32)
    au, su = torch.full((R, K), 0.999, device=dev), torch.rand(R, device=dev)
    out = gpu_ops.DraftVerdict(R, K, dev)
    return lambda: gpu_ops.verify_drafts(target, tokens, draft, start, qlen, au, su, out=out), R * 2 * V * 4, "fd_verify_kernel"


CASES = {
    "store_kv_prefill": lambda dev: case_store_kv(dev, False),
    "store_kv_decode": lambda dev: case_store_kv(dev, True),
    "merge2": case_merge2,
    "merge_partials": case_merge_partials,
    "split_merge": case_split_merge,
    "combine": case_combine,
    "host_mapped": case_host_mapped,
    "prefill": case_prefill,
    "prefill_fa": case_prefill_fa,
    "plan": case_plan,
    "exchange1": case_exchange1,
    "extend_tables": case_extend_tables, "rope_store_kv": case_rope_store_kv, "chunk_few": case_chunk_few,
    "chunk_many": case_chunk_many, "cross_few": case_cross_few, "cross_fp32": case_cross_fp32,
    "weights_few": case_weights_few, "weights_many": case_weights_many, "select_keys": case_select_keys,
    "move_keys": case_move_keys, "trim_tables": case_trim_tables, "verify_drafts": case_verify_drafts,
}


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("cases", nargs="*", default=list(CASES))
    ap.add_argument("--launches", type=int, default=20)
    args = ap.parse_args()
    dev = torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    peak = _hbm_peak()
    for name in args.cases:
        fn, nbytes, kernel = CASES[name](dev)
        t = _time(fn, args.launches)
        gpu_ops.check_device_errors(dev)
        gbs = nbytes / t / 1e9
        line = {"case": name, "kernel": kernel, "us_per_launch": round(t * 1e6, 2),
                "algorithmic_bytes": int(nbytes), "achieved_gbs": round(gbs, 1)}
        if name == "cross_fp32":  # flops of the fp32 pipe
            line = {"case": name, "kernel": kernel, "us_per_launch": round(t * 1e6, 2), "flops": int(nbytes),
                    "achieved_tflops": round(nbytes / t / 1e12, 1), "launches": args.launches}
            print(json.dumps(line), flush=True)
            continue
        if name in ("prefill", "prefill_fa", "chunk_many", "weights_many"):  # flops, not bytes
            tf = nbytes / t / 1e12
            peak_tf = _bf16_peak()
            line = {"case": name, "kernel": kernel, "us_per_launch": round(t * 1e6, 2), "flops": int(nbytes),
                    "achieved_tflops": round(tf, 1), "frac_of_bf16_peak": round(tf / peak_tf, 4),
                    "launches": args.launches}
            print(json.dumps(line), flush=True)
            del fn
            torch.cuda.empty_cache()
            continue
        if name == "host_mapped":
            pcie = pinned_copy_gbs(dev)
            line.update({"pinned_copy_gbs": round(pcie, 1), "frac_of_pinned_copy": round(gbs / pcie, 4),
                         "frac_of_pcie5_x16_nominal": round(gbs / PCIE5_X16_GBS, 4)})
        else:
            line["frac_of_hbm"] = round(gbs / peak, 4)
        line["launches"] = args.launches
        print(json.dumps(line), flush=True)
        del fn
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
