"""Cases, plain forms and exact values of the multi-token step's operators.

The operators are those of a serving step in which requests bring several new
tokens on top of context that is already cached:

  tables  block tables, slots and positions built on the GPU from lengths
  rope    rotary positions of one to four axes, fused with the KV write
  chunk   attention of a chunk of new tokens over the two-tier paged cache
  cross   attention of ragged queries to an encoder's states

`run` computes them with elementary torch operations, or, where `own` is set,
with this package's kernels.  Lengths follow from the case alone, values from
the seed.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one decode step of a full batch: a block boundary here and there, a few requests ending
        dict(name="tables_decode", op="tables", reqs=256, new_lo=1, new_hi=1, ctx_lo=16, ctx_hi=4096, block=16,
             end_every=64, gpu_share=0.7, mix=1),
        # a step that admits prompts among decodes, ragged, the pool spilling into the host tier
        dict(name="tables_prompts", op="tables", reqs=601, new_lo=0, new_hi=400, ctx_lo=0, ctx_hi=1000, block=16,
             end_every=7, gpu_share=0.4, mix=2),
        # three axes (time, height, width) for the tokens of a decode step
        dict(name="rope_decode", op="rope", dtype="bf16", tokens=128, heads=32, kv_heads=8, dim=128, rot=128, axes=3,
             style="halves", order="blocks", block=16, mix=3),
        # an image or video prompt, axes taken in turn
        dict(name="rope_prompt", op="rope", dtype="bf16", tokens=16384, heads=32, kv_heads=8, dim=128, rot=128, axes=3,
             style="halves", order="turns", block=16, mix=4),
        # text positions only, neighbouring pairs, part of the head rotated, an odd number of tokens
        dict(name="rope_odd", op="rope", dtype="fp16", tokens=1777, heads=20, kv_heads=20, dim=80, rot=32, axes=1,
             style="pairs", order="blocks", block=24, mix=5),
        # one request's draft tokens verified: latency
        dict(name="chunk_small", op="chunk", dtype="fp16", reqs=1, q_lo=5, q_hi=5, k_lo=700, k_hi=700, heads=32,
             kv_heads=8, dim=64, block=16, host=0.0, mix=6),
        # a batch's draft tokens verified over ragged contexts: the cache's bytes
        dict(name="chunk_verify", op="chunk", dtype="bf16", reqs=32, q_lo=2, q_hi=8, k_lo=512, k_hi=8192, heads=32,
             kv_heads=8, dim=128, block=16, host=0.0, mix=7),
        # chunks of prompts whose context has spilled into host memory: PCIe
        dict(name="chunk_spilled", op="chunk", dtype="bf16", reqs=3, q_lo=60, q_hi=70, k_lo=900, k_hi=2500, heads=32,
             kv_heads=8, dim=128, block=16, host=0.4, mix=8),
        # long chunks of long prompts: the tensor cores
        dict(name="chunk_long", op="chunk", dtype="bf16", reqs=2, q_lo=2048, q_hi=2048, k_lo=9000, k_hi=12288, heads=32,
             kv_heads=8, dim=128, block=16, host=0.0, mix=9),
        # single tokens of a batch over 1500 encoder states each
        dict(name="cross_token", op="cross", dtype="fp16", reqs=24, q_lo=1, q_hi=1, k_lo=1500, k_hi=1500, heads=20,
             kv_heads=20, dim=64, mix=10),
        # prompts against images' states of ragged lengths
        dict(name="cross_prompt", op="cross", dtype="bf16", reqs=6, q_lo=300, q_hi=2000, k_lo=1601, k_hi=6404, heads=32,
             kv_heads=8, dim=128, mix=11),
        # 32-bit values, short ragged texts
        dict(name="cross_fp32", op="cross", dtype="fp32", reqs=8, q_lo=1, q_hi=77, k_lo=77, k_hi=512, heads=8,
             kv_heads=8, dim=64, mix=12),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "rope", "chunk", "chunk", "cross"])
    mix = rng.randrange(1 << 30)
    if op == "tables":
        return dict(op=op, reqs=_spread(rng, 1, 900), new_lo=rng.choice([0, 1]), new_hi=_spread(rng, 1, 250),
                    ctx_lo=0, ctx_hi=_spread(rng, 8, 4096), block=rng.choice([8, 16, 32, 64]),
                    end_every=rng.choice([0, 3, 20]), gpu_share=rng.choice([0.1, 0.5, 1.0]), mix=mix)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        kvh = rng.choice([1, 2, 4, 8])
        return dict(op=op, dtype=dtype, tokens=_spread(rng, 1, 4000), heads=kvh * rng.choice([1, 3, 4]), kv_heads=kvh,
                    dim=dim, rot=rng.choice([dim, dim, dim // 2]), axes=rng.choice([1, 2, 3, 4]),
                    style=rng.choice(["halves", "pairs"]), order=rng.choice(["blocks", "turns"]),
                    block=rng.choice([8, 16, 24, 64]), mix=mix)
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128])
    kvh = rng.choice([1, 2, 4, 8])
    heads = kvh * rng.choice([1, 2, 4, 5, 8])
    q_hi = _spread(rng, 1, 1500 if dtype != "fp32" else 100)
    reqs = max(1, min(_spread(rng, 1, 40), 3000 // q_hi))
    case = dict(op=op, dtype=dtype, reqs=reqs, q_lo=max(1, q_hi // rng.choice([1, 2, 8])), q_hi=q_hi,
                k_lo=1, k_hi=_spread(rng, max(40, q_hi), 8192 if dtype != "fp32" else 1500), heads=heads, kv_heads=kvh,
                dim=dim, mix=mix)
    while case["reqs"] * case["heads"] * case["q_hi"] * case["k_hi"] > 1 << 30 and case["reqs"] > 1:
        case["reqs"] //= 2
    if op == "chunk":
        case.update(block=rng.choice([8, 16, 16, 16, 24, 64]), host=rng.choice([0.0, 0.0, 0.0, 0.1]))
    return case


def _lens(case):
    """Query and key lengths of an attention case; a chunk's keys hold its queries."""
    r = random.Random(case["mix"])
    ql = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["reqs"])]
    kl = [r.randint(case["k_lo"], case["k_hi"]) for _ in range(case["reqs"])]
    if case["op"] == "chunk":
        kl = [max(a, b) for a, b in zip(ql, kl)]
    return ql, kl


def _table_lens(case):
    """(prior, new) of a table case; new = -1: the request ends."""
    r = random.Random(case["mix"])
    prior = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["reqs"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["reqs"])]
    if case["end_every"]:
        new = [-1 if i % case["end_every"] == case["end_every"] - 1 else x for i, x in enumerate(new)]
    return prior, new


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    s = {"tables": _prepare_tables, "rope": _prepare_rope, "chunk": _prepare_attn, "cross": _prepare_attn}[case["op"]](
        case, seed)
    s["op"] = case["op"]
    return s


def _prepare_tables(case, seed):
    bs = case["block"]
    prior, new = _table_lens(case)
    held = [-(-p // bs) for p in prior]
    need = [0 if n < 0 else -(-(p + n) // bs) - h for p, n, h in zip(prior, new, held)]
    total = sum(held) + sum(need) + 8
    n_gpu = max(1, int(total * case["gpu_share"]))
    n_cpu = total - n_gpu
    width = max(h + max(0, k) for h, k in zip(held, need)) + 3
    rnd = random.Random(seed)
    ids = list(range(total))
    rnd.shuffle(ids)
    rows, at = [], 0
    for h in held:
        rows.append(ids[at:at + h] + [0] * (width - h))
        at += h
    rest = ids[at:]
    gpu = [b for b in rest if b < n_gpu]
    cpu = [b for b in rest if b >= n_gpu]
    tokens = sum(max(0, n) for n in new) + 5
    stack = torch.full((2, total), -1, dtype=torch.int32)
    stack[0, :len(gpu)] = torch.tensor(gpu, dtype=torch.int32)
    stack[1, :len(cpu)] = torch.tensor(cpu, dtype=torch.int32)
    s = dict(new=_i32(new), prior=_i32(prior), table=_i32(rows), stack=stack.to(DEV), counts=_i32([len(gpu), len(cpu)]),
             n_gpu=n_gpu, n_cpu=n_cpu, bs=bs, tokens=tokens, reqs=case["reqs"])
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        s["free"] = gpu_ops.FreeBlocks(s["stack"][0], s["stack"][1], s["counts"])
        s["step"] = gpu_ops.StepTables(case["reqs"], tokens, DEV)
    return s


def _axis_of_pair(case):
    """The axis of each rotated pair: blocks of pairs per axis, or the axes in turn."""
    pairs, axes = case["rot"] // 2, case["axes"]
    part = [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]
    if case["order"] == "blocks":
        return part, [a for a in range(axes) for _ in range(part[a])]
    return part, [i % axes for i in range(pairs)]


def _angles(case, positions):
    freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEV) / case["rot"])
    return torch.arange(positions, dtype=torch.float64, device=DEV).unsqueeze(1) * freq


def _prepare_rope(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    T, H, KVH, D, bs = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "block"))
    positions = 32768
    qkv = torch.randn(T, (H + 2 * KVH) * D, generator=g, device=DEV).to(dt)  # one projection's output, split in views
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((H * D, KVH * D, KVH * D), dim=1))
    blocks = -(-T // bs) + 7
    cache = torch.zeros(blocks, bs, KVH, 2 * D, dtype=dt, device=DEV)
    slots = torch.randperm(blocks * bs, generator=g, device=DEV)[:T]
    slots[::61] = -1  # padding tokens write no K/V
    ang = _angles(case, positions)
    s = dict(q=q, k=k, v=v, cache=cache, slots=slots, bs=bs, dim=D, rot=case["rot"], style=case["style"],
             pos=torch.randint(0, positions, (case["axes"], T), generator=g, device=DEV),
             cos_sin=torch.cat([ang.cos(), ang.sin()], dim=1).float(), axes=case["axes"],
             sections=tuple(_axis_of_pair(case)[0]), turns=case["order"] == "turns",
             axis=torch.tensor(_axis_of_pair(case)[1], device=DEV), q_out=torch.empty(T, H, D, dtype=dt, device=DEV))
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        kv = cache.permute(0, 2, 1, 3)
        s["tiers"] = (gpu_ops.KVTier(kv[..., :D], kv[..., D:]), None)
    return s


def _prepare_attn(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    ql, kl = _lens(case)
    q_start = [sum(ql[:i]) for i in range(len(ql))]
    T = sum(ql)
    s = dict(q=torch.randn(T, H, D, generator=g, device=DEV).to(dt), kvh=KVH, scale=D ** -0.5, max_q=max(ql),
             max_k=max(kl), q_start=_i32(q_start), q_len=_i32(ql), k_len=_i32(kl), n=len(ql),
             out=torch.empty(T, H, D, dtype=dt, device=DEV), lse=torch.empty(H, T, device=DEV),
             row=torch.repeat_interleave(torch.arange(len(ql), device=DEV), torch.tensor(ql, device=DEV)),
             nth=torch.tensor([i for n in ql for i in range(n)], device=DEV))
    if case["op"] == "cross":
        s["k"] = torch.randn(sum(kl), KVH, D, generator=g, device=DEV).to(dt)
        s["v"] = torch.randn(sum(kl), KVH, D, generator=g, device=DEV).to(dt)
        s["k_start"] = _i32([sum(kl[:i]) for i in range(len(kl))])
        return s
    bs = case["block"]
    held = [-(-x // bs) for x in kl]
    total = sum(held)
    n_cpu = int(total * case["host"])
    n_gpu = total - n_cpu + 5
    rnd = random.Random(seed)
    gpu, cpu = rnd.sample(range(n_gpu), n_gpu), [n_gpu + i for i in rnd.sample(range(n_cpu), n_cpu)]
    width = max(held)
    # the pool fills HBM first; what came last has spilled
    flat = gpu[:total - n_cpu] + cpu
    rows, at = [], 0
    for h in held:
        rows.append(flat[at:at + h] + [0] * (width - h))
        at += h
    s.update(table=_i32(rows), bs=bs, n_gpu=n_gpu, dim=D,
             cache=torch.randn(n_gpu, bs, KVH, 2 * D, generator=g, device=DEV).to(dt), hk=None, hv=None)
    if n_cpu:
        s["hk"] = torch.randn(n_cpu, KVH, bs, D, generator=g, device=DEV).to(dt).cpu().pin_memory()
        s["hv"] = torch.randn(n_cpu, KVH, bs, D, generator=g, device=DEV).to(dt).cpu().pin_memory()
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        kv = s["cache"].permute(0, 2, 1, 3)
        s["tiers"] = (gpu_ops.KVTier(kv[..., :D], kv[..., D:]), gpu_ops.KVTier(s["hk"], s["hv"]) if n_cpu else None)
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    return {"tables": _run_tables, "rope": _run_rope, "chunk": _run_chunk, "cross": _run_cross}[state["op"]](state)


def _run_tables(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        t = gpu_ops.extend_tables(s["new"], s["prior"], s["table"], s["free"], s["n_gpu"], s["n_cpu"], s["bs"], s["step"])
        return [s["table"], s["stack"], t.counts, t.seq_lens, t.query_start_loc, t.slot_mapping, t.positions]
    new, prior, table, stack, bs = s["new"].long(), s["prior"].long(), s["table"], s["stack"], s["bs"]
    R, W = table.shape
    cap = stack.shape[1]
    ends = new < 0
    add = new.clamp(min=0)
    seq = torch.where(ends, 0, prior + add)
    held = (prior + bs - 1) // bs
    want = (seq + bs - 1) // bs
    need = torch.where(ends, 0, want - held)
    qsl = torch.cat([add.new_zeros(1), add.cumsum(0)])
    col = torch.arange(W, device=DEV)
    # ended requests' blocks go onto their tier's stack, in table order
    freed = ends[:, None] & (col < held[:, None])
    on_gpu = table < s["n_gpu"]
    stacks, counts = [], []
    for t, mine in enumerate((freed & on_gpu, freed & ~on_gpu)):
        flat = mine.flatten().long()
        place = torch.where(mine.flatten(), s["counts"][t] + flat.cumsum(0) - 1, cap)
        grown = torch.cat([stack[t], stack.new_zeros(1)]).scatter(0, place, table.flatten())
        stacks.append(grown[:cap])
        counts.append(s["counts"][t] + flat.sum())
    # new blocks come off the HBM stack first, then off the host stack
    j = (need.cumsum(0) - need)[:, None] + col - held[:, None]
    takes = ~ends[:, None] & (col >= held[:, None]) & (col < want[:, None])
    from_gpu = stacks[0][(counts[0] - 1 - j).clamp(0, cap - 1)]
    from_cpu = stacks[1][(counts[1] - 1 - (j - counts[0])).clamp(0, cap - 1)]
    table = torch.where(takes, torch.where(j < counts[0], from_gpu, from_cpu), table)
    taken = need.sum()
    left = torch.stack([counts[0] - torch.minimum(taken, counts[0]),
                        counts[1] - (taken - counts[0]).clamp(min=0)]).int()
    tok = torch.arange(s["tokens"], device=DEV)
    r = torch.searchsorted(qsl[1:], tok, right=True).clamp(max=R - 1)
    real = tok < qsl[-1]
    pos = torch.where(real, prior[r] + tok - qsl[r], 0)
    block = table[r, (pos // bs).clamp(max=W - 1)].long()
    slots = torch.where(real, block * bs + pos % bs, -1)
    return [table, torch.stack(stacks), left, seq.int(), qsl.int(), slots, pos]


def _rotated(x, cos, sin, rot, style):
    x = x.float()
    turn, rest = x[..., :rot], x[..., rot:]
    if style == "halves":
        a, b = turn[..., :rot // 2], turn[..., rot // 2:]
        turn = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turn, rest], dim=-1)


def _run_rope(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        gpu_ops.rope_store_kv(s["q"], s["k"], s["v"], s["pos"], s["cos_sin"], s["slots"], s["tiers"], s["cache"].shape[0],
                              sections=s["sections"], turns=s["turns"], pairs=s["style"] == "pairs", q_out=s["q_out"])
        return [s["q_out"], s["cache"]]
    cache, dt = s["cache"], s["q"].dtype
    rot = s["rot"]
    pair = torch.arange(rot // 2, device=DEV)
    at = s["pos"][s["axis"]].T  # [T, pairs]: the position of each pair's axis
    cos, sin = s["cos_sin"][at, pair][:, None], s["cos_sin"][at, rot // 2 + pair][:, None]
    q = _rotated(s["q"], cos, sin, rot, s["style"]).to(dt)
    k = _rotated(s["k"], cos, sin, rot, s["style"]).to(dt)
    rows = cache.view(-1, cache.shape[2], cache.shape[3])
    keep = (s["slots"] >= 0)[:, None, None]
    slot = s["slots"].clamp(min=0)
    # padding tokens share a row behind the cache's last one
    spare = torch.cat([rows, rows[:1]])
    spare[torch.where(keep[:, 0, 0], slot, rows.shape[0])] = torch.cat([k, s["v"]], dim=-1)
    return [q, spare[:-1].view_as(cache)]


def _attend(s, keys, vals, causal):
    """Softmax attention of padded requests: keys, vals [n, mk, KVH, D] in 32 bits."""
    q, n, kvh = s["q"], s["n"], s["kvh"]
    T, H, D = q.shape
    G, mq, mk = H // kvh, s["max_q"], keys.shape[1]
    at = (s["q_start"][:, None] + torch.arange(mq, device=DEV)).clamp(max=T - 1)
    qp = q[at].float().view(n, mq, kvh, G, D).permute(0, 2, 3, 1, 4).reshape(n, kvh, G * mq, D)
    j = torch.arange(mk, device=DEV)
    real = j < s["k_len"][:, None]
    vals = torch.where(real[:, :, None, None], vals, 0.0)
    sc = (torch.matmul(qp, keys.permute(0, 2, 3, 1)) * s["scale"]).view(n, kvh, G, mq, mk)
    i = torch.arange(mq, device=DEV)
    sees = real[:, None, :].expand(n, mq, mk)
    if causal:
        sees = sees & (j <= (s["k_len"] - s["q_len"])[:, None, None] + i[:, None])
    sc = sc.masked_fill_(~sees[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = sc.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kvh, G * mq, mk), vals.transpose(1, 2)).view(n, kvh, G, mq, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n, mq, H, D)
    lse = (top + total.log()).squeeze(-1).permute(1, 2, 0, 3).reshape(H, n, mq)
    return [o[s["row"], s["nth"]].to(q.dtype), lse[:, s["row"], s["nth"]].contiguous()]


def _run_chunk(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        gpu_ops.chunk_attn(s["q"], s["tiers"], s["n_gpu"], s["table"], s["q_start"], s["q_len"], s["k_len"], s["scale"],
                           s["out"], s["lse"], max_q_len=s["max_q"], max_k_len=s["max_k"])
        return [s["out"], s["lse"]]
    D = s["dim"]
    cache = s["cache"].permute(0, 2, 1, 3)
    k, v = cache[..., :D], cache[..., D:]
    if s["hk"] is not None:
        k = torch.cat([k, s["hk"].to(DEV, non_blocking=True)])
        v = torch.cat([v, s["hv"].to(DEV, non_blocking=True)])
    ids = s["table"].long()
    n, kvh = s["n"], s["kvh"]
    keys = k[ids].float().transpose(2, 3).reshape(n, -1, kvh, D)[:, :s["max_k"]]
    vals = v[ids].float().transpose(2, 3).reshape(n, -1, kvh, D)[:, :s["max_k"]]
    return _attend(s, keys, vals, True)


def _run_cross(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        gpu_ops.cross_attn(s["q"], s["k"], s["v"], s["q_start"], s["q_len"], s["k_start"], s["k_len"], s["scale"],
                           s["out"], s["lse"], max_q_len=s["max_q"], max_k_len=s["max_k"])
        return [s["out"], s["lse"]]
    at = (s["k_start"][:, None] + torch.arange(s["max_k"], device=DEV)).clamp(max=s["k"].shape[0] - 1)
    return _attend(s, s["k"][at].float(), s["v"][at].float(), False)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    es = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "tables":
        prior, new = _table_lens(case)
        bs, R = case["block"], case["reqs"]
        taken = sum(-(-(p + n) // bs) - -(-p // bs) for p, n in zip(prior, new) if n >= 0)
        freed = sum(-(-p // bs) for p, n in zip(prior, new) if n < 0)
        tokens = sum(max(0, n) for n in new) + 5
        return {"bytes": 4 * (4 * R + 1) + 16 * tokens + 8 * (taken + freed) + 16, "flops": 0}
    if case["op"] == "rope":
        T, H, KVH, D, rot = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot"))
        moved = 2 * T * (H + 2 * KVH) * D * es
        return {"bytes": moved + T * (rot * 4 + 8 * case["axes"] + 8), "flops": 3 * T * (H + KVH) * rot}
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    ql, kl = _lens(case)
    if case["op"] == "chunk":
        pairs = sum(q * k - q * (q - 1) // 2 for q, k in zip(ql, kl))
        extra = sum(4 * -(-k // case["block"]) for k in kl)
    else:
        pairs, extra = sum(q * k for q, k in zip(ql, kl)), 0
    return {"bytes": sum(kl) * 2 * KVH * D * es + sum(ql) * H * (2 * D * es + 4) + extra, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------ exact values


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return _exact_tables(case, s)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    return _exact_attn(case, s)


def _exact_tables(case, s):
    """One request after the other, on lists."""
    bs = s["bs"]
    prior, new = _table_lens(case)
    table = s["table"].tolist()
    counts = s["counts"].tolist()
    stack = s["stack"].tolist()
    for r, n in enumerate(new):
        if n < 0:
            for b in table[r][:-(-prior[r] // bs)]:
                t = 0 if b < s["n_gpu"] else 1
                stack[t][counts[t]] = b
                counts[t] += 1
    seq, start, slots, places = [], [0], [], []
    for r, n in enumerate(new):
        for p in range(prior[r], prior[r] + max(0, n)):
            if p % bs == 0:
                t = 0 if counts[0] > 0 else 1
                counts[t] -= 1
                table[r][p // bs] = stack[t][counts[t]]
            slots.append(table[r][p // bs] * bs + p % bs)
            places.append(p)
        seq.append(0 if n < 0 else prior[r] + n)
        start.append(start[-1] + max(0, n))
    pad = s["tokens"] - len(slots)
    i64 = lambda x: torch.tensor(x, dtype=torch.int64)  # noqa: E731
    return [_i32(table), _i32(stack), _i32(counts), _i32(seq), _i32(start), i64(slots + [-1] * pad), i64(places + [0] * pad)]


def _exact_rope(case, s):
    rot, D = case["rot"], case["dim"]
    axis = torch.tensor(_axis_of_pair(case)[1], device=DEV)
    ang_c, ang_s = s["cos_sin"][:, :rot // 2].double(), s["cos_sin"][:, rot // 2:].double()
    at = s["pos"].index_select(0, axis).T
    z = torch.complex(ang_c.gather(0, at), ang_s.gather(0, at))[:, None, :]

    def turned(x):
        y = x.double().clone()
        first, second = ((slice(0, rot // 2), slice(rot // 2, rot)) if case["style"] == "halves"
                         else (slice(0, rot, 2), slice(1, rot, 2)))
        w = torch.complex(y[..., first], y[..., second]) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y

    cache = s["cache"].double()
    rows = cache.view(-1, case["kv_heads"], 2 * D)
    kept = (s["slots"] >= 0).nonzero().flatten()
    rows[s["slots"][kept], :, :D] = turned(s["k"])[kept]
    rows[s["slots"][kept], :, D:] = s["v"].double()[kept]
    return [turned(s["q"]), cache]


def _exact_attn(case, s):
    """One request and kv head at a time."""
    q = s["q"].double()
    T, H, D = q.shape
    kvh = s["kvh"]
    G = H // kvh
    ql, kl = _lens(case)
    out = torch.zeros(T, H, D, dtype=torch.float64, device=DEV)
    lse = torch.zeros(H, T, dtype=torch.float64, device=DEV)
    at = kat = 0
    for r, (nq, nk) in enumerate(zip(ql, kl)):
        if case["op"] == "chunk":
            ids = s["table"][r, :-(-nk // s["bs"])].tolist()
            near = s["cache"].transpose(1, 2)
            pages = [(near[b, ..., :D], near[b, ..., D:]) if b < s["n_gpu"] else
                     (s["hk"][b - s["n_gpu"]].to(DEV), s["hv"][b - s["n_gpu"]].to(DEV)) for b in ids]
            k = torch.cat([p[0] for p in pages], dim=1)[:, :nk].double()
            v = torch.cat([p[1] for p in pages], dim=1)[:, :nk].double()
            limit = nk - nq + torch.arange(nq, device=DEV)
        else:
            k = s["k"][kat:kat + nk].transpose(0, 1).double()
            v = s["v"][kat:kat + nk].transpose(0, 1).double()
            limit = torch.full((nq,), nk - 1, device=DEV)
        hidden = torch.arange(nk, device=DEV) > limit[:, None]
        for h in range(kvh):
            sc = torch.einsum("qgd,kd->gqk", q[at:at + nq, h * G:(h + 1) * G], k[h]) * s["scale"]
            sc = sc.masked_fill(hidden, -math.inf)
            lse[h * G:(h + 1) * G, at:at + nq] = torch.logsumexp(sc, -1)
            out[at:at + nq, h * G:(h + 1) * G] = torch.einsum("gqk,kd->qgd", torch.softmax(sc, -1), v[h])
        at += nq
        kat += nk
    return [out, lse]
