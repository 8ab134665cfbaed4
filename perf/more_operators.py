"""Cases, plain forms and exact values of the operators behind a step's attention.

What a serving step does with its attention's results, and with the cache that
has grown too long for its budget:

  weights  the attention weight that each cached key received, added up per key
  select   which keys stay when a request's cache is cut to a budget: the first
           and the newest ones, and those with the most weight
  move     the keys that stay moved to the front of their request's blocks
  trim     the blocks behind the new lengths given back to the free stacks
  verify   drafted tokens accepted or rejected against the target's
           probabilities, and the token that follows drawn, from given numbers

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
        # every step of a batch: single tokens over ragged contexts, the keys' bytes
        dict(name="weights_step", op="weights", dtype="bf16", reqs=32, q_lo=1, q_hi=1, k_lo=512, k_hi=8192, heads=32,
             kv_heads=8, dim=128, block=16, host=0.0, mix=1),
        # draft tokens and short chunks, padded head size, blocks that tiles do not divide
        dict(name="weights_odd", op="weights", dtype="fp16", reqs=9, q_lo=1, q_hi=40, k_lo=40, k_hi=1500, heads=20,
             kv_heads=4, dim=80, block=24, host=0.0, mix=2),
        # long chunks of long prompts: the tensor cores
        dict(name="weights_prompt", op="weights", dtype="bf16", reqs=2, q_lo=2048, q_hi=2048, k_lo=9000, k_hi=12288,
             heads=32, kv_heads=8, dim=128, block=16, host=0.0, mix=3),
        # 32-bit values, short ragged texts
        dict(name="weights_fp32", op="weights", dtype="fp32", reqs=8, q_lo=1, q_hi=77, k_lo=77, k_hi=512, heads=8,
             kv_heads=8, dim=64, block=16, host=0.0, mix=4),
        # a batch at its budget: every few steps a few keys too many
        dict(name="select_step", op="select", reqs=32, kv_heads=8, block=16, over_lo=0, over_hi=32, keep_lo=2048,
             keep_hi=2048, sinks=4, recent=256, mix=5),
        # prompts just read, far beyond the budget
        dict(name="select_prompt", op="select", reqs=4, kv_heads=8, block=16, over_lo=9000, over_hi=30000, keep_lo=2048,
             keep_hi=2048, sinks=4, recent=512, mix=6),
        dict(name="move_step", op="move", dtype="bf16", reqs=32, kv_heads=8, dim=128, block=16, over_lo=0, over_hi=32,
             keep_lo=2048, keep_hi=2048, share=0.9, mix=7),
        dict(name="move_prompt", op="move", dtype="bf16", reqs=4, kv_heads=8, dim=128, block=16, over_lo=9000,
             over_hi=30000, keep_lo=2048, keep_hi=2048, share=0.8, mix=8),
        # rejected draft tokens: a block here and there
        dict(name="trim_verify", op="trim", reqs=256, block=16, seq_lo=16, seq_hi=4096, cut_lo=0, cut_hi=7, gpu_share=0.7,
             mix=9),
        # long prompts cut to their budget, some blocks in the host tier
        dict(name="trim_budget", op="trim", reqs=100, block=16, seq_lo=4000, seq_hi=16000, cut_lo=2000, cut_hi=14000,
             gpu_share=0.5, mix=10),
        # one request's draft tokens: latency
        dict(name="verify_one", op="verify", dtype="fp32", reqs=1, drafts=4, vocab=32000, with_draft=True, mix=11),
        # a batch's draft tokens over a large vocabulary
        dict(name="verify_batch", op="verify", dtype="fp32", reqs=64, drafts=5, vocab=131072, with_draft=True, mix=12),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["weights", "weights", "select", "move", "trim", "verify"])
    mix = rng.randrange(1 << 30)
    if op == "weights":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
        kvh = rng.choice([1, 2, 4, 8])
        q_hi = _spread(rng, 1, 1500 if dtype != "fp32" else 100)
        case = dict(op=op, dtype=dtype, reqs=max(1, min(_spread(rng, 1, 40), 3000 // q_hi)),
                    q_lo=max(1, q_hi // rng.choice([1, 2, 8])), q_hi=q_hi, k_lo=1,
                    k_hi=_spread(rng, max(40, q_hi), 8192 if dtype != "fp32" else 1500), heads=kvh * rng.choice([1, 2, 4, 5, 8]),
                    kv_heads=kvh, dim=rng.choice([64, 64, 80, 96, 128, 128, 128]), block=rng.choice([8, 16, 16, 16, 24, 64]),
                    host=rng.choice([0.0, 0.0, 0.0, 0.1]), mix=mix)
        while case["reqs"] * case["heads"] * case["q_hi"] * case["k_hi"] > 1 << 30 and case["reqs"] > 1:
            case["reqs"] //= 2
        return case
    if op in ("select", "move"):
        keep, over = _spread(rng, 1, 4096), _spread(rng, 1, 20000)
        case = dict(op=op, reqs=max(1, min(_spread(rng, 1, 64), 150000 // (keep + over))), kv_heads=rng.choice([1, 2, 4, 8]),
                    block=rng.choice([8, 16, 16, 24, 64]), over_lo=rng.choice([0, over // 2]), over_hi=over,
                    keep_lo=max(1, keep // rng.choice([1, 4])), keep_hi=keep, mix=mix)
        if op == "select":
            return dict(case, sinks=rng.choice([0, 0, 1, 4]), recent=rng.choice([0, keep // 8, keep // 2]))
        return dict(case, dtype=rng.choice(["bf16", "fp16", "fp32"]), dim=rng.choice([64, 80, 96, 128, 256]),
                    share=rng.choice([0.1, 0.5, 1.0]))
    if op == "trim":
        seq = _spread(rng, 8, 16000)
        return dict(op=op, reqs=min(_spread(rng, 1, 900), 1600000 // seq), block=rng.choice([8, 16, 24, 32, 64]), seq_lo=0,
                    seq_hi=seq, cut_lo=0, cut_hi=_spread(rng, 1, seq), gpu_share=rng.choice([0.1, 0.5, 1.0]), mix=mix)
    vocab = _spread(rng, 100, 150000)
    drafts = rng.choice([1, 2, 3, 5, 8])
    return dict(op=op, dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                reqs=max(1, min(_spread(rng, 1, 200), 50000000 // vocab // (drafts + 1))), drafts=drafts, vocab=vocab,
                with_draft=rng.choice([True, True, False]), mix=mix)


def _lens(case):
    """Query and key lengths of a weights case; a request's keys hold its queries."""
    r = random.Random(case["mix"])
    ql = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["reqs"])]
    kl = [r.randint(case["k_lo"], case["k_hi"]) for _ in range(case["reqs"])]
    return ql, [max(a, b) for a, b in zip(ql, kl)]


def _budgets(case):
    """(keys, keys that stay) of each request of a select or move case."""
    r = random.Random(case["mix"])
    keep = [r.randint(case["keep_lo"], case["keep_hi"]) for _ in range(case["reqs"])]
    return [k + r.randint(case["over_lo"], case["over_hi"]) for k in keep], keep


def _cuts(case):
    """(tokens, tokens that stay) of each request of a trim case."""
    r = random.Random(case["mix"])
    seq = [r.randint(case["seq_lo"], case["seq_hi"]) for _ in range(case["reqs"])]
    return seq, [max(0, n - r.randint(case["cut_lo"], case["cut_hi"])) for n in seq]


def _moves(case):
    """Moves per request and kv head: the case's share of the most there can be."""
    r = random.Random(case["mix"] + 1)
    n, keep = _budgets(case)
    return [[int(min(b, a - b) * min(1.0, case["share"] * r.uniform(0.8, 1.0))) for _ in range(case["kv_heads"])]
            for a, b in zip(n, keep)]


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    s = {"weights": _prepare_weights, "select": _prepare_select, "move": _prepare_move, "trim": _prepare_trim,
         "verify": _prepare_verify}[case["op"]](case, seed)
    s["op"] = case["op"]
    return s


def _table(lens, bs, total, rnd):
    """Block tables of requests with these lengths, out of `total` shuffled blocks."""
    ids = list(range(total))
    rnd.shuffle(ids)
    held = [-(-n // bs) for n in lens]
    width = max(held) + 1
    rows, at = [], 0
    for h in held:
        rows.append(ids[at:at + h] + [0] * (width - h))
        at += h
    return rows, ids[at:]


def _flat(lens):
    """Request and number within it of every one of its keys or tokens."""
    n = torch.tensor(lens, device=DEV)
    row = torch.repeat_interleave(torch.arange(len(lens), device=DEV), n)
    return row, torch.arange(int(sum(lens)), device=DEV) - (n.cumsum(0) - n)[row]


def _key_positions(lens, gone, kvh, g):
    """Distinct positions [R, KVH, longest] of the keys: what earlier cuts left of 0 .. len + gone - 1."""
    full = torch.rand(len(lens), kvh, max(a + b for a, b in zip(lens, gone)), generator=g, device=DEV)
    at = torch.arange(full.shape[2], device=DEV)
    full = full.masked_fill(at >= (_i32(lens) + _i32(gone))[:, None, None], 2.0)
    return full.argsort(-1)[..., :max(lens)].int()


def _prepare_weights(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    H, KVH, D, bs = case["heads"], case["kv_heads"], case["dim"], case["block"]
    ql, kl = _lens(case)
    T, n = sum(ql), len(ql)
    total = sum(-(-x // bs) for x in kl)
    n_cpu = int(total * case["host"])
    n_gpu = total - n_cpu + 5
    rows, _ = _table(kl, bs, total, random.Random(seed))
    rows = [[b if b < total - n_cpu else b - (total - n_cpu) + n_gpu for b in row] for row in rows]
    blocks = n_gpu + n_cpu
    q_start = [sum(ql[:i]) for i in range(n)]
    krow, kth = _flat(kl)
    qrow, qth = _flat(ql)
    s = dict(q=torch.randn(T, H, D, generator=g, device=DEV).to(dt), scale=D ** -0.5, kvh=KVH, dim=D, bs=bs, n=n, n_gpu=n_gpu,
             q_start=_i32(q_start), q_len=_i32(ql), k_len=_i32(kl), max_q=max(ql), max_k=max(kl), table=_i32(rows),
             cache=torch.randn(n_gpu, bs, KVH, 2 * D, generator=g, device=DEV).to(dt), hk=None, hv=None,
             evicted=torch.randint(0, 1000, (n,), generator=g, device=DEV, dtype=torch.int32),
             weights=torch.rand(blocks, KVH, bs, generator=g, device=DEV) * 4,
             positions=torch.randint(0, 1000, (blocks, KVH, bs), generator=g, device=DEV, dtype=torch.int32),
             krow=krow, kth=kth, qrow=qrow, qth=qth)
    if n_cpu:
        s["hk"] = torch.randn(n_cpu, KVH, bs, D, generator=g, device=DEV).to(dt).cpu().pin_memory()
        s["hv"] = torch.zeros(n_cpu, KVH, bs, D, dtype=dt).pin_memory()
    # the attention's log-sum-exp, which such a program has from it
    lse = torch.empty(H, T, device=DEV)
    for r in range(n):
        k = _keys_of(s, r, kl[r]).float()
        hidden = torch.arange(kl[r], device=DEV) > (kl[r] - ql[r] + torch.arange(ql[r], device=DEV))[:, None]
        for h in range(H):
            sc = s["q"][q_start[r]:q_start[r] + ql[r], h].float() @ k[h // (H // KVH)].T * s["scale"]
            lse[h, q_start[r]:q_start[r] + ql[r]] = sc.masked_fill_(hidden, -math.inf).logsumexp(-1)
    s["lse"] = lse
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        kv = s["cache"].permute(0, 2, 1, 3)
        s["tiers"] = (gpu_ops.KVTier(kv[..., :D], kv[..., D:]), gpu_ops.KVTier(s["hk"], s["hv"]) if n_cpu else None)
        s["stats"] = gpu_ops.KeyStats(s["weights"], s["positions"])
    return s


def _keys_of(s, r, nk):
    """[KVH, nk, D]: one request's keys."""
    ids = s["table"][r, :-(-nk // s["bs"])].tolist()
    near = s["cache"].transpose(1, 2)[..., :s["dim"]]
    if s["hk"] is None:
        k = near[s["table"][r, :len(ids)].long()].transpose(0, 1).flatten(1, 2)
    else:
        k = torch.cat([near[b] if b < s["n_gpu"] else s["hk"][b - s["n_gpu"]].to(DEV) for b in ids], dim=1)
    return k[:, :nk]


def _prepare_select(case, seed):
    g = _gen(seed)
    KVH, bs = case["kv_heads"], case["block"]
    seq, keep = _budgets(case)
    n = len(seq)
    total = sum(-(-x // bs) for x in seq) + 3
    rows, _ = _table(seq, bs, total, random.Random(seed))
    table = _i32(rows)
    r = random.Random(case["mix"] + 2)
    gone = [r.randint(0, 500) for _ in seq]
    weights = torch.randn(total, KVH, bs, generator=g, device=DEV).mul_(2).exp_()
    weights *= torch.rand(total, KVH, bs, generator=g, device=DEV) > 0.05  # keys that no query looked at tie at 0
    positions = torch.zeros(total, KVH, bs, dtype=torch.int32, device=DEV)
    row, j = _flat(seq)
    positions[table[row, j // bs].long(), :, j % bs] = _key_positions(seq, gone, KVH, g)[row, :, j]
    room = max(1, max(min(b, a - b) for a, b in zip(seq, keep)))
    s = dict(weights=weights, positions=positions, table=table, seq=_i32(seq), keep=_i32(keep), evicted=_i32(gone), bs=bs,
             kvh=KVH, max_k=max(seq), room=room, sinks=case["sinks"], recent=case["recent"], n=n)
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        s["stats"] = gpu_ops.KeyStats(weights, positions)
        s["moves"] = gpu_ops.KeyMoves(n, KVH, room, DEV)
    return s


def _prepare_move(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    KVH, D, bs = case["kv_heads"], case["dim"], case["block"]
    seq, keep = _budgets(case)
    n = len(seq)
    total = sum(-(-x // bs) for x in seq) + 3
    rows, _ = _table(seq, bs, total, random.Random(seed))
    counts = _moves(case)
    room = max(1, max(min(b, a - b) for a, b in zip(seq, keep)))
    src = torch.zeros(n, KVH, room, dtype=torch.int32, device=DEV)
    dst = torch.zeros(n, KVH, room, dtype=torch.int32, device=DEV)
    for r in range(n):
        for h in range(KVH):
            c = counts[r][h]
            src[r, h, :c] = (torch.randperm(seq[r] - keep[r], generator=g, device=DEV)[:c].sort()[0] + keep[r]).int()
            dst[r, h, :c] = torch.randperm(keep[r], generator=g, device=DEV)[:c].sort()[0].int()
    pair, nth = _flat([c for row in counts for c in row])
    s = dict(cache=torch.randn(total, bs, KVH, 2 * D, generator=g, device=DEV).to(dt), table=_i32(rows), src=src, dst=dst,
             counts=_i32(counts), weights=torch.rand(total, KVH, bs, generator=g, device=DEV),
             positions=torch.randint(0, 1 << 20, (total, KVH, bs), generator=g, device=DEV, dtype=torch.int32), bs=bs, dim=D,
             total=total, req=pair // KVH, head=pair % KVH, nth=nth)
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        kv = s["cache"].permute(0, 2, 1, 3)
        s["tiers"] = (gpu_ops.KVTier(kv[..., :D], kv[..., D:]), None)
        s["stats"] = gpu_ops.KeyStats(s["weights"], s["positions"])
        s["moves"] = gpu_ops.KeyMoves(n, KVH, room, DEV, src=src, dst=dst, counts=s["counts"])
    return s


def _prepare_trim(case, seed):
    bs = case["block"]
    seq, keep = _cuts(case)
    total = sum(-(-x // bs) for x in seq) + 8
    n_gpu = max(1, int(total * case["gpu_share"]))
    rows, rest = _table(seq, bs, total, random.Random(seed))
    free = [[b for b in rest if b < n_gpu], [b for b in rest if b >= n_gpu]]
    stack = torch.full((2, total), -1, dtype=torch.int32)
    for t in range(2):
        stack[t, :len(free[t])] = torch.tensor(free[t], dtype=torch.int32)
    s = dict(seq=_i32(seq), keep=_i32(keep), table=_i32(rows), stack=stack.to(DEV), counts=_i32([len(f) for f in free]),
             n_gpu=n_gpu, n_cpu=total - n_gpu, bs=bs, max_cut=case["cut_hi"])
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        s["free"] = gpu_ops.FreeBlocks(s["stack"][0], s["stack"][1], s["counts"])
        s["out"] = gpu_ops.TrimTables(len(seq), DEV)
    return s


def _prepare_verify(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    R, K, V = case["reqs"], case["drafts"], case["vocab"]
    r = random.Random(case["mix"])
    q_len = [K + 1 if r.random() < 0.7 else r.randint(1, K + 1) for _ in range(R)]
    T = sum(q_len)
    start = [sum(q_len[:i]) for i in range(R)]
    logits = torch.randn(T, V, generator=g, device=DEV) * 2.5
    target = logits.softmax(-1)
    # the draft's own view of the same contexts
    row = (_i32(start)[:, None] + torch.arange(K, device=DEV)).clamp(max=T - 1)
    draft = torch.empty(R, K, V, dtype=dt, device=DEV)
    tokens = torch.empty(R, K, dtype=torch.int64, device=DEV)
    for d in range(K):
        p = (logits[row[:, d]] + 0.7 * torch.randn(R, V, generator=g, device=DEV)).softmax(-1)
        draft[:, d] = p
        # a token by the draft's probabilities: the first of independent waiting times
        tokens[:, d] = (p / torch.empty_like(p).exponential_(generator=g)).argmax(-1)
    s = dict(target=target.to(dt), draft=draft if case["with_draft"] else None, tokens=tokens, q_start=_i32(start),
             q_len=_i32(q_len), accept_u=torch.rand(R, K, generator=g, device=DEV), sample_u=torch.rand(R, generator=g, device=DEV),
             seq=torch.randint(K + 1, 4096, (R,), generator=g, device=DEV, dtype=torch.int32))
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        s["out"] = gpu_ops.DraftVerdict(R, K, DEV)
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    return {"weights": _run_weights, "select": _run_select, "move": _run_move, "trim": _run_trim,
            "verify": _run_verify}[state["op"]](state)


def _run_weights(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        gpu_ops.key_weights(s["q"], s["tiers"], s["n_gpu"], s["table"], s["q_start"], s["q_len"], s["k_len"], s["scale"],
                            s["lse"], s["stats"], evicted=s["evicted"], max_q_len=s["max_q"], max_k_len=s["max_k"])
        return [s["weights"], s["positions"]]
    q, n, kvh, D, bs = s["q"], s["n"], s["kvh"], s["dim"], s["bs"]
    T, H, _ = q.shape
    G, mq, mk = H // kvh, s["max_q"], s["max_k"]
    k = s["cache"].permute(0, 2, 1, 3)[..., :D]
    if s["hk"] is not None:
        k = torch.cat([k, s["hk"].to(DEV, non_blocking=True)])
    keys = k[s["table"].long()].float().transpose(2, 3).reshape(n, -1, kvh, D)[:, :mk]
    at = (s["q_start"][:, None] + torch.arange(mq, device=DEV)).clamp(max=T - 1)
    qp = q[at].float().view(n, mq, kvh, G, D).permute(0, 2, 3, 1, 4).reshape(n, kvh, G * mq, D)
    lse = s["lse"].view(kvh, G, T)[:, :, at].permute(2, 0, 1, 3)  # [n, kvh, G, mq]
    p = (torch.matmul(qp, keys.permute(0, 2, 3, 1)) * s["scale"]).view(n, kvh, G, mq, mk)
    p = p.sub_(lse[..., None]).exp_()
    i, j = torch.arange(mq, device=DEV)[:, None], torch.arange(mk, device=DEV)
    sees = (i < s["q_len"][:, None, None]) & (j <= (s["k_len"] - s["q_len"])[:, None, None] + i)
    total = p.masked_fill_(~sees[:, None, None], 0.0).sum((2, 3))  # [n, kvh, mk]
    row, kth = s["krow"], s["kth"]
    block, off = s["table"][row, kth // bs].long(), kth % bs
    old = kth < (s["k_len"] - s["q_len"])[row]
    mine = total[row, :, kth]
    weights, positions = s["weights"], s["positions"]
    weights[block, :, off] = torch.where(old[:, None], weights[block, :, off] + mine, mine)
    place = (kth + s["evicted"][row]).int()[:, None].expand(-1, kvh)
    positions[block, :, off] = torch.where(old[:, None], positions[block, :, off], place)
    return [weights, positions]


def _run_select(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        m = gpu_ops.select_keys(s["stats"], s["table"], s["seq"], s["keep"], s["moves"], sinks=s["sinks"],
                                recent=s["recent"], evicted=s["evicted"], max_k_len=s["max_k"])
        return [m.src, m.dst, m.counts]
    bs, mk, kvh, n, room = s["bs"], s["max_k"], s["kvh"], s["n"], s["room"]
    j = torch.arange(mk, device=DEV)
    block = s["table"][:, j // bs].long()
    w = s["weights"][block, :, j % bs].transpose(1, 2).double()  # [n, kvh, mk]
    pos = s["positions"][block, :, j % bs].transpose(1, 2)
    seq, keep = s["seq"][:, None, None], s["keep"][:, None, None]
    newest = pos >= seq + s["evicted"][:, None, None] - s["recent"]
    score = torch.where(w.isnan(), -4e38, w.clamp(max=4e38))
    score = torch.where((pos < s["sinks"]) | newest, math.inf, score)
    score = torch.where(j < seq, score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True)[1]
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order))
    stays = (rank < keep) & (j < seq)
    hole, mover = ~stays & (j < keep) & (keep < seq), stays & (j >= keep) & (keep < seq)
    lists = []
    for picked in (mover, hole):
        place = torch.where(picked, picked.long().cumsum(-1) - 1, room)
        full = torch.zeros(n, kvh, room + 1, dtype=torch.int32, device=DEV)
        lists.append(full.scatter_(-1, place, j.int().expand_as(place))[..., :room])
    return [lists[0], lists[1], mover.sum(-1).int()]


def _run_move(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        gpu_ops.move_keys(s["moves"], s["tiers"], s["total"], s["table"], s["stats"])
        return [s["cache"], s["weights"], s["positions"]]
    req, head, nth, bs = s["req"], s["head"], s["nth"], s["bs"]
    a, b = s["src"][req, head, nth].long(), s["dst"][req, head, nth].long()
    ab, bb = s["table"][req, a // bs].long(), s["table"][req, b // bs].long()
    s["cache"][bb, b % bs, head] = s["cache"][ab, a % bs, head]
    for x in (s["weights"], s["positions"]):
        x[bb, head, b % bs] = x[ab, head, a % bs]
    return [s["cache"], s["weights"], s["positions"]]


def _run_trim(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        t = gpu_ops.trim_tables(s["keep"], s["seq"], s["table"], s["free"], s["n_gpu"], s["n_cpu"], s["bs"], s["out"],
                                max_cut=s["max_cut"])
        return [s["stack"], t.counts, t.seq_lens]
    seq, table, stack, bs = s["seq"], s["table"], s["stack"], s["bs"]
    cap = stack.shape[1]
    left = torch.minimum(s["keep"], seq)
    col = torch.arange(table.shape[1], device=DEV)
    freed = (col >= ((left + bs - 1) // bs)[:, None]) & (col < ((seq + bs - 1) // bs)[:, None])
    on_gpu = table < s["n_gpu"]
    stacks, counts = [], []
    for t, mine in enumerate((freed & on_gpu, freed & ~on_gpu)):
        flat = mine.flatten().long()
        place = torch.where(mine.flatten(), s["counts"][t] + flat.cumsum(0) - 1, cap)
        stacks.append(torch.cat([stack[t], stack.new_zeros(1)]).scatter(0, place, table.flatten())[:cap])
        counts.append(s["counts"][t] + flat.sum())
    return [torch.stack(stacks), torch.stack(counts).int(), left]


def _run_verify(s):
    if own:
        from vllm_fastdecoder_b200 import gpu_ops

        v = gpu_ops.verify_drafts(s["target"], s["tokens"], s["draft"], s["q_start"], s["q_len"], s["accept_u"],
                                  s["sample_u"], seq_lens=s["seq"], out=s["out"])
        return [v.tokens, v.accepted, v.keep_lens]
    target, draft, tokens = s["target"], s["draft"], s["tokens"]
    T, V = target.shape
    R, K = tokens.shape
    r, d = torch.arange(R, device=DEV), torch.arange(K, device=DEV)
    first, drafts = s["q_start"].long(), s["q_len"].long() - 1
    at = (first[:, None] + d).clamp(max=T - 1)
    p = target[at, tokens].double()
    q = torch.ones_like(p) if draft is None else draft.gather(2, tokens[..., None])[..., 0].double()
    good = (s["accept_u"].double() * q < p) & (d < drafts[:, None])
    accepted = good.long().cumprod(1).sum(1)
    rejected = accepted < drafts
    row = target[first + accepted].double()
    which = accepted.clamp(max=K - 1)
    if draft is None:
        other = torch.where(torch.arange(V, device=DEV) == tokens[r, which][:, None], math.inf, 0.0)
    else:
        other = draft[r, which].double()
    left = (row - torch.where(rejected[:, None], other, 0.0)).clamp(min=0.0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, row)
    run_sum = left.cumsum(1)
    drawn = (run_sum > s["sample_u"].double()[:, None] * run_sum[:, -1:]).long().argmax(1)
    col = torch.arange(K + 1, device=DEV)
    out = torch.where(col < accepted[:, None], torch.cat([tokens, tokens[:, :1]], 1), -1)
    out = torch.where(col == accepted[:, None], drawn[:, None], out)
    return [out, accepted.int(), (s["seq"] - (drafts - accepted)).int()]


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["op"] == "weights":
        es = 4 if case["dtype"] == "fp32" else 2
        H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
        ql, kl = _lens(case)
        pairs = sum(q * k - q * (q - 1) // 2 for q, k in zip(ql, kl))
        old = sum(kl) - sum(ql)
        stats = KVH * (8 * old + 8 * sum(ql))  # old keys: a weight read and written; new ones: weight and position written
        return {"bytes": sum(kl) * KVH * D * es + sum(ql) * H * (D * es + 4) + stats + sum(4 * -(-k // case["block"]) for k in kl),
                "flops": 2 * pairs * H * D}
    if case["op"] == "select":
        seq, keep = _budgets(case)
        cut = [(a, b) for a, b in zip(seq, keep) if b < a]
        # about keep (1 - keep / n) of the kept keys lie behind the budget when weights do not depend on the place
        moves = sum(int(b * (1 - b / a)) for a, b in cut)
        return {"bytes": case["kv_heads"] * (sum(8 * a for a, _ in cut) + 8 * moves + 4 * len(seq))
                + sum(4 * -(-a // case["block"]) for a, _ in cut) + 12 * len(seq), "flops": 0}
    if case["op"] == "move":
        es = 4 if case["dtype"] == "fp32" else 2
        moves = sum(sum(row) for row in _moves(case))
        return {"bytes": moves * (2 * (2 * case["dim"] * es + 8) + 8) + 4 * case["reqs"] * case["kv_heads"] + 8, "flops": 0}
    if case["op"] == "trim":
        seq, keep = _cuts(case)
        freed = sum(-(-a // case["block"]) - -(-b // case["block"]) for a, b in zip(seq, keep))
        return {"bytes": 12 * len(seq) + 8 * freed + 16, "flops": 0}
    es = 4 if case["dtype"] == "fp32" else 2
    R, K, V = case["reqs"], case["drafts"], case["vocab"]
    # one row of the target per request, and one of the draft's where a token is rejected (about all requests)
    return {"bytes": R * (V * es * (2 if case["with_draft"] else 1) + K * (2 * es + 12) + 4 + 12 + 8 * (K + 1) + 8), "flops": 0}


# ------------------------------------------------------------------ exact values


def exact(case, seed):
    s = prepare(case, seed)
    return {"weights": _exact_weights, "select": _exact_select, "move": _exact_move, "trim": _exact_trim,
            "verify": _exact_verify}[case["op"]](case, s)


def _exact_weights(case, s):
    """One request and kv head at a time."""
    ql, kl = _lens(case)
    KVH, bs = s["kvh"], s["bs"]
    G = case["heads"] // KVH
    weights, positions = s["weights"].double(), s["positions"].clone()
    at = 0
    for r, (nq, nk) in enumerate(zip(ql, kl)):
        keys = _keys_of(s, r, nk).double()
        hidden = torch.arange(nk, device=DEV) > (nk - nq + torch.arange(nq, device=DEV))[:, None]
        j = torch.arange(nk, device=DEV)
        block, off = s["table"][r].long().index_select(0, j // bs), j % bs
        for h in range(KVH):
            total = torch.zeros(nk, dtype=torch.float64, device=DEV)
            for x in range(h * G, (h + 1) * G):
                e = s["q"][at:at + nq, x].double() @ keys[h].T * s["scale"] - s["lse"][x, at:at + nq].double()[:, None]
                total += e.exp().masked_fill(hidden, 0.0).sum(0)
            kept = weights[block, h, off]
            kept[nk - nq:] = 0.0
            weights[block, h, off] = kept + total
            positions[block[nk - nq:], h, off[nk - nq:]] = (j[nk - nq:] + s["evicted"][r]).int()
        at += nq
    return [weights, positions]


def _exact_select(case, s):
    """Sorted on lists, one request and kv head at a time."""
    seq, keep = _budgets(case)
    bs = s["bs"]
    w, pos, table, gone = s["weights"].cpu().numpy(), s["positions"].cpu().numpy(), s["table"].tolist(), s["evicted"].tolist()
    src, dst = (torch.zeros(s["n"], s["kvh"], s["room"], dtype=torch.int32) for _ in range(2))
    counts = torch.zeros(s["n"], s["kvh"], dtype=torch.int32)
    for r, (n, b) in enumerate(zip(seq, keep)):
        if b >= n:
            continue
        blocks = table[r][:-(-n // bs)]
        for h in range(s["kvh"]):
            ws, ps = w[blocks, h].reshape(-1)[:n].tolist(), pos[blocks, h].reshape(-1)[:n].tolist()
            guarded = [p < s["sinks"] or p >= n + gone[r] - s["recent"] for p in ps]
            order = sorted(range(n), key=lambda j: (not guarded[j], 0.0 if guarded[j] else -ws[j], j))
            stays = set(order[:b])
            a = sorted(j for j in stays if j >= b)
            src[r, h, :len(a)] = torch.tensor(a, dtype=torch.int32)
            dst[r, h, :len(a)] = torch.tensor([j for j in range(b) if j not in stays], dtype=torch.int32)
            counts[r, h] = len(a)
    return [src, dst, counts]


def _exact_move(case, s):
    """Row after row of the flattened cache."""
    bs = s["bs"]
    counts = _moves(case)
    cache, weights, positions = s["cache"].double(), s["weights"].double(), s["positions"].clone()
    rows = cache.view(-1, *cache.shape[2:])
    for r, row in enumerate(counts):
        line = s["table"][r].long()
        for h, c in enumerate(row):
            a, b = s["src"][r, h, :c].long(), s["dst"][r, h, :c].long()
            a, b = line[a // bs] * bs + a % bs, line[b // bs] * bs + b % bs
            rows[b, h] = rows[a, h]
            for x in (weights, positions):
                y = x[:, h].reshape(-1)
                y[b] = y[a]
                x[:, h] = y.view(-1, bs)
    return [cache, weights, positions]


def _exact_trim(case, s):
    """One request after the other, on lists."""
    seq, keep = _cuts(case)
    bs, counts, stack, table = s["bs"], s["counts"].tolist(), s["stack"].tolist(), s["table"].tolist()
    left = []
    for r, (n, b) in enumerate(zip(seq, keep)):
        left.append(min(n, b))
        for block in table[r][-(-left[r] // bs):-(-n // bs)]:
            t = 0 if block < s["n_gpu"] else 1
            stack[t][counts[t]] = block
            counts[t] += 1
    return [_i32(stack), _i32(counts), _i32(left)]


def _exact_verify(case, s):
    """One request and token at a time."""
    import numpy as np

    tokens, start, q_len = s["tokens"].tolist(), s["q_start"].tolist(), s["q_len"].tolist()
    au, su, seq = s["accept_u"].double().tolist(), s["sample_u"].double().tolist(), s["seq"].tolist()
    K = case["drafts"]
    out, accepted, keep = [], [], []
    for r in range(case["reqs"]):
        got, a = [], 0
        while a < q_len[r] - 1:
            t = tokens[r][a]
            q = 1.0 if s["draft"] is None else float(s["draft"][r, a, t])
            if not au[r][a] * q < float(s["target"][start[r] + a, t]):
                break
            got.append(t)
            a += 1
        p = s["target"][start[r] + a].double().cpu().numpy()
        left = p.copy()
        if a < q_len[r] - 1 and s["draft"] is None:
            left[tokens[r][a]] = 0.0
        elif a < q_len[r] - 1:
            left = np.maximum(p - s["draft"][r, a].double().cpu().numpy(), 0.0)
        if not left.sum() > 0:
            left = p
        line = np.cumsum(left)
        got.append(int(np.searchsorted(line, su[r] * line[-1], side="right")))
        out.append(got + [-1] * (K + 1 - len(got)))
        accepted.append(a)
        keep.append(seq[r] - (q_len[r] - 1 - a))
    return [torch.tensor(out), _i32(accepted).cpu(), _i32(keep).cpu()]
