"""GPU tests of the multi-token step's operators against plain 64-bit forms
(tests/step_ref.py): block tables from lengths (exact), multi-axis rotary
positions with the KV write, chunk attention over both tiers, cross attention,
and a run of them together."""

from __future__ import annotations

import random

import pytest
import step_ref as ref
import torch

from vllm_fastdecoder_b200 import gpu_ops, plan
from vllm_fastdecoder_b200.gpu_ops import FreeBlocks, KVTier, StepTables

pytestmark = pytest.mark.gpu
NAN = float("nan")


def dev():
    return torch.device("cuda", torch.cuda.current_device())


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ tables


def _table_case(R, block, ctx, new_hi, end_every, hbm_share, seed, slack=6):
    rnd = random.Random(seed)
    prior = [rnd.randint(0, ctx) for _ in range(R)]
    new = [rnd.choice([0, 1, rnd.randint(0, new_hi)]) for _ in range(R)]
    if end_every:
        new = [-1 if i % end_every == end_every - 1 else n for i, n in enumerate(new)]
    held = [-(-p // block) for p in prior]
    need = sum(-(-(p + n) // block) - h for p, n, h in zip(prior, new, held) if n >= 0)
    total = sum(held) + need + slack
    hbm = max(1, int(total * hbm_share))
    ids = list(range(total))
    rnd.shuffle(ids)
    W = max(-(-(p + max(0, n)) // block) for p, n in zip(prior, new)) + 2
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-7] * (W - h))
        at += h
    s0, s1 = [b for b in ids[at:] if b < hbm], [b for b in ids[at:] if b >= hbm]
    counts = [len(s0), len(s1)]
    return prior, new, table, [s0 + [-1] * (total - len(s0)), s1 + [-1] * (total - len(s1))], counts, hbm, total - hbm


def _run_tables(prior, new, table, stacks, counts, hbm, host, block, T, W=None, in_place=False):
    tt, st, ct, pr = i32(table), i32(stacks), i32(counts), i32(prior)
    free = FreeBlocks(st[0], st[1], ct)
    out = StepTables(len(prior), T, dev(), seq_lens=pr if in_place else None, counts=ct if in_place else None)
    out.slot_mapping.fill_(99)
    out.positions.fill_(99)
    gpu_ops.extend_tables(i32(new), pr, tt, free, hbm, host, block, out)
    return tt, st, out


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("R,block,ctx,new_hi,end_every,share,T", [
    (1, 16, 0, 1, 0, 1.0, 4), (1, 1, 5, 3, 0, 0.5, 9), (3, 16, 40, 20, 2, 0.5, 70), (33, 8, 100, 9, 4, 0.3, 300),
    (256, 16, 500, 2, 16, 0.6, 700), (1023, 16, 64, 5, 3, 0.5, 2048), (1024, 32, 64, 5, 0, 0.01, 6000),
    (1025, 24, 300, 40, 5, 0.5, 50000), (8192, 16, 100, 3, 9, 0.5, 20000), (5, 64, 3000, 9000, 0, 0.7, 50000),
    (150, 16, 300, 2000, 5, 0.5, 70000), (700, 8, 90, 400, 3, 0.4, 60000), (8, 16, 30, 40000, 0, 0.9, 90000),
])
def test_tables_match_lists(R, block, ctx, new_hi, end_every, share, T, in_place):
    prior, new, table, stacks, counts, hbm, host = _table_case(R, block, ctx, new_hi, end_every, share, R + T)
    want = ref.tables(new, prior, table, stacks, counts, hbm, block, T)
    assert want is not None
    tt, st, out = _run_tables(prior, new, table, stacks, counts, hbm, host, block, T, in_place=in_place)
    gpu_ops.check_device_errors(dev())
    h = out.read_header()
    w_table, w_stacks, w_counts, w_seq, w_qsl, w_slots, w_pos = want
    assert tt.tolist() == w_table and out.counts.tolist() == w_counts
    for t in range(2):
        top = max(w_counts[t], counts[t])
        assert st[t].tolist()[:w_counts[t]] == w_stacks[t][:w_counts[t]]
        assert st[t].tolist()[top:] == w_stacks[t][top:]
    assert out.seq_lens.tolist() == w_seq and out.query_start_loc.tolist() == w_qsl
    assert out.slot_mapping.tolist() == w_slots and out.positions.tolist() == w_pos
    assert h["n_tok"] == w_qsl[-1] and h["max_seq"] == max(s for s, n in zip(w_seq, new))
    assert h["max_new"] == max(0, max(new))


def test_tables_of_no_requests_and_no_tokens():
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = StepTables(0, 3, dev())
    gpu_ops.extend_tables(e, e, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), FreeBlocks(e, None, i32([0, 0])), 4, 0,
                          16, out)
    assert out.read_header()["n_tok"] == 0 and out.slot_mapping.tolist() == [-1] * 3
    out = StepTables(2, 0, dev())
    gpu_ops.extend_tables(i32([0, -1]), i32([5, 5]), i32([[1], [2]]), FreeBlocks(i32([0]), i32([0]), i32([0, 0])), 8, 0, 16,
                          out)
    assert out.read_header()["freed_hbm"] == 1 and out.seq_lens.tolist() == [5, 0] and out.counts.tolist() == [1, 0]


def test_tables_whose_rows_overlap_are_refused():
    with pytest.raises(RuntimeError, match="overlap"):
        _run_tables_on(i32([[1, 2]]).expand(3, 2))
    _run_tables_on(i32([[1, 2]]))


def _run_tables_on(table):
    R = table.shape[0]
    gpu_ops.extend_tables(i32([0] * R), i32([0] * R), table, FreeBlocks(i32([0]), None, i32([1, 0])), 8, 0, 16, max_tokens=4)
    gpu_ops.check_device_errors(dev())


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("why,flag", [("blocks", 1), ("width", 2), ("tokens", 4), ("prior", 8), ("new", 8), ("block", 16),
                                      ("count", 32), ("room", 32)])
def test_refused_steps_change_nothing(why, flag, big):
    R = 1500 if big else 6
    prior, new = [20] * R, [3] * R
    table = [[2 * r, 2 * r + 1, -7] for r in range(R)]
    T, counts, caps = 4 * R + 10, [4, 4], [8 * R, 8 * R]
    new[1] = -1
    if why == "blocks":
        new = [13] * R  # a block more for every request
        T = 20 * R
        counts = [R - 2, 1]
    elif why == "width":
        new[R - 1] = 29
        counts = [R, R]
    elif why == "tokens":
        T = 3 * (R - 1) - 1
    elif why == "prior":
        prior[0] = -1
    elif why == "new":
        new[0] = -2
    elif why == "block":
        table[1][1] = 8 * R
    elif why == "count":
        counts = [-1, 3]
    elif why == "room":
        caps = [5, 5]
    stacks = [[1000000 + i for i in range(caps[0])], [2000000 + i for i in range(caps[1])]]
    tt, st, out = _run_tables(prior, new, table, stacks, counts, 4 * R, 4 * R, 16, T)
    with pytest.raises(RuntimeError, match="block tables"):
        gpu_ops.check_device_errors(dev())
    assert out.header.tolist()[0] & flag
    with pytest.raises(RuntimeError, match="refused"):
        out.read_header()
    assert tt.tolist() == table and st.tolist() == stacks and out.counts.tolist() == counts
    assert out.seq_lens.tolist() == prior and out.query_start_loc.tolist() == [0] * (R + 1)
    assert out.slot_mapping.tolist() == [-1] * T and out.positions.tolist() == [0] * T


@pytest.mark.parametrize("R", [1, 40, 257, 3000])
@pytest.mark.parametrize("in_place", [False, True])
def test_query_lens_are_what_the_attention_takes(R, in_place):
    prior, new, table, stacks, counts, hbm, host = _table_case(R, 16, 60, 9, 3, 0.5, R)
    free = FreeBlocks(i32(stacks[0]), i32(stacks[1]), i32(counts))
    given = i32(new)
    T = sum(max(0, n) for n in new) + 1
    out = StepTables(R, T, dev())
    if in_place:
        out.query_lens = given
    else:
        out.query_lens.fill_(77)
    gpu_ops.extend_tables(given, i32(prior), i32(table), free, hbm, host, 16, out)
    assert out.read_header()["n_tok"] == T - 1
    gpu_ops.check_device_errors(dev())
    assert out.query_lens.tolist() == [max(0, n) for n in new]
    # a step that is refused (more tokens than room) has none
    given.copy_(i32([2] * R))
    gpu_ops.extend_tables(given, i32(prior), i32(table), free, hbm, host, 16, out, max_tokens=2 * R - 1 if 2 * R <= T else 0)
    with pytest.raises(RuntimeError, match="block tables"):
        gpu_ops.check_device_errors(dev())
    assert out.query_lens.tolist() == [0] * R and given.tolist() == ([0] * R if in_place else [2] * R)


# ------------------------------------------------------------------ rope


def _cos_sin(positions, rot):
    ang = torch.arange(positions, dtype=torch.float64).unsqueeze(1) * 10000.0 ** (
        -torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.cat([ang.cos(), ang.sin()], 1).float().cuda()


def _rope_ok(got, want, x, dtype):
    # two products and a sum in fp32 (three half steps of at most |x1| + |x2|), rounded once to the type
    tol = ref.half_step(dtype) * want.abs() + 3 * 2.0 ** -24 * 2 * x.double().abs().max() + 2.0 ** -24
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,KVH,D,rot,sections,turns,pairs,block", [
    (1, 4, 1, 64, 64, None, False, False, 16), (37, 8, 2, 128, 128, (24, 20, 20), False, False, 16),
    (130, 8, 2, 128, 128, (24, 20, 20), True, False, 16), (65, 6, 3, 80, 40, (7, 7, 6), True, True, 24),
    (50, 5, 5, 80, 20, (10,), False, False, 1), (33, 2, 1, 256, 256, (32, 32, 32, 32), True, True, 7),
    (3000, 4, 2, 64, 32, (16,), False, True, 64), (20, 3, 1, 96, 2, None, False, True, 16),
])
def test_rope_writes_rotated_rows(dtype, T, H, KVH, D, rot, sections, turns, pairs, block):
    g = torch.Generator(device="cuda").manual_seed(T)
    A = 1 if sections is None else len(sections)
    qkv = torch.randn(T, (H + 2 * KVH) * D, generator=g, device="cuda").to(dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((H * D, KVH * D, KVH * D), 1))
    pos = torch.randint(0, 5000, (A, T + 3), generator=g, device="cuda")
    pos[:, 0] = 4999
    cs = _cos_sin(5000, rot)
    hbm, host = -(-T // block) // 2 + 1, -(-T // block) // 2 + 2
    cache = torch.full((hbm, block, KVH, 2 * D), NAN, device="cuda").to(dtype)
    hk = torch.full((host, KVH, block, D), NAN).to(dtype).pin_memory()
    hv = torch.full((host, KVH, block, D), NAN).to(dtype).pin_memory()
    logical = cache.permute(0, 2, 1, 3)
    tiers = (KVTier(logical[..., :D], logical[..., D:]), KVTier(hk, hv))
    slots = torch.randperm((hbm + host) * block, generator=g, device="cuda")[:T]
    slots[::5] = -1
    q_out = torch.full((T, H + 1, D), NAN, device="cuda").to(dtype)[:, :H]
    k_out = torch.full((T, KVH, D), NAN, device="cuda").to(dtype)
    before = qkv.clone()
    got = gpu_ops.rope_store_kv(q, k, v, pos[0] if sections is None else pos, cs, slots, tiers, hbm, sections=sections,
                                turns=turns, pairs=pairs, q_out=q_out, k_out=k_out)
    gpu_ops.check_device_errors(dev())
    assert got is q_out and torch.equal(qkv, before)
    axis = gpu_ops.rope_axes((rot // 2,) if sections is None else sections, turns)
    want_k = ref.rope(k, pos[:, :T], cs, axis, pairs)
    _rope_ok(q_out, ref.rope(q, pos[:, :T], cs, axis, pairs), q, dtype)
    _rope_ok(k_out, want_k, k, dtype)
    rows_k = torch.cat([logical[..., :D].transpose(1, 2).reshape(-1, KVH, D),
                        hk.transpose(1, 2).reshape(-1, KVH, D).cuda()])
    rows_v = torch.cat([logical[..., D:].transpose(1, 2).reshape(-1, KVH, D),
                        hv.transpose(1, 2).reshape(-1, KVH, D).cuda()])
    kept = slots >= 0
    assert torch.equal(rows_k[slots[kept]], k_out[kept]) and torch.equal(rows_v[slots[kept]], v[kept])
    rest = torch.ones(rows_k.shape[0], dtype=torch.bool, device="cuda")
    rest[slots[kept]] = False
    assert bool(rows_k[rest].isnan().all()) and bool(rows_v[rest].isnan().all())
    # in place, without a KV write
    q2, k2 = q.clone(), k.clone()
    assert gpu_ops.rope_store_kv(q2, k2, v, pos[0] if sections is None else pos, cs, None, (None, None), 0,
                                 sections=sections, turns=turns, pairs=pairs, k_out=k2) is q2
    assert torch.equal(q2, q_out) and torch.equal(k2, k_out)


@pytest.mark.parametrize("dtype,D,rot", [
    (torch.float32, 264, 2), (torch.bfloat16, 320, 20), (torch.float16, 264, 6), (torch.bfloat16, 1032, 8),
    (torch.float16, 2056, 16), (torch.bfloat16, 256, 2), (torch.float32, 1028, 8), (torch.float32, 516, 4),
])
def test_rope_of_heads_with_more_vectors_than_threads(dtype, D, rot):
    """v's rows of more than 256 vectors (of 1, 2, 4 and 8 elements) reach the cache whole."""
    T, H, KVH, block = 11, 2, 2, 4
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").to(dtype) for h in (H, KVH, KVH))
    cache = torch.full((5, block, KVH, 2 * D), NAN, device="cuda").to(dtype)
    lg = cache.permute(0, 2, 1, 3)
    pos = torch.randint(0, 50, (T,), generator=g, device="cuda")
    cs = _cos_sin(50, rot)
    slots = torch.randperm(5 * block, generator=g, device="cuda")[:T]
    slots[3] = -1
    q_out, k_out = torch.full_like(q, NAN), torch.full_like(k, NAN)
    gpu_ops.rope_store_kv(q, k, v, pos, cs, slots, (KVTier(lg[..., :D], lg[..., D:]), None), 5, q_out=q_out, k_out=k_out)
    gpu_ops.check_device_errors(dev())
    axis = gpu_ops.rope_axes((rot // 2,))
    _rope_ok(q_out, ref.rope(q, pos[None], cs, axis, False), q, dtype)
    _rope_ok(k_out, ref.rope(k, pos[None], cs, axis, False), k, dtype)
    rows, kept = cache.view(-1, KVH, 2 * D), slots >= 0
    assert torch.equal(rows[slots[kept], :, D:], v[kept]) and torch.equal(rows[slots[kept], :, :D], k_out[kept])
    rest = torch.ones(rows.shape[0], dtype=torch.bool, device="cuda")
    rest[slots[kept]] = False
    assert bool(rows[rest].isnan().all())


def test_rope_skips_what_is_out_of_range():
    T, H, KVH, D = 6, 2, 1, 64
    q, k, v = (torch.randn(T, h, D, device="cuda") for h in (H, KVH, KVH))
    cache = torch.zeros(2, 4, KVH, 2 * D, device="cuda")
    lg = cache.permute(0, 2, 1, 3)
    tiers = (KVTier(lg[..., :D], lg[..., D:]), None)
    pos = torch.tensor([[0, 1, 8, 3, 4, 5], [0, -1, 2, 3, 4, 5]], device="cuda")
    slots = torch.tensor([0, 1, 2, 8, 5, 6], device="cuda")
    out = torch.full_like(q, NAN)
    gpu_ops.rope_store_kv(q, k, v, pos, _cos_sin(8, 64), slots, tiers, 2, sections=(16, 16), q_out=out)
    with pytest.raises(RuntimeError, match="position|slot"):
        gpu_ops.check_device_errors(dev())
    assert bool(out[1:3].isnan().all()) and not bool(out[[0, 3, 4, 5]].isnan().any())
    rows = cache.view(8, 2 * D)
    assert bool((rows[[1, 2, 3, 4, 7]] == 0).all()) and torch.equal(rows[[0, 5, 6], D:], v[[0, 4, 5], 0])


def test_rope_of_no_tokens_and_refusals():
    z = torch.zeros(0, 2, 64, device="cuda", dtype=torch.float16)
    gpu_ops.rope_store_kv(z, z, z, torch.zeros(0, dtype=torch.int64, device="cuda"), _cos_sin(4, 64), None, (None, None), 0)
    q = torch.zeros(3, 2, 64, device="cuda", dtype=torch.float16)
    pos, cs = torch.zeros(3, dtype=torch.int64, device="cuda"), _cos_sin(4, 64)
    for kw, match in ((dict(sections=(16, 16)), "row per axis"), (dict(sections=(30,)), "add up"),
                      (dict(q_out=q[:2]), "shape")):
        with pytest.raises(RuntimeError, match=match):
            gpu_ops.rope_store_kv(q, q, q, pos, cs, None, (None, None), 0, **kw)
    for args, match in (((q, q, q.float(), pos, cs), "dtype"), ((q, q, q, pos.int(), cs), "int64"),
                        ((q, q, q, pos, cs.double()), "fp32"), ((q, q, q, pos[:2], cs), "int64"),
                        ((q, q[:2], q[:2], pos, cs), "KVH")):
        with pytest.raises(RuntimeError, match=match):
            gpu_ops.rope_store_kv(*args, None, (None, None), 0)
    with pytest.raises(RuntimeError, match="tier is required"):
        gpu_ops.rope_store_kv(q, q, q, pos, cs, pos, (None, None), 0)


# ------------------------------------------------------------------ attention


def _rounded(dtype):
    return dtype != torch.float32


def _paged(kl, KVH, D, block, dtype, g, host_share=0.0, pad=0):
    """A cache whose blocks hold the requests' K/V and NaN everywhere else."""
    held = [-(-x // block) for x in kl]
    total = sum(held) + 3
    n_host = int(total * host_share)
    n_hbm = total - n_host
    cache = torch.full((n_hbm, block, KVH, 2 * D + pad), NAN, device="cuda").to(dtype)
    hk = torch.full((max(1, n_host), KVH, block, D), NAN).to(dtype)
    hv = hk.clone()
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(5)).tolist()
    W = max(held) + 2
    table = torch.full((len(kl), W), 1 << 29, dtype=torch.int32)  # unused entries are never read
    keys, vals = [], []
    for r, n in enumerate(kl):
        k = torch.randn(n, KVH, D, generator=g, device="cuda").to(dtype)
        v = torch.randn(n, KVH, D, generator=g, device="cuda").to(dtype)
        keys.append(k)
        vals.append(v)
        kc, vc = k.cpu(), v.cpu()
        for b in range(held[r]):
            i = perm.pop()
            table[r, b] = i
            lo, hi = b * block, min(n, (b + 1) * block)
            if i < n_hbm:
                cache[i, :hi - lo, :, :D], cache[i, :hi - lo, :, D:2 * D] = k[lo:hi], v[lo:hi]
            else:
                hk[i - n_hbm, :, :hi - lo] = kc[lo:hi].transpose(0, 1)
                hv[i - n_hbm, :, :hi - lo] = vc[lo:hi].transpose(0, 1)
    lg = cache.permute(0, 2, 1, 3)
    tiers = (KVTier(lg[..., :D], lg[..., D:2 * D]), KVTier(hk.pin_memory(), hv.pin_memory()) if n_host else None)
    return keys, vals, table.cuda(), tiers, n_hbm


def _queries(ql, H, D, dtype, g, gap=2):
    start, at = [], 1
    for n in ql:
        start.append(at)
        at += n + gap
    T = at + 1
    q = torch.randn(T, H + 1, D, generator=g, device="cuda").to(dtype)[:, :H]
    covered = torch.zeros(T, dtype=torch.bool, device="cuda")
    for s, n in zip(start, ql):
        covered[s:s + n] = True
    q.masked_fill_(~covered[:, None, None], NAN)  # rows of no request are never used
    out = torch.full((T, H, D), NAN, device="cuda").to(dtype)
    lse = torch.full((T, H), NAN, device="cuda").T
    return q, start, out, lse


def _refs(q, start, ql, keys, vals, limits, scale):
    return [ref.attend(q[s:s + n], k, v, lim, scale) + (k.shape[0],)
            for s, n, k, v, lim in zip(start, ql, keys, vals, limits)]


LENS = {
    "edges": ([1, 0, 3, 1, 5, 130, 2], [1, 4, 3, 700, 2, 130, 0]),
    "verify": ([4, 7, 1, 5], [1000, 33, 129, 2049]),
    "one": ([3], [5000]),
    "chunks": ([300, 65, 257], [300, 1100, 640]),
    "tokens": ([1, 1, 0, 1, 1, 1, 1, 1], [1, 5000, 4, 0, 129, 128, 127, 640]),
}


@pytest.mark.parametrize("dtype,H,KVH,D,block,host,lens", [
    (torch.bfloat16, 8, 2, 128, 16, 0.0, "edges"), (torch.bfloat16, 8, 2, 128, 16, 0.0, "verify"),
    (torch.bfloat16, 8, 2, 128, 16, 0.0, "chunks"), (torch.bfloat16, 32, 8, 128, 16, 0.0, "one"),
    (torch.float16, 4, 4, 64, 16, 0.0, "edges"), (torch.float16, 8, 1, 64, 32, 0.0, "chunks"),
    (torch.float16, 8, 2, 128, 16, 0.4, "edges"), (torch.bfloat16, 8, 2, 128, 16, 0.4, "chunks"),
    (torch.float16, 5, 1, 80, 24, 0.3, "edges"), (torch.bfloat16, 14, 2, 96, 8, 0.0, "chunks"),
    (torch.bfloat16, 6, 2, 72, 1, 0.2, "verify"), (torch.float16, 3, 1, 40, 16, 0.0, "edges"),
    (torch.bfloat16, 20, 4, 128, 64, 0.0, "chunks"), (torch.float16, 64, 1, 128, 16, 0.0, "verify"),
    (torch.bfloat16, 4, 2, 8, 5, 0.0, "edges"), (torch.bfloat16, 8, 2, 192, 16, 0.3, "edges"),
    (torch.float16, 4, 1, 256, 16, 0.0, "chunks"), (torch.float32, 8, 2, 64, 16, 0.3, "edges"),
    (torch.bfloat16, 8, 2, 128, 16, 0.0, "tokens"), (torch.float16, 4, 4, 64, 16, 0.5, "tokens"),
    (torch.bfloat16, 32, 1, 64, 16, 0.0, "tokens"), (torch.float16, 20, 1, 112, 8, 0.2, "tokens"),
    (torch.float16, 8, 2, 64, 16, 0.0, "verify"), (torch.bfloat16, 2, 2, 80, 64, 0.0, "verify"),
    (torch.float16, 3, 1, 64, 24, 0.0, "verify"), (torch.bfloat16, 4, 2, 128, 128, 0.3, "chunks"),
    (torch.float16, 4, 2, 64, 12, 0.3, "chunks"), (torch.bfloat16, 8, 2, 128, 40, 0.0, "verify"),
    (torch.float16, 8, 8, 128, 256, 0.0, "tokens"), (torch.bfloat16, 8, 2, 64, 32, 0.2, "edges"),
    (torch.float32, 8, 2, 128, 16, 0.0, "verify"), (torch.float32, 4, 4, 256, 24, 0.0, "edges"),
    (torch.float32, 6, 2, 36, 16, 0.0, "chunks"), (torch.float32, 64, 1, 64, 16, 0.0, "verify"),
])
def test_chunk_attention(dtype, H, KVH, D, block, host, lens):
    ql, kl = LENS[lens]
    g = torch.Generator(device="cuda").manual_seed(H * D + block)
    keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, block, dtype, g, host, pad=8 if dtype != torch.float32 else 4)
    q, start, out, lse = _queries(ql, H, D, dtype, g)
    scale = D ** -0.5
    lim = [k - n + torch.arange(n, device="cuda") for n, k in zip(ql, kl)]
    refs = _refs(q, start, ql, keys, vals, lim, scale)
    gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), scale, out, lse, max_q_len=max(ql),
                       max_k_len=max(kl))
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, ql, dtype, D, _rounded(dtype))
    # bounds that are too small cost time, not the result
    out3 = torch.full_like(out, NAN)
    gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), scale, out3, lse, max_q_len=1, max_k_len=1)
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out3, lse, refs, start, ql, dtype, D, _rounded(dtype))
    # table rows in another order, no bounds, no lse: the same result
    order = list(range(len(ql)))[::-1]
    out2 = torch.full_like(out, NAN)
    gpu_ops.chunk_attn(q, tiers, n_hbm, table[order].contiguous(), i32(start), i32(ql), i32(kl), scale, out2,
                       bt_row=i32([order.index(r) for r in range(len(ql))]))
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out2, None, refs, start, ql, dtype, D, _rounded(dtype))


@pytest.mark.parametrize("dtype,D,ql,kl", [
    (torch.float32, 64, 3, 6000), (torch.float32, 256, 1, 6000), (torch.float16, 256, 2, 6000), (torch.bfloat16, 64, 1, 40000),
    (torch.float16, 128, 20, 30000), (torch.bfloat16, 128, 50, 40000), (torch.float16, 80, 200, 20000),
])
def test_one_item_over_most_of_the_gpu(dtype, D, ql, kl):
    """An item cut into more parts than the combine takes per round."""
    g = torch.Generator(device="cuda").manual_seed(kl + D)
    keys, vals, table, tiers, n_hbm = _paged([kl], 1, D, 16, dtype, g)
    q, start, out, lse = _queries([ql], 1, D, dtype, g)
    scale = D ** -0.5
    refs = _refs(q, start, [ql], keys, vals, [kl - ql + torch.arange(ql, device="cuda")], scale)
    gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32([ql]), i32([kl]), scale, out, lse, max_q_len=ql, max_k_len=kl)
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, [ql], dtype, D, _rounded(dtype))


@pytest.mark.parametrize("dtype,D,block", [(torch.bfloat16, 128, 16), (torch.float16, 128, 8), (torch.float16, 64, 16),
                                           (torch.bfloat16, 96, 64), (torch.float32, 64, 16)])
@pytest.mark.parametrize("lens", ["verify", "chunks"])
@pytest.mark.parametrize("layout", ["heads first", "gap behind blocks", "tokens first"])
def test_chunk_attention_over_other_layouts(dtype, D, block, lens, layout):
    ql, kl = LENS[lens]
    H, KVH = 6, 2
    g = torch.Generator(device="cuda").manual_seed(D + block)
    keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, block, dtype, g)
    _, start, out, lse = _queries(ql, H, D, dtype, g)

    def lay(t):
        B = t.shape[0]
        if layout == "heads first":
            return t.contiguous()
        if layout == "tokens first":
            return t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        n = KVH * block * D  # the block stride is no multiple of the head stride
        x = torch.full((B, n + 16), NAN, device="cuda").to(dtype).as_strided((B, KVH, block, D), (n + 16, block * D, D, 1))
        return x.copy_(t)

    tiers = (KVTier(lay(tiers[0].k), lay(tiers[0].v)), None)
    q = torch.randn(1, H, D, generator=g, device="cuda").to(dtype).expand(out.shape)  # one query row for all tokens
    scale = D ** -0.5
    lim = [k - n + torch.arange(n, device="cuda") for n, k in zip(ql, kl)]
    refs = _refs(q, start, ql, keys, vals, lim, scale)
    gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), scale, out, lse, max_q_len=max(ql),
                       max_k_len=max(kl))
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, ql, dtype, D, _rounded(dtype))


@pytest.mark.parametrize("dtype,H,KVH,D", [
    (torch.bfloat16, 8, 2, 128), (torch.float16, 20, 20, 64), (torch.float16, 5, 1, 80), (torch.bfloat16, 7, 1, 112),
    (torch.float32, 4, 4, 64), (torch.float32, 8, 1, 128), (torch.bfloat16, 4, 2, 256),
])
@pytest.mark.parametrize("lens", ["edges", "verify", "chunks", "tokens"])
def test_cross_attention(dtype, H, KVH, D, lens):
    ql, kl = LENS[lens]
    g = torch.Generator(device="cuda").manual_seed(H * D)
    S = sum(kl) + 9
    kv = torch.randn(S, KVH, 2 * D, generator=g, device="cuda").to(dtype)
    k_start = [3 + sum(kl[:i]) for i in range(len(kl))]
    k_start[-1] = min(k_start[-1], 2)  # shares the first requests' states
    used = torch.zeros(S, dtype=torch.bool, device="cuda")
    for s, n in zip(k_start, kl):
        used[s:s + n] = True
    kv.masked_fill_(~used[:, None, None], NAN)
    k, v = kv[..., :D], kv[..., D:]
    q, start, out, lse = _queries(ql, H, D, dtype, g)
    lim = [torch.full((n,), x - 1, device="cuda") for n, x in zip(ql, kl)]
    refs = _refs(q, start, ql, [k[s:s + n] for s, n in zip(k_start, kl)], [v[s:s + n] for s, n in zip(k_start, kl)], lim,
                 0.11)
    for bound in (0, max(ql)):
        out.fill_(NAN)
        gpu_ops.cross_attn(q, k, v, i32(start), i32(ql), i32(k_start), i32(kl), 0.11, out, lse, max_q_len=bound)
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, ql, dtype, D, _rounded(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_requests_more_than_one_scan_round(dtype):
    rnd = random.Random(3)
    n = 700
    ql = [rnd.choice([0, 1, 2, 40]) for _ in range(n)]
    kl = [rnd.choice([0, q, q + rnd.randint(0, 90)]) for q in ql]
    g = torch.Generator(device="cuda").manual_seed(1)
    H, KVH, D = 4, 2, 64
    keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, 16, dtype, g)
    q, start, out, lse = _queries(ql, H, D, dtype, g, gap=0)
    refs = _refs(q, start, ql, keys, vals, [k - m + torch.arange(m, device="cuda") for m, k in zip(ql, kl)], 0.125)
    gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), 0.125, out, lse)
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, ql, dtype, D, _rounded(dtype))


@pytest.mark.parametrize("bound", [0, 6])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_scores_far_apart(dtype, bound):
    """Rows whose maximum grows late and by a lot, and rows of equal scores."""
    H, KVH, D, nk = 4, 1, 64, 2500
    g = torch.Generator(device="cuda").manual_seed(2)
    keys, vals, table, tiers, n_hbm = _paged([nk], KVH, D, 16, dtype, g)
    q, start, out, lse = _queries([6], H, D, dtype, g)
    q[1:7, 0] *= 40
    q[1:7, 1] = 0
    for i, j in enumerate(range(200, nk, 450)):  # ever larger scores, far apart
        page, at = int(table[0, j // 16]), j % 16
        keys[0][j] = (q[3, 2] * (1 + i)).unsqueeze(0)
        tiers[0].k[page, :, at] = keys[0][j]
    refs = _refs(q, start, [6], keys, vals, [nk - 6 + torch.arange(6, device="cuda")], 0.7)
    gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32([6]), i32([nk]), 0.7, out, lse, max_q_len=bound)
    ref.check_attn(out, lse, refs, start, [6], dtype, D, _rounded(dtype))


@pytest.mark.parametrize("dtype,D,ql,kl", [
    (torch.bfloat16, 128, [1, 4], [70, 9000]), (torch.float16, 64, [2, 1], [3000, 5]), (torch.bfloat16, 128, [20, 30], [40, 9000]),
    (torch.float16, 64, [90, 300], [90, 5000]), (torch.float32, 64, [3, 40], [100, 4000]), (torch.bfloat16, 256, [2, 9], [50, 3000]),
])
def test_a_nan_in_a_query_is_its_own_rows_alone(dtype, D, ql, kl):
    """o and lse of the (query, head) are NaN, whole or cut into parts; the lse of a
    row without keys, -inf, stays apart."""
    H, KVH = 4, 2
    g = torch.Generator(device="cuda").manual_seed(D)
    keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, 16, dtype, g)
    q, start, out, lse = _queries(ql, H, D, dtype, g)
    scale = D ** -0.5
    lim = [k - n + torch.arange(n, device="cuda") for n, k in zip(ql, kl)]
    refs = _refs(q, start, ql, keys, vals, lim, scale)
    hit = [(start[0], 1, 0), (start[1] + ql[1] - 1, 3, D - 1), (start[1], 0, 7)]
    for t, h, d in hit:
        q[t, h, d] = NAN
    gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), scale, out, lse, max_q_len=max(ql),
                       max_k_len=max(kl))
    gpu_ops.check_device_errors(dev())
    for t, h, _ in hit:
        assert bool(out[t, h].isnan().all()) and bool(lse[h, t].isnan())
        r = 0 if t == start[0] else 1
        out[t, h], lse[h, t] = refs[r][0][t - start[r], h].to(dtype), refs[r][1][h, t - start[r]].float()
    ref.check_attn(out, lse, refs, start, ql, dtype, D, _rounded(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_requests_that_do_not_fit_write_nothing(dtype):
    H, KVH, D = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    ql, kl = [2, 3, 2, 2], [40, 30, 50, 20]
    keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, 16, dtype, g)
    q, start, out, lse = _queries(ql, H, D, dtype, g)
    T = q.shape[0]
    refs = _refs(q, start, ql, keys, vals, [k - n + torch.arange(n, device="cuda") for n, k in zip(ql, kl)], 0.1)
    W = table.shape[1]
    for bad in ([start, ql, [40, 30, 16 * W + 1, 20]], [start[:2] + [T - 1] + start[3:], ql, kl], [start, [2, 3, -1, 2], kl],
                [start, ql, [40, 30, -5, 20]], [start[:2] + [-1] + start[3:], ql, kl]):
        out.fill_(NAN)
        lse.fill_(NAN)
        gpu_ops.chunk_attn(q, tiers, n_hbm, table, *(i32(x) for x in bad), 0.1, out, lse)
        with pytest.raises(RuntimeError, match="sequence length"):
            gpu_ops.check_device_errors(dev())
        some = [0, 1, 3]
        ref.check_attn(out, lse, [refs[i] for i in some], [start[i] for i in some], [ql[i] for i in some], dtype, D,
                       _rounded(dtype))
    # a block id outside both tiers is not read, the others' rows are right
    t2 = table.clone()
    t2[2, 1] = n_hbm + 100
    out.fill_(NAN)
    gpu_ops.chunk_attn(q, tiers, n_hbm, t2, i32(start), i32(ql), i32(kl), 0.1, out)
    with pytest.raises(RuntimeError, match="block id"):
        gpu_ops.check_device_errors(dev())
    ref.check_attn(out, None, [refs[i] for i in some], [start[i] for i in some], [ql[i] for i in some], dtype, D,
                   _rounded(dtype), untouched=False)
    k = torch.randn(50, KVH, D, device="cuda").to(dtype)
    o2 = torch.full_like(out, NAN)
    gpu_ops.cross_attn(q, k, k, i32(start), i32(ql), i32([0, 30, -1, 49]), i32([5, 21, 3, 2]), 0.1, o2)
    with pytest.raises(RuntimeError, match="sequence length"):
        gpu_ops.check_device_errors(dev())
    assert bool(o2[start[1]:].isnan().all()) and not bool(o2[start[0]:start[0] + 2].isnan().any())


@pytest.mark.parametrize("dtype,H,q_extra", [(torch.bfloat16, 4, 0), (torch.float16, 8, 60), (torch.float32, 4, 0)])
def test_requests_whose_table_row_does_not_exist_write_nothing(dtype, H, q_extra):
    KVH, D = 2, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    ql, kl = [2, 3, 2 + q_extra, 2], [40, 30, 80, 20]
    keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, 16, dtype, g, host_share=0.3)
    q, start, out, lse = _queries(ql, H, D, dtype, g)
    refs = _refs(q, start, ql, keys, vals, [k - n + torch.arange(n, device="cuda") for n, k in zip(ql, kl)], 0.1)
    some = [0, 1, 3]
    for row in (4, -1, 1 << 30, -(1 << 31), 2**31 - 1):
        out.fill_(NAN)
        lse.fill_(NAN)
        gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), 0.1, out, lse, bt_row=i32([0, 1, row, 3]),
                           max_q_len=max(ql))
        with pytest.raises(RuntimeError, match="sequence length"):
            gpu_ops.check_device_errors(dev())
        ref.check_attn(out, lse, [refs[i] for i in some], [start[i] for i in some], [ql[i] for i in some], dtype, D,
                       _rounded(dtype))
    # a request without queries needs no row
    gpu_ops.chunk_attn(q, tiers, n_hbm, table, i32(start), i32([2, 3, 0, 2]), i32(kl), 0.1, out, lse, bt_row=i32([0, 1, 99, 3]))
    gpu_ops.check_device_errors(dev())


def test_attention_refusals():
    q = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    i, one = i32([0]), i32([1])
    for args, match in (((q, q.float(), q, i, one, i, one), "dtype"), ((q, q, q, i.long(), one, i, one), "int32"),
                        ((q, q, q, i, one, i[:0], one), "int32"), ((q, q[..., :56], q[..., :56], i, one, i, one), "head size")):
        with pytest.raises(RuntimeError, match=match):
            gpu_ops.cross_attn(*args, 1.0, torch.empty_like(q))
    with pytest.raises(RuntimeError, match="lse"):
        gpu_ops.cross_attn(q, q, q, i, one, i, one, 1.0, torch.empty_like(q), torch.empty(4, 2, device="cuda"))
    with pytest.raises(RuntimeError, match="scale"):
        gpu_ops.cross_attn(q, q, q, i, one, i, one, 0.0, torch.empty_like(q))
    with pytest.raises(RuntimeError, match="workspace_buf"):
        gpu_ops.cross_attn(q, q, q, i, one, i, one, 1.0, torch.empty_like(q),
                           workspace_buf=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="row per request"):
        gpu_ops.chunk_attn(q, (KVTier(q.view(1, 4, 2, 64), q.view(1, 4, 2, 64)), None), 1, i32([[0]]), i32([0, 1]),
                           i32([1, 1]), i32([1, 1]), 1.0, torch.empty_like(q))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_two_streams_and_two_graphs_at_once(dtype, many):
    """Calls share no scratch memory: two captured graphs replayed on two
    streams at the same time give what each gives alone, bit for bit."""
    H, KVH, D = 8, 2, 128
    g = torch.Generator(device="cuda").manual_seed(4)
    sides = []
    for ql, kl in ((([300, 5], [3000, 2000]), ([2, 400, 1], [2500, 500, 4000])) if many else
                   (([3, 5], [3000, 2000]), ([2, 4, 1], [2500, 100, 4000]))):
        keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, 16, dtype, g)
        q, start, out, lse = _queries(ql, H, D, dtype, g)
        args = (q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), 0.1)
        args_kw = dict(max_q_len=max(ql))
        gpu_ops.chunk_attn(*args, out, lse, **args_kw)
        torch.cuda.synchronize()
        alone = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gpu_ops.chunk_attn(*args, out, lse, **args_kw)
        sides.append((graph, torch.cuda.Stream(), out, alone, args, (lse, args_kw)))
    for _ in range(20):
        for graph, stream, out, *_ in sides:
            with torch.cuda.stream(stream):
                out.fill_(NAN)
                graph.replay()
    torch.cuda.synchronize()
    for _, stream, out, alone, args, lse in sides:
        assert torch.equal(torch.nan_to_num(out.float()), torch.nan_to_num(alone.float()))
    for _ in range(20):
        for _, stream, out, alone, args, (lse, kw) in sides:
            with torch.cuda.stream(stream):
                gpu_ops.chunk_attn(*args, out, lse, **kw)
    torch.cuda.synchronize()
    for _, stream, out, alone, *_ in sides:
        assert torch.equal(torch.nan_to_num(out.float()), torch.nan_to_num(alone.float()))


def _repeat_beside_copies(call, out, times):
    """Call again and again while another stream copies, so that loads land late
    and out of order; every result has to be the first one, bit for bit."""
    out.fill_(NAN)
    call()
    gpu_ops.check_device_errors(dev())
    first, differ = out.clone(), torch.zeros((), dtype=torch.int64, device="cuda")
    side, big = torch.cuda.Stream(), torch.empty(1 << 27, dtype=torch.uint8, device="cuda")
    bits = torch.int16 if out.element_size() == 2 else torch.int32
    for i in range(times):
        if i % 8 == 0:
            with torch.cuda.stream(side):
                big[: 1 << 26].copy_(big[1 << 26:])
        out.fill_(NAN)
        call()
        differ += (out.view(bits) != first.view(bits)).sum()
    torch.cuda.synchronize()
    gpu_ops.check_device_errors(dev())
    assert int(differ) == 0


@pytest.mark.parametrize("dtype,D,block", [(torch.bfloat16, 128, 16), (torch.float16, 64, 16), (torch.bfloat16, 96, 64)])
def test_single_tiles_over_many_key_tiles(dtype, D, block):
    """Requests of one query tile, whose key tiles both streams of the tensor-core
    kernel share: over more tiles than the rings hold, the last one half or
    barely seen."""
    H, KVH = 8, 2
    ql = [9, 32, 20, 31, 12, 32, 10]
    kl = [9000, 4097, 129, 2048, 2049, 6464, 65]
    g = torch.Generator(device="cuda").manual_seed(D)
    keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, block, dtype, g)
    q, start, out, lse = _queries(ql, H, D, dtype, g)
    scale = D ** -0.5
    refs = _refs(q, start, ql, keys, vals, [k - n + torch.arange(n, device="cuda") for n, k in zip(ql, kl)], scale)
    args = (q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), scale, out, lse)
    call = lambda: gpu_ops.chunk_attn(*args, max_q_len=max(ql), max_k_len=max(kl))  # noqa: E731
    call()
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, ql, dtype, D, True)
    _repeat_beside_copies(call, out, 400)


@pytest.mark.parametrize("dtype,D,nq", [(torch.bfloat16, 128, 1), (torch.float16, 64, 40), (torch.float32, 64, 3),
                                        (torch.bfloat16, 256, 5)])
def test_cross_attention_without_any_states(dtype, D, nq):
    H, KVH, n = 8, 2, 3
    q = torch.randn(n * nq + 2, H, D, device="cuda").to(dtype)
    k = torch.empty(0, KVH, D, device="cuda", dtype=dtype)
    start, ql, none = i32([i * nq for i in range(n)]), i32([nq] * n), i32([0] * n)
    for bound in (0, nq):
        out, lse = torch.full_like(q, NAN), torch.full((H, q.shape[0]), NAN, device="cuda")
        gpu_ops.cross_attn(q, k, k, start, ql, none, none, 0.1, out, lse, max_q_len=bound)
        gpu_ops.check_device_errors(dev())
        assert bool((out[:n * nq] == 0).all()) and bool((lse[:, :n * nq] == float("-inf")).all())
        assert bool(out[n * nq:].isnan().all()) and bool(lse[:, n * nq:].isnan().all())
    # a request that claims a key writes nothing
    out.fill_(NAN)
    gpu_ops.cross_attn(q, k, k, start, ql, none, i32([0, 1, 0]), 0.1, out, lse)
    with pytest.raises(RuntimeError, match="sequence length"):
        gpu_ops.check_device_errors(dev())
    assert bool(out[nq:2 * nq].isnan().all()) and bool((out[:nq] == 0).all())


def _keyless_batch(dtype, KVH, G, D, nq, n, seed):
    """cross_attn of n requests of up to nq tokens, most of which have no states."""
    rnd = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    ql = [rnd.randint(max(1, nq // 2), nq) for _ in range(n)]
    kl = [rnd.choice([0, 0, 0, rnd.randint(1, 700)]) for _ in range(n)]
    S = sum(kl)
    k, v = (torch.randn(S, KVH, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    k_start = [sum(kl[:i]) for i in range(n)]
    q, start, out, lse = _queries(ql, KVH * G, D, dtype, g, gap=0)
    refs = _refs(q, start, ql, [k[s:s + x] for s, x in zip(k_start, kl)], [v[s:s + x] for s, x in zip(k_start, kl)],
                 [torch.full((m,), x - 1, device="cuda") for m, x in zip(ql, kl)], 0.1)
    return ql, start, out, lse, refs, (q, k, v, i32(start), i32(ql), i32(k_start), i32(kl), 0.1, out, lse)


@pytest.mark.parametrize("dtype,KVH,G,D,nq", [(torch.bfloat16, 2, 4, 128, 1), (torch.float16, 5, 1, 64, 1),
                                              (torch.bfloat16, 2, 4, 128, 4), (torch.float16, 3, 2, 64, 14)])
def test_requests_without_keys_among_others_few_rows(dtype, KVH, G, D, nq):
    ql, start, out, lse, refs, args = _keyless_batch(dtype, KVH, G, D, nq, 300, nq + D)
    call = lambda: gpu_ops.cross_attn(*args, max_q_len=nq)  # noqa: E731
    call()
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, ql, dtype, D, True)
    _repeat_beside_copies(call, out, 2000)


@pytest.mark.parametrize("dtype,KVH,G,D,nq", [(torch.bfloat16, 2, 4, 128, 30), (torch.float16, 3, 1, 64, 90),
                                              (torch.bfloat16, 1, 4, 96, 150)])
def test_requests_without_keys_among_others_many_rows(dtype, KVH, G, D, nq):
    ql, start, out, lse, refs, args = _keyless_batch(dtype, KVH, G, D, nq, 300, nq + D)
    call = lambda: gpu_ops.cross_attn(*args, max_q_len=nq)  # noqa: E731
    call()
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, ql, dtype, D, True)
    _repeat_beside_copies(call, out, 1000)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_pairs_of_tiles_of_which_the_first_sees_nothing(dtype, D):
    """Chunks with more queries than keys: whole pairs of query tiles without keys,
    and pairs whose first tile (32 tokens of 4 heads) has none."""
    H, KVH = 4, 1
    ql = [64, 200, 64, 33, 128, 64, 300, 64] * 12
    kl = [32, 30, 1, 1, 90, 10, 20, 0] * 12
    g = torch.Generator(device="cuda").manual_seed(D)
    keys, vals, table, tiers, n_hbm = _paged(kl, KVH, D, 16, dtype, g)
    q, start, out, lse = _queries(ql, H, D, dtype, g)
    refs = _refs(q, start, ql, keys, vals, [k - n + torch.arange(n, device="cuda") for n, k in zip(ql, kl)], 0.1)
    args = (q, tiers, n_hbm, table, i32(start), i32(ql), i32(kl), 0.1, out, lse)
    call = lambda: gpu_ops.chunk_attn(*args, max_q_len=300)  # noqa: E731
    call()
    gpu_ops.check_device_errors(dev())
    ref.check_attn(out, lse, refs, start, ql, dtype, D, True)
    _repeat_beside_copies(call, out, 1000)


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_steps_together(dtype, D):
    """Several steps of a changing batch: tables from lengths, planned on the
    GPU, rotated K/V written to both tiers, the new tokens attending over the
    cache and over an encoder's states, all inputs staying on the device;
    against dense attention over each request's own history."""
    H, KVH, block, R, W = 8, 2, 16, 5, 24
    hbm, host = 20, 60
    g = torch.Generator(device="cuda").manual_seed(9)
    cache = torch.full((hbm, block, KVH, 2 * D), NAN, device="cuda").to(dtype)
    lg = cache.permute(0, 2, 1, 3)
    hk = torch.full((host, KVH, block, D), NAN).to(dtype).pin_memory()
    tiers = (KVTier(lg[..., :D], lg[..., D:]), KVTier(hk, hk.clone().pin_memory()))
    table = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    free = FreeBlocks(torch.zeros(hbm, dtype=torch.int32, device="cuda"), torch.zeros(host, dtype=torch.int32, device="cuda"),
                      i32([hbm, host]))
    free.hbm.copy_(torch.arange(hbm))
    free.host.copy_(hbm + torch.arange(host))
    enc_len, enc_start = [90, 1, 200, 33, 64], [0, 90, 91, 291, 324]
    enc_k = torch.randn(400, KVH, D, generator=g, device="cuda").to(dtype)
    enc_v = torch.randn(400, KVH, D, generator=g, device="cuda").to(dtype)
    cs = _cos_sin(600, D)
    axis = gpu_ops.rope_axes((D // 4, D // 8, D // 8))
    hist = [([], []) for _ in range(R)]
    out_tabs = StepTables(R, 700, dev(), seq_lens=lens, counts=free.counts)
    steps = [[100, 1, 257, 0, 40], [1, 4, 1, 70, 5], [5, 5, -1, 1, 0], [3, 1, 60, -1, 8], [1, 1, 1, 1, 1]]
    for new in steps:
        qsl_before = [0]
        for n in new:
            qsl_before.append(qsl_before[-1] + max(0, n))
        T = qsl_before[-1]
        gpu_ops.extend_tables(i32(new), lens, table, free, hbm, host, block, out_tabs)
        plan.plan_on_device(out_tabs.query_start_loc, lens, table, out_tabs.slot_mapping, hbm, host, block, max_tokens=T)
        if max(new) > 1:  # the planner's own refusal of extended requests in the host tier is expected here
            gpu_ops.error_word(dev()).zero_()
        q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").to(dtype) for h in (H, KVH, KVH))
        pos = out_tabs.positions[:T].expand(3, T).contiguous()
        k_rot, q_in = torch.empty_like(k), q.clone()
        gpu_ops.rope_store_kv(q, k, v, pos, cs, out_tabs.slot_mapping[:T], tiers, hbm,
                              sections=(D // 4, D // 8, D // 8), k_out=k_rot)
        q_start = out_tabs.query_start_loc[:R]
        q_len = i32([max(0, n) for n in new])
        out, lse = torch.full((T, H, D), NAN, device="cuda").to(dtype), torch.full((H, T), NAN, device="cuda")
        gpu_ops.chunk_attn(q, tiers, hbm, table, q_start, q_len, lens, D ** -0.5, out, lse)
        out_x = torch.full_like(out, NAN)
        gpu_ops.cross_attn(q, enc_k, enc_v, q_start, q_len, i32(enc_start), i32(enc_len), D ** -0.5, out_x)
        gpu_ops.check_device_errors(dev())
        _rope_ok(q, ref.rope(q_in, pos, cs, axis, False), q_in, dtype)
        refs, refs_x = [], []
        for r, n in enumerate(new):
            a, b = qsl_before[r], qsl_before[r + 1]
            if n < 0:
                hist[r] = ([], [])
            hist[r][0].append(k_rot[a:b])
            hist[r][1].append(v[a:b])
            kk, vv = torch.cat(hist[r][0]), torch.cat(hist[r][1])
            assert int(lens[r]) == kk.shape[0]
            refs.append(ref.attend(q[a:b], kk, vv, kk.shape[0] - (b - a) + torch.arange(b - a, device="cuda"), D ** -0.5)
                        + (kk.shape[0],))
            e, s = enc_len[r], enc_start[r]
            refs_x.append(ref.attend(q[a:b], enc_k[s:s + e], enc_v[s:s + e], torch.full((b - a,), e - 1, device="cuda"),
                                     D ** -0.5) + (e,))
        ql = [max(0, n) for n in new]
        ref.check_attn(out, lse, refs, qsl_before[:R], ql, dtype, D, True)
        ref.check_attn(out_x, None, refs_x, qsl_before[:R], ql, dtype, D, True)
    assert bool((table >= hbm).any())  # the batch did spill


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_one_graph_of_a_step_serves_every_step(dtype, D):
    """The step as it is documented, captured once with room for T tokens: steps
    of any size, that end requests, and one that does not fit, each a replay.
    The device's error word is read after every one."""
    H, KVH, block, R, W, T = 8, 2, 16, 6, 20, 420
    hbm, host = 24, 70
    g = torch.Generator(device="cuda").manual_seed(19)
    cache = torch.full((hbm, block, KVH, 2 * D), NAN, device="cuda").to(dtype)
    lg = cache.permute(0, 2, 1, 3)
    hk = torch.full((host, KVH, block, D), NAN).to(dtype).pin_memory()
    tiers = (KVTier(lg[..., :D], lg[..., D:]), KVTier(hk, hk.clone().pin_memory()))
    table = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    new_lens, prior_lens = (torch.zeros(R, dtype=torch.int32, device="cuda") for _ in range(2))
    free = FreeBlocks(torch.arange(hbm, dtype=torch.int32, device="cuda"),
                      hbm + torch.arange(host, dtype=torch.int32, device="cuda"), i32([hbm, host]))
    cs = _cos_sin(600, D)
    axis = gpu_ops.rope_axes((D // 2,))
    t = StepTables(R, T, dev(), seq_lens=prior_lens, counts=free.counts)
    q, k, v = (torch.zeros(T, h, D, device="cuda").to(dtype) for h in (H, KVH, KVH))
    q_rot, k_rot, out = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
    lse = torch.empty(H, T, device="cuda")

    def step():
        gpu_ops.extend_tables(new_lens, prior_lens, table, free, hbm, host, block, t)
        gpu_ops.rope_store_kv(q, k, v, t.positions, cs, t.slot_mapping, tiers, hbm, q_out=q_rot, k_out=k_rot)
        gpu_ops.chunk_attn(q_rot, tiers, hbm, table, t.query_start_loc[:-1], t.query_lens, t.seq_lens, D ** -0.5, out, lse)

    step()  # no new tokens: nothing but the warm-up
    gpu_ops.check_device_errors(dev())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    hist = [([], []) for _ in range(R)]
    for new in ([100, 1, 257, 0, 40, 7], [1, 4, 1, 70, 5, -1], [5, 5, -1, 1, 0, 33], [500, 1, 1, 1, 1, 1], [-1, -1, 9, -1, 8, 1],
                [-1] * R, [2, 130, 1, 0, 1, 19]):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        out.fill_(NAN)
        lse.fill_(NAN)
        before = (table.clone(), prior_lens.clone(), free.counts.clone())
        new_lens.copy_(i32(new))
        graph.replay()
        if sum(max(0, n) for n in new) > T:  # refused: nothing changes, no row is written
            with pytest.raises(RuntimeError, match="block tables"):
                gpu_ops.check_device_errors(dev())
            assert all(torch.equal(a, b) for a, b in zip(before, (table, prior_lens, free.counts)))
            assert bool(out.isnan().all()) and bool(lse.isnan().all())
            continue
        gpu_ops.check_device_errors(dev())
        assert t.read_header()["n_tok"] == sum(max(0, n) for n in new)
        # the planner takes the tables; its own error alone may follow, where a
        # request extends a context in the host tier by several tokens
        plan.plan_on_device(t.query_start_loc, prior_lens, table, t.slot_mapping, hbm, host, block, max_tokens=T)
        code = int(gpu_ops.error_word(dev()))
        assert code == 0 or (code == 6 and max(new) > 1)
        gpu_ops.error_word(dev()).zero_()
        ql = [max(0, n) for n in new]
        start = [sum(ql[:r]) for r in range(R)]
        refs = []
        for r, n in enumerate(new):
            a, b = start[r], start[r] + ql[r]
            if n < 0:
                hist[r] = ([], [])
            hist[r][0].append(k_rot[a:b].clone())
            hist[r][1].append(v[a:b].clone())
            kk, vv = torch.cat(hist[r][0]), torch.cat(hist[r][1])
            assert int(prior_lens[r]) == kk.shape[0]
            refs.append(ref.attend(q_rot[a:b], kk, vv, kk.shape[0] - ql[r] + torch.arange(ql[r], device="cuda"), D ** -0.5)
                        + (kk.shape[0],))
        n = sum(ql)
        if n > 0:
            _rope_ok(q_rot[:n], ref.rope(q[:n], t.positions[None, :n], cs, axis, False), q[:n], dtype)
        ref.check_attn(out, lse, refs, start, ql, dtype, D, _rounded(dtype))
    assert bool((table >= hbm).any())  # the batch did spill
