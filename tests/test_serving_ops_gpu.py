"""GPU tests of the operators behind a step's attention against plain forms
(tests/serving_ref.py): weights per cached key, the choice and the move of the
keys that stay, trimmed tables, verified drafts, and a run of them together."""

from __future__ import annotations

import math
import random
from pathlib import Path

import pytest
import serving_ref as ref
import torch

from vllm_fastdecoder_b200 import gpu_ops
from vllm_fastdecoder_b200.gpu_ops import DraftVerdict, FreeBlocks, KeyMoves, KeyStats, KVTier, StepTables, TrimTables

pytestmark = pytest.mark.gpu
NAN = float("nan")


def dev():
    return torch.device("cuda", torch.cuda.current_device())


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def ok():
    gpu_ops.check_device_errors(dev())


def fails(text):
    with pytest.raises(RuntimeError, match=text):
        gpu_ops.check_device_errors(dev())


# ------------------------------------------------------------------ a paged cache


class Paged:
    """Requests of these lengths over shuffled blocks of both tiers; what no
    request holds is NaN."""

    def __init__(self, lens, KVH, BS, D, dtype, host=0.0, seed=0, layout="interleaved", spare=3):
        rnd = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        held = [-(-n // BS) for n in lens]
        total = sum(held)
        self.C = int(total * host)
        self.G = total - self.C + spare
        ids = [b if b < total - self.C else self.G + b - (total - self.C) for b in range(total)]
        rnd.shuffle(ids)
        W = max(held + [1]) + 2
        rows, at = [], 0
        for h in held:
            rows.append(ids[at:at + h] + [-9] * (W - h))
            at += h
        self.rows, self.lens, self.BS, self.KVH, self.D = rows, lens, BS, KVH, D
        self.table = i32(rows)
        blocks = self.G + self.C
        keys = [torch.randn(n, KVH, D, generator=g).to(dtype) for n in lens]
        vals = [torch.randn(n, KVH, D, generator=g).to(dtype) for n in lens]
        k = torch.full((blocks, KVH, BS, D), NAN).to(dtype)
        v = k.clone()
        for r, n in enumerate(lens):
            for b in range(held[r]):
                m = min(BS, n - b * BS)
                k[rows[r][b], :, :m] = keys[r][b * BS:b * BS + m].transpose(0, 1)
                v[rows[r][b], :, :m] = vals[r][b * BS:b * BS + m].transpose(0, 1)
        self.k0, self.v0, self.keys, self.vals = k, v, keys, vals
        if layout == "interleaved":
            c = torch.cat([k[:self.G], v[:self.G]], -1).transpose(1, 2).contiguous().cuda()
            hk, hv = c.transpose(1, 2)[..., :D], c.transpose(1, 2)[..., D:]
        elif layout == "tokens":
            hk, hv = (x[:self.G].transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (k, v))
        else:
            hk, hv = (x[:self.G].contiguous().cuda() for x in (k, v))
        host_tier = KVTier(k[self.G:].contiguous().pin_memory(), v[self.G:].contiguous().pin_memory()) if self.C else None
        self.tiers = (KVTier(hk, hv), host_tier)

    def now(self):
        """K and V of all blocks as they are now, on the host."""
        torch.cuda.synchronize()
        out = []
        for name in ("k", "v"):
            parts = [getattr(self.tiers[0], name).cpu()]
            if self.tiers[1] is not None:
                parts.append(getattr(self.tiers[1], name).clone())
            out.append(torch.cat(parts))
        return out

    def stats(self, seed=1):
        g = torch.Generator().manual_seed(seed)
        shape = (self.G + self.C, self.KVH, self.BS)
        return KeyStats(torch.rand(shape, generator=g).cuda(), torch.randint(0, 99, shape, generator=g, dtype=torch.int32).cuda())

    def places(self, r, n=None):
        """(blocks, offsets) of request r's keys."""
        j = torch.arange(self.lens[r] if n is None else n)
        return torch.tensor(self.rows[r], dtype=torch.int64)[j // self.BS], j % self.BS


# ------------------------------------------------------------------ weights


def _lse(q, keys, q_lens, scale):
    """[H, T] fp32, of float64."""
    H = q.shape[1]
    out, at = torch.zeros(H, q.shape[0], device="cuda"), 0
    for k, nq in zip(keys, q_lens):
        nk, KVH = k.shape[0], k.shape[1]
        kd = k.cuda().double().transpose(0, 1).repeat_interleave(H // KVH, 0)
        s = q[at:at + nq].double().transpose(0, 1) @ kd.transpose(1, 2) * scale
        seen = torch.arange(nk, device="cuda") <= (nk - nq + torch.arange(nq, device="cuda"))[:, None]
        s = s.masked_fill(~seen, -math.inf)
        out[:, at:at + nq] = (torch.logsumexp(s, -1) if nk else torch.full((H, nq), -math.inf, device="cuda")).float()
        at += nq
    return out


def _weights_case(q_lens, k_lens, H, KVH, D, BS, dtype, host=0.0, layout="interleaved", seed=0, gap=0, hints=None, evicted=True):
    pg = Paged(k_lens, KVH, BS, D, dtype, host, seed, layout)
    T = sum(q_lens) + gap
    g = torch.Generator().manual_seed(seed + 9)
    q = torch.randn(T, H, D, generator=g).to(dtype).cuda()
    q[sum(q_lens):] = NAN
    scale = D ** -0.5
    lse = _lse(q[:sum(q_lens)], pg.keys, q_lens, scale)
    lse = torch.cat([lse, torch.full((H, gap), NAN, device="cuda")], 1)
    start = [sum(q_lens[:i]) for i in range(len(q_lens))]
    stats = pg.stats()
    w0, p0 = stats.weights.clone(), stats.positions.clone()
    gone = [7 * r for r in range(len(q_lens))]
    mq, mk = hints if hints is not None else (max(q_lens), max(k_lens))
    gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, i32(start), i32(q_lens), i32(k_lens), scale, lse, stats,
                        evicted=i32(gone) if evicted else None, max_q_len=mq, max_k_len=mk)
    ok()
    _check_weights(pg, q, lse, q_lens, k_lens, start, scale, stats, w0, p0, gone if evicted else [0] * len(gone))
    return pg, q, lse, start, scale, stats


def _check_weights(pg, q, lse, q_lens, k_lens, start, scale, stats, w0, p0, gone):
    want, tol, pos = w0.cpu().double(), torch.zeros(w0.shape, dtype=torch.float64), p0.cpu()
    for r, (nq, nk) in enumerate(zip(q_lens, k_lens)):
        if nq == 0 or nk == 0:
            continue
        blk, off = pg.places(r, nk)
        old = w0.cpu()[blk, :, off].T
        w, e = ref.key_weights(q[start[r]:start[r] + nq], pg.keys[r][:nk].cuda(), lse[:, start[r]:start[r] + nq], old.cuda(), scale)
        want[blk, :, off], tol[blk, :, off] = w.T.cpu(), e.T.cpu()
        first = max(0, nk - nq)
        pos[blk[first:], :, off[first:]] = (torch.arange(first, nk) + gone[r]).int()[:, None].expand(-1, pg.KVH)
    got = stats.weights.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    err = torch.where(want.isnan(), 0.0, (got - want).abs())
    assert bool((err <= torch.where(tol.isnan(), math.inf, tol)).all()), (float((err - tol).max()), float(err.max()))
    assert torch.equal(stats.positions.cpu(), pos)


@pytest.mark.parametrize("layout", ["interleaved", "tokens", "heads"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_weights_ragged(dtype, layout):
    _weights_case([1, 5, 0, 3, 2, 1], [1, 300, 40, 3, 129, 128], 8, 2, 64, 16, dtype, layout=layout, gap=3)


@pytest.mark.parametrize("D,BS,H,KVH", [(64, 16, 4, 4), (128, 16, 32, 8), (80, 24, 20, 4), (96, 8, 6, 2), (128, 64, 8, 1), (16, 16, 4, 2),
                                        (256, 16, 4, 2), (128, 1, 4, 2), (72, 5, 12, 4), (128, 128, 64, 1), (64, 32, 32, 1), (112, 48, 3, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_shapes(dtype, D, BS, H, KVH):
    _weights_case([1, 40, 7], [200, 77, 600], H, KVH, D, BS, dtype, seed=D + BS)
    _weights_case([1, 1, 1], [513, 1, 128], H, KVH, D, BS, dtype, seed=D + BS + 1)


@pytest.mark.parametrize("D,BS,H,KVH", [(64, 16, 8, 8), (128, 24, 8, 2), (256, 16, 2, 1), (4, 3, 4, 1)])
def test_weights_fp32(D, BS, H, KVH):
    _weights_case([1, 70, 7], [200, 77, 300], H, KVH, D, BS, torch.float32, seed=D)


@pytest.mark.parametrize("q_lens,k_lens", [([1], [1]), ([1], [20000]), ([700], [700]), ([300, 2, 900], [5000, 2, 901]), ([64], [64]),
                                           ([257, 31, 32, 33], [1000, 31, 64, 3000]), ([1] * 300, list(range(1, 301))),
                                           ([9, 9], [5, 1]), ([1, 200], [0, 0]), ([2000], [4096])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_lengths(dtype, q_lens, k_lens):
    if dtype == torch.float32 and max(k_lens) > 6000:
        k_lens = [min(k, 6000) for k in k_lens]
    _weights_case(q_lens, k_lens, 8, 2, 128 if dtype == torch.bfloat16 else 64, 16, dtype, seed=len(q_lens))


@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (100000, 100000), (1, 0), (0, 1)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_weights_hints_change_only_the_time(dtype, hints):
    _weights_case([3, 150, 1], [600, 150, 90], 8, 2, 64, 16, dtype, host=0.3, hints=hints)


@pytest.mark.parametrize("host", [0.2, 1.0])
@pytest.mark.parametrize("dtype,D,BS", [(torch.bfloat16, 128, 16), (torch.float16, 64, 24), (torch.float32, 64, 16)])
def test_weights_of_host_blocks(dtype, D, BS, host):
    _weights_case([1, 30, 5], [400, 333, 50], 8, 2, D, BS, dtype, host=host, evicted=False)


@pytest.mark.parametrize("dtype,ql", [(torch.bfloat16, 3), (torch.bfloat16, 200), (torch.float32, 100)])
def test_weights_of_rows_without_keys_and_nan(dtype, ql):
    """lse = -inf or +inf gives nothing, a NaN spoils the keys that its row sees and no other."""
    pg = Paged([400, 300], 2, 16, 64, dtype, seed=3)
    T, H, scale = 2 * ql, 4, 0.125
    q = torch.randn(T, H, 64, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    lse = _lse(q, pg.keys, [ql, ql], scale)
    lse[0, 1], lse[1, 2], lse[2, ql] = -math.inf, math.inf, NAN
    stats = pg.stats()
    w0, p0 = stats.weights.clone(), stats.positions.clone()
    gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, i32([0, ql]), i32([ql, ql]), i32([400, 300]), scale, lse, stats,
                        max_q_len=ql, max_k_len=400)
    ok()
    _check_weights(pg, q, lse, [ql, ql], [400, 300], [0, ql], scale, stats, w0, p0, [0, 0])
    assert int(stats.weights.isnan().sum()) == 300 - ql + 1


@pytest.mark.parametrize("dtype,H,ql", [(torch.bfloat16, 8, 3), (torch.float16, 8, 7), (torch.bfloat16, 8, 90), (torch.float16, 20, 200),
                                        (torch.float32, 8, 70)])
def test_weights_of_infinite_rows_whatever_their_queries_hold(dtype, H, ql):
    """A row with lse = -inf or +inf gives nothing where its scores are NaN, infinite or overflow, too."""
    k_lens, KVH, D, scale = [700, 300, 513], 2, 64, 0.125
    pg = Paged(k_lens, KVH, 16, D, dtype, seed=13)
    T = 3 * ql
    q = torch.randn(T, H, D, generator=torch.Generator().manual_seed(12)).to(dtype).cuda()
    lse = _lse(q, pg.keys, [ql] * 3, scale)
    big = torch.finfo(dtype).max
    at = 0
    for out in (-math.inf, math.inf):
        for fill in (NAN, math.inf, -math.inf, big, -big):  # one row of some token and head each, and two whole tokens
            t, h = (7 * at + 1) % T, (3 * at) % H
            lse[h, t], q[t, h] = out, fill
            at += 1
        t = 0 if out < 0 else T - 1
        lse[:, t], q[t] = out, NAN
    stats = pg.stats()
    w0, p0 = stats.weights.clone(), stats.positions.clone()
    gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, i32([0, ql, 2 * ql]), i32([ql] * 3), i32(k_lens), scale, lse, stats,
                        max_q_len=ql, max_k_len=700)
    ok()
    assert not bool(torch.cat([stats.weights[pg.places(r)[0].cuda(), :, pg.places(r)[1].cuda()] for r in range(3)]).isnan().any())
    _check_weights(pg, q, lse, [ql] * 3, k_lens, [0, ql, 2 * ql], scale, stats, w0, p0, [0, 0, 0])


@pytest.mark.parametrize("dtype,ql", [(torch.bfloat16, 3), (torch.float16, 7), (torch.bfloat16, 90), (torch.float32, 70)])
def test_weights_of_keys_with_an_infinite_value(dtype, ql):
    """A key whose scores are +inf makes its rows' lse +inf: they give nothing; to those that it scores -inf it is nothing."""
    k_lens, KVH, H, D, scale = [700, 300], 2, 8, 64, 0.125
    pg = Paged(k_lens, KVH, 16, D, dtype, seed=14)
    for r, j in ((0, 5), (0, 300), (1, 299)):
        blk, off = pg.rows[r][j // 16], j % 16
        pg.tiers[0].k[blk, 1, off, 3] = pg.keys[r][j, 1, 3] = math.inf
    q = torch.randn(2 * ql, H, D, generator=torch.Generator().manual_seed(15)).to(dtype)
    q[..., 3] = torch.where(q[..., 3] == 0, 1.0, q[..., 3])
    q = q.cuda()
    lse = _lse(q, pg.keys, [ql] * 2, scale)
    assert 0 < int(lse.isinf().sum()) < lse.numel() and not bool(lse.isnan().any())
    stats = pg.stats()
    w0, p0 = stats.weights.clone(), stats.positions.clone()
    gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, i32([0, ql]), i32([ql] * 2), i32(k_lens), scale, lse, stats, max_q_len=ql, max_k_len=700)
    ok()
    _check_weights(pg, q, lse, [ql] * 2, k_lens, [0, ql], scale, stats, w0, p0, [0, 0])
    assert not bool(torch.cat([stats.weights[pg.places(r)[0].cuda(), :, pg.places(r)[1].cuda()] for r in range(2)]).isnan().any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_strides_and_table_rows(dtype):
    """q out of a wider projection, lse [T, H] transposed, requests on other table rows."""
    pg = Paged([200, 333, 90], 2, 16, 64, dtype, seed=5)
    q_lens, rows, H = [4, 50], [2, 1], 4
    g = torch.Generator().manual_seed(4)
    q = torch.randn(54 + 6, 3 * H, 64, generator=g).to(dtype).cuda()[6:, H:2 * H]
    keys = [pg.keys[r] for r in rows]
    lse = _lse(q, keys, q_lens, 0.125).T.contiguous().T
    assert lse.stride(0) == 1
    stats = pg.stats()
    w0, p0 = stats.weights.clone(), stats.positions.clone()
    gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, i32([0, 4]), i32(q_lens), i32([90, 333]), 0.125, lse, stats, bt_row=i32(rows),
                        max_q_len=50, max_k_len=333)
    ok()
    pg.rows, pg.lens, pg.keys = [pg.rows[r] for r in rows], [90, 333], keys
    _check_weights(pg, q, lse, q_lens, [90, 333], [0, 4], 0.125, stats, w0, p0, [0, 0])


@pytest.mark.parametrize("dtype,ql", [(torch.float16, 2), (torch.float16, 90), (torch.float32, 2)])
def test_weights_refuse_bad_requests_alone(dtype, ql):
    def call(k_len, start, table_edit=None, nstat=None, bt_row=None):
        pg = Paged([100, 200, 300], 2, 16, 64, dtype, seed=6)
        q = torch.randn(3 * ql, 4, 64, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
        lse = _lse(q, pg.keys, [ql] * 3, 0.125)
        stats = pg.stats()
        if nstat is not None:
            stats = KeyStats(stats.weights[:nstat].clone(), stats.positions[:nstat].clone())
        w0 = stats.weights.clone()
        if table_edit is not None:
            pg.table[table_edit[0], table_edit[1]] = table_edit[2]
        gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, i32(start), i32([ql] * 3), i32(k_len), 0.125, lse, stats,
                            bt_row=bt_row, max_q_len=ql, max_k_len=300)
        return pg, stats, w0

    for k_len, start, bt_row in (([100, 5000, 300], [0, ql, 2 * ql], None), ([100, 200, 300], [0, 2 * ql + 1, 2 * ql], None),
                                 ([100, -1, 300], [0, ql, 2 * ql], None), ([100, 200, 300], [0, ql, 2 * ql], [0, 9, 2])):
        pg, stats, w0 = call(k_len, start, bt_row=None if bt_row is None else i32(bt_row))
        fails("sequence length")
        for r, changed in ((0, True), (1, False), (2, True)):
            blk, off = pg.places(r)
            assert torch.equal(stats.weights.cpu()[blk, :, off], w0.cpu()[blk, :, off]) != changed
    for bad in (-1, 1 << 20):
        pg, stats, w0 = call([100, 200, 300], [0, ql, 2 * ql], (1, 3, bad))
        fails("block id")
        blk, off = pg.places(2)
        assert not torch.equal(stats.weights.cpu()[blk, :, off], w0.cpu()[blk, :, off])
    pg, stats, w0 = call([100, 200, 300], [0, ql, 2 * ql], nstat=10)  # blocks behind the stats
    fails("block id")


def test_weights_of_chunks_add_up_to_the_prompt_s():
    """A prompt in chunks gives each key what the prompt as a whole gives it."""
    n, cuts, H, KVH, D = 500, [200, 250, 251, 500], 8, 2, 128
    pg = Paged([n], KVH, 16, D, torch.bfloat16, seed=8)
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    lse = _lse(q, pg.keys, [n], D ** -0.5)
    a, b = pg.stats(2), pg.stats(3)
    gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, i32([0]), i32([n]), i32([n]), D ** -0.5, lse, a)
    at = 0
    for c in cuts:
        gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, i32([at]), i32([c - at]), i32([c]), D ** -0.5, lse, b)
        at = c
    ok()
    blk, off = pg.places(0)
    wa, wb = a.weights.cpu()[blk, :, off], b.weights.cpu()[blk, :, off]
    # the same terms, summed in another order: n G roundings each
    assert bool(((wa - wb).abs() <= 2 * (n * 4 + 64) * 2.0 ** -24 * wa).all())
    # every query spreads a weight of 1 per head: off by its exponents' errors, 2^-12 at |s| below 2^6
    assert abs(float(wa.double().sum()) / (n * H) - 1) <= 2.0 ** -12
    assert torch.equal(a.positions.cpu()[blk, :, off], b.positions.cpu()[blk, :, off])


# ------------------------------------------------------------------ select


def _select(lens, keep, KVH=2, BS=16, sinks=0, recent=0, gone=None, seed=0, room=None, hint=None, weights=None, gaps=True):
    pg = Paged(lens, KVH, BS, 8, torch.float32, seed=seed)
    stats = pg.stats()
    g = torch.Generator().manual_seed(seed + 1)
    gone = [3 * r for r in range(len(lens))] if gone is None else gone
    w_l, p_l = [], []
    for r, n in enumerate(lens):
        w = torch.randn(KVH, n, generator=g).exp() if weights is None else weights(KVH, n, g)
        p = torch.stack([torch.randperm(n + gone[r], generator=g)[:n].int() for _ in range(KVH)]) if n else torch.zeros(KVH, 0)
        blk, off = pg.places(r)
        stats.weights[blk.cuda(), :, off.cuda()] = w.T.cuda()
        stats.positions[blk.cuda(), :, off.cuda()] = p.T.int().cuda()
        w_l.append(w)
        p_l.append(p)
    room = max([1] + [min(b, n - b) for n, b in zip(lens, keep) if 0 <= b < n]) if room is None else room
    m = KeyMoves(len(lens), KVH, room, dev())
    m.src.fill_(-5)
    m.dst.fill_(-6)
    gpu_ops.select_keys(stats, pg.table, i32(lens), i32(keep), m, sinks=sinks, recent=recent, evicted=i32(gone),
                        max_k_len=max(lens) if hint is None else hint)
    return pg, stats, m, w_l, p_l, gone


def _check_select(m, lens, keep, w_l, p_l, gone, sinks, recent, skip=()):
    src, dst, counts = m.src.tolist(), m.dst.tolist(), m.counts.tolist()
    for r, n in enumerate(lens):
        for h in range(m.KVH):
            a, b = ([], []) if r in skip else ref.select(w_l[r][h].tolist(), p_l[r][h].tolist(), n, keep[r], gone[r], sinks, recent)
            assert counts[r][h] == len(a) == len(b), (r, h)
            assert src[r][h] == a + [-5] * (m.room - len(a)) and dst[r][h] == b + [-6] * (m.room - len(b)), (r, h)


@pytest.mark.parametrize("sinks,recent", [(0, 0), (4, 0), (0, 40), (4, 16), (1000, 0), (0, 100000)])
def test_select_ragged(sinks, recent):
    lens = [1, 2, 50, 200, 0, 333, 1000, 64]
    keep = [0, 1, 20, 200, 0, 332, 100, -1]
    _, _, m, w, p, gone = _select(lens, keep, sinks=sinks, recent=recent)
    ok()
    _check_select(m, lens, keep, w, p, gone, sinks, recent)


@pytest.mark.parametrize("BS,KVH", [(1, 1), (5, 3), (64, 8), (24, 2)])
def test_select_blocks_and_heads(BS, KVH):
    lens, keep = [77, 500, 129], [33, 499, 64]
    _, _, m, w, p, gone = _select(lens, keep, KVH, BS, 2, 10, seed=BS)
    ok()
    _check_select(m, lens, keep, w, p, gone, 2, 10)


def _ties(KVH, n, g):
    return torch.randint(0, 3, (KVH, n), generator=g).float() * torch.where(torch.rand(KVH, n, generator=g) < 0.5, -1.0, 1.0)


def _odd(KVH, n, g):
    v = torch.tensor([NAN, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42, 3e38, 1.0, -NAN])
    return v[torch.randint(0, len(v), (KVH, n), generator=g)]


@pytest.mark.parametrize("weights", [_ties, _odd, lambda K, n, g: torch.zeros(K, n), lambda K, n, g: torch.full((K, n), NAN)])
def test_select_ties_go_to_the_lowest_index(weights):
    lens, keep = [300, 1025, 40], [100, 512, 39]
    _, _, m, w, p, gone = _select(lens, keep, 2, 16, 3, 9, seed=4, weights=weights)
    ok()
    _check_select(m, lens, keep, w, p, gone, 3, 9)


@pytest.mark.parametrize("n,keep,KVH,hint", [(20000, 2048, 2, None), (70000, 30000, 1, None), (70000, 69000, 1, 100), (100000, 5, 1, 0),
                                             (9000, 8999, 3, 1 << 30)])
def test_select_long(n, keep, KVH, hint):
    """Several CTAs, keys beyond a CTA's shared memory (a hint that is too small), exact order against a stable sort."""
    _, stats, m, w, p, gone = _select([n, 5], [keep, 5], KVH, 16, 4, keep // 3, seed=n, hint=hint)
    ok()
    for h in range(KVH):
        guard = (p[0][h] < 4) | (p[0][h] >= n + gone[0] - keep // 3)
        score = torch.where(guard, math.inf, w[0][h].double())
        order = torch.sort(score, descending=True, stable=True)[1]
        stays = torch.zeros(n, dtype=torch.bool)
        stays[order[:keep]] = True
        a, b = stays[keep:].nonzero().flatten() + keep, (~stays[:keep]).nonzero().flatten()
        c = int(m.counts[0, h])
        assert c == len(a) and m.src[0, h, :c].tolist() == a.tolist() and m.dst[0, h, :c].tolist() == b.tolist()
        assert int(m.counts[1, h]) == 0


def test_select_refuses_bad_requests_alone():
    lens, keep = [100, 90, 80], [50, 45, 40]
    _, _, m, w, p, gone = _select(lens, keep, room=45)
    fails("sequence length")
    _check_select(m, lens, keep, w, p, gone, 0, 0, skip=(0,))
    for n in (-1, 10000):
        pg, stats, m, w, p, gone = _select(lens, keep)
        ok()
        m.src.fill_(-5), m.dst.fill_(-6)
        gpu_ops.select_keys(stats, pg.table, i32([100, n, 80]), i32(keep), m, evicted=i32(gone), max_k_len=100)
        fails("sequence length")
        _check_select(m, lens, keep, w, p, gone, 0, 0, skip=(1,))
    for bad in (-1, 1 << 20):
        pg, stats, m, w, p, gone = _select(lens, keep)
        ok()
        m.src.fill_(-5), m.dst.fill_(-6)
        pg.table[1, 4] = bad
        gpu_ops.select_keys(stats, pg.table, i32(lens), i32(keep), m, evicted=i32(gone), max_k_len=100)
        fails("block id")
        _check_select(m, lens, keep, w, p, gone, 0, 0, skip=(1,))


def test_select_refuses_a_bad_block_in_a_cluster():
    pg, stats, m, w, p, gone = _select([40000], [1000], KVH=1, seed=2)
    ok()
    m.src.fill_(-5)
    pg.table[0, 2400] = -1
    gpu_ops.select_keys(stats, pg.table, i32([40000]), i32([1000]), m, evicted=i32(gone), max_k_len=40000)
    fails("block id")
    assert m.counts.tolist() == [[0]] and bool((m.src == -5).all())


def test_select_in_clusters_again_and_again():
    """Many calls on two streams, each request on a cluster of CTAs that write to one another's counters: the same lists every time."""
    lens, keep = [33000, 20000, 30000], [500, 19000, 3000]
    sides = []
    for _ in range(2):
        pg, stats, m, _, _, gone = _select(lens, keep, KVH=4, seed=9, recent=100)
        ok()
        sides.append((torch.cuda.Stream(), stats, pg.table, i32(lens), i32(keep), m, i32(gone)))
    torch.cuda.synchronize()
    want = [sides[0][5].src.clone(), sides[0][5].dst.clone(), sides[0][5].counts.clone()]
    wrong = torch.zeros(2, dtype=torch.int64, device="cuda")
    for _ in range(300):
        for i, (stream, stats, table, ln, kp, m, gone) in enumerate(sides):
            with torch.cuda.stream(stream):
                gpu_ops.select_keys(stats, table, ln, kp, m, recent=100, evicted=gone, max_k_len=33000)
                for x, y in zip((m.src, m.dst, m.counts), want):
                    wrong[i] += (x != y).any()
    torch.cuda.synchronize()
    ok()
    assert wrong.tolist() == [0, 0]


# ------------------------------------------------------------------ move


@pytest.mark.parametrize("layout", ["interleaved", "tokens", "heads"])
@pytest.mark.parametrize("dtype,D,BS,host", [(torch.bfloat16, 128, 16, 0.0), (torch.float16, 64, 24, 0.4), (torch.float32, 4, 5, 0.5),
                                             (torch.bfloat16, 8, 16, 1.0), (torch.float32, 256, 64, 0.0)])
def test_move_selected_keys(dtype, D, BS, host, layout):
    """After select and move the first keys of every request are those that stay, with their weights and positions."""
    lens, keep, KVH = [500, 33, 70, 1, 200], [200, 20, 69, 1, 0], 3
    pg = Paged(lens, KVH, BS, D, dtype, host, seed=D, layout=layout)
    stats = pg.stats()
    w0, p0 = stats.weights.cpu(), stats.positions.cpu()
    k0, v0 = pg.now()
    m = gpu_ops.select_keys(stats, pg.table, i32(lens), i32(keep), KeyMoves(5, KVH, 200, dev()), recent=5)
    gpu_ops.move_keys(m, pg.tiers, pg.G, pg.table, stats)
    ok()
    k1, v1 = pg.now()
    w1, p1 = stats.weights.cpu(), stats.positions.cpu()
    for r, n in enumerate(lens):
        blk, off = pg.places(r)
        for h in range(KVH):
            c = int(m.counts[r, h])
            a, b = m.src[r, h, :c].cpu().long(), m.dst[r, h, :c].cpu().long()
            at = torch.arange(n)
            at[b] = a
            for x0, x1 in ((k0, k1), (v0, v1), (w0, w1), (p0, p1)):
                want = x0[blk, h, off][at]
                assert torch.equal(x1[blk, h, off], want), (r, h)
                x0[blk, h, off] = want
    for x0, x1 in ((k0, k1), (v0, v1), (w0, w1), (p0, p1)):  # nothing else changed
        assert torch.equal(x0.nan_to_num(123.0) if x0.is_floating_point() else x0, x1.nan_to_num(123.0) if x1.is_floating_point() else x1)


def test_move_without_stats_and_many_small_units():
    lens = [40] * 300
    pg = Paged(lens, 1, 16, 64, torch.bfloat16, seed=1)
    k0, v0 = pg.now()
    src = torch.arange(20, 30, dtype=torch.int32).repeat(300, 1, 1).cuda()
    dst = torch.arange(0, 20, 2, dtype=torch.int32).repeat(300, 1, 1).cuda()
    gpu_ops.move_keys(KeyMoves(300, 1, 10, dev(), src=src, dst=dst, counts=i32([[10]] * 300)), pg.tiers, pg.G, pg.table)
    ok()
    k1, v1 = pg.now()
    for r in range(300):
        blk, off = pg.places(r)
        at = torch.arange(40)
        at[0:20:2] = torch.arange(20, 30)
        assert torch.equal(k1[blk, 0, off], k0[blk, 0, off][at]) and torch.equal(v1[blk, 0, off], v0[blk, 0, off][at])


def test_move_passes_over_bad_pairs():
    pg = Paged([60, 60], 1, 16, 64, torch.float16, seed=2)
    k0, v0 = pg.now()
    W = pg.table.shape[1] * 16
    m = KeyMoves(2, 1, 4, dev(), src=i32([[[30, W, -1, 33]], [[30, 31, 32, 33]]]), dst=i32([[[0, 1, 2, 3]], [[0, 1, 2, 3]]]),
                 counts=i32([[4], [5]]))
    gpu_ops.move_keys(m, pg.tiers, pg.G, pg.table)
    fails("sequence length")
    k1, _ = pg.now()
    blk, off = pg.places(0)
    at = torch.arange(60)
    at[0], at[3] = 30, 33
    assert torch.equal(k1[blk, 0, off], k0[blk, 0, off][at])
    blk, off = pg.places(1)  # a count beyond the room: nothing
    assert torch.equal(k1[blk, 0, off], k0[blk, 0, off])
    m.counts.copy_(i32([[0], [4]]))
    pg.table[1, 0] = 1 << 20
    gpu_ops.move_keys(m, pg.tiers, pg.G, pg.table)
    fails("block id")
    assert torch.equal(pg.now()[0][blk, 0, off], k0[blk, 0, off])


# ------------------------------------------------------------------ trim


def _trim(lens, keep, block, share, seed=0, slack=4, cap=None):
    rnd = random.Random(seed)
    held = [-(-max(0, n) // block) for n in lens]
    total = sum(held) + slack
    hbm = max(1, int(total * share))
    ids = list(range(total))
    rnd.shuffle(ids)
    W = max(held + [1]) + 1
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-3] * (W - h))
        at += h
    s0, s1 = [b for b in ids[at:] if b < hbm], [b for b in ids[at:] if b >= hbm]
    cap = total if cap is None else cap
    return table, [s0 + [-1] * (cap - len(s0)), s1 + [-1] * (cap - len(s1))], [len(s0), len(s1)], hbm, total - hbm


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("hint", [0, 1])
@pytest.mark.parametrize("R,block,hi,cut,share", [(1, 16, 5, 9, 1.0), (3, 1, 40, 50, 0.5), (40, 24, 500, 300, 0.3), (256, 16, 900, 7, 0.7),
                                                  (1000, 16, 700, 700, 0.5), (8192, 8, 60, 60, 0.5), (4, 16, 200000, 200000, 0.6),
                                                  (1025, 64, 100, 100, 0.0), (600, 1, 300, 300, 0.5)])
def test_trim_matches_lists(R, block, hi, cut, share, hint, in_place):
    rnd = random.Random(R + block)
    lens = [rnd.randint(0, hi) for _ in range(R)]
    keep = [rnd.choice([-1, n + rnd.randint(0, 5), max(0, n - rnd.randint(0, cut))]) for n in lens]
    table, stacks, counts, hbm, host = _trim(lens, keep, block, share, R)
    w_stacks, w_counts, left = ref.trim(keep, lens, table, stacks, counts, hbm, block)
    tt, st, ct, ln, gone = i32(table), i32(stacks), i32(counts), i32(lens), i32([5] * R)
    out = TrimTables(R, dev(), seq_lens=ln if in_place else None, counts=ct if in_place else None)
    gpu_ops.trim_tables(i32(keep), ln, tt, FreeBlocks(st[0], st[1], ct), hbm, host, block, out, evicted=gone, max_cut=hint)
    ok()
    h = out.read_header()
    assert out.seq_lens.tolist() == left and out.counts.tolist() == w_counts
    assert st.tolist() == w_stacks and tt.tolist() == table
    assert gone.tolist() == [5 + n - b for n, b in zip(lens, left)]
    assert (h["freed_hbm"], h["freed_host"], h["max_seq"]) == (w_counts[0] - counts[0], w_counts[1] - counts[1], max(left))
    assert h["n_tok"] == h["taken_hbm"] == h["taken_host"] == h["max_new"] == 0


@pytest.mark.parametrize("R", [3, 900])
@pytest.mark.parametrize("why,flag", [("len", "bad length"), ("long", "bad length"), ("block", "bad block id"), ("count", "bad free stack"),
                                      ("room", "bad free stack")])
def test_refused_trims_change_nothing(R, why, flag):
    lens, keep = [50] * R, [20] * R
    table, stacks, counts, hbm, host = _trim(lens, keep, 16, 0.5, 1)
    if why == "room":
        stacks = [s[:c + 1] for s, c in zip(stacks, counts)]
        stacks = [s + [0] * (max(map(len, stacks)) - len(s)) for s in stacks]
    if why == "block":
        table[R - 1][3] = hbm + host
    if why == "count":
        counts[1] = -1
    if why == "len":
        lens[R // 2] = -1
    if why == "long":
        lens[R // 2] = 5 * 16 + 1
    tt, st, ct, ln, gone = i32(table), i32(stacks), i32(counts), i32(lens), i32([5] * R)
    out = TrimTables(R, dev())
    gpu_ops.trim_tables(i32(keep), ln, tt, FreeBlocks(st[0], st[1], ct), hbm, host, 16, out, evicted=gone)
    fails("block tables")
    with pytest.raises(RuntimeError, match="trim_tables refused the step: " + flag):
        out.read_header()
    assert out.seq_lens.tolist() == lens and out.counts.tolist() == counts and st.tolist() == stacks
    assert tt.tolist() == table and gone.tolist() == [5] * R


def test_trim_of_no_requests():
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = gpu_ops.trim_tables(e, e, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), FreeBlocks(e, None, i32([0, 0])), 4, 0, 16)
    ok()
    assert out.read_header()["freed_hbm"] == 0 and out.counts.tolist() == [0, 0]


def test_extend_tables_positions_run_ahead_of_evicted_tokens():
    """Positions are index plus evicted, for each way of placing tokens; an ended request's count becomes 0."""
    for new in ([1, 3, -1, 0, 4], [1, 9, -1, 0, 40], [1, 5000, -1, 0, 4000]):
        prior, gone = [5, 16, 20, 7, 0], [100, 0, 9, 3, 50]
        need = [0 if n < 0 else -(-(p + n) // 16) for p, n in zip(prior, new)]
        W, at, table = max(need) + 2, 0, []
        for p in prior:
            h = -(-p // 16)
            table.append(list(range(at, at + h)) + [0] * (W - h))
            at += h
        free = list(range(at, at + sum(need)))
        tt, g = i32(table), i32(gone)
        t = StepTables(5, sum(max(0, n) for n in new) + 3, dev())
        plain = StepTables(5, t.T, dev())
        stack = i32(free)
        for out, ev, tab in ((plain, None, tt.clone()), (t, g, tt)):
            pool = FreeBlocks(torch.cat([stack, i32([-1] * 9)]), None, i32([len(free), 0]))
            gpu_ops.extend_tables(i32(new), i32(prior), tab, pool, 10 ** 6, 0, 16, out, evicted=ev)
        ok()
        assert torch.equal(t.slot_mapping, plain.slot_mapping)
        want = [p + gone[r] + i for r, (p, n) in enumerate(zip(prior, new)) for i in range(max(0, n))]
        assert t.positions.tolist() == want + [0] * 3
        assert g.tolist() == [100, 0, 0, 3, 50]


# ------------------------------------------------------------------ verify


def _probs(g, *shape, dtype=torch.float32, spread=2.0):
    return (torch.randn(*shape, generator=g) * spread).softmax(-1).to(dtype)


def _verify(target, tokens, draft, start, q_len, au, su, seq=None, out=None):
    v = gpu_ops.verify_drafts(target.cuda(), tokens.cuda(), None if draft is None else draft.cuda(), i32(start), i32(q_len), au.cuda(),
                              su.cuda(), seq_lens=None if seq is None else i32(seq), out=out)
    return v


def _check_verify(v, target, tokens, draft, start, q_len, au, su, seq=None):
    K = tokens.shape[1]
    t64 = target.double().tolist()
    for r in range(len(q_len)):
        got, a = ref.verify(t64, tokens[r].tolist(), None if draft is None else draft[r].double().tolist(), start[r], q_len[r],
                            au[r].double().tolist(), float(su[r]))
        assert v.tokens[r].tolist() == got + [-1] * (K + 1 - len(got)), r
        assert int(v.accepted[r]) == a
        if seq is not None:
            assert int(v.keep_lens[r]) == seq[r] - (max(0, q_len[r] - 1) - a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,K,R", [(1, 1, 2), (2, 3, 5), (100, 4, 9), (1003, 3, 6), (5000, 2, 4), (33001, 1, 3), (32768, 2, 2)])
@pytest.mark.parametrize("with_draft", [True, False])
def test_verify(V, K, R, dtype, with_draft):
    g = torch.Generator().manual_seed(V + K)
    q_len = [min(K + 1, max(0, r % (K + 2))) for r in range(R - 1)] + [K + 1]
    start = [sum(q_len[:r]) for r in range(R)]
    target = _probs(g, sum(q_len), V, dtype=dtype)
    draft = _probs(g, R, K, V, dtype=dtype)
    for r in range(R):  # drafts near the target, so that some are accepted
        for d in range(max(0, q_len[r] - 1)):
            draft[r, d] = (0.7 * target[start[r] + d].float() + 0.3 * draft[r, d].float()).to(dtype)
    tokens = torch.stack([torch.multinomial(draft[r].float(), 1, generator=g).flatten() for r in range(R)])
    au, su = torch.rand(R, K, generator=g), torch.rand(R, generator=g)
    seq = [50 + r for r in range(R)]
    v = _verify(target, tokens, draft if with_draft else None, start, q_len, au, su, seq)
    ok()
    _check_verify(v, target, tokens, draft if with_draft else None, start, q_len, au, su, seq)


def test_verify_more_drafts_than_a_warp_and_no_drafts():
    g = torch.Generator().manual_seed(3)
    for K, q_len in ((70, [71, 40, 33, 32, 1, 0]), (0, [1, 1, 0, 1])):
        R, V = len(q_len), 64
        start = [sum(q_len[:r]) for r in range(R)]
        target, draft = _probs(g, sum(q_len), V, spread=0.1), _probs(g, R, K, V, spread=0.1)
        tokens = torch.randint(0, V, (R, K), generator=g)
        au, su = torch.rand(R, K, generator=g) * 0.9, torch.rand(R, generator=g)
        if K:
            au[0], au[1, 36] = 0.0, 0.999999
        v = _verify(target, tokens, draft, start, q_len, au, su)
        ok()
        _check_verify(v, target, tokens, draft, start, q_len, au, su)
        if K:
            assert int(v.accepted[0]) == 70


def test_verify_greedy_rows_and_extreme_numbers():
    """One-hot rows accept their token alone and are drawn for any number; numbers of 0, almost 1, 1, NaN."""
    V = 5000
    hot = torch.zeros(3, V)
    hot[0, 4999] = hot[1, 17] = hot[2, 0] = 1.0
    tokens = torch.tensor([[4999, 17], [4999, 3], [5, 17]])
    for u in (0.0, 1.0 - 2.0 ** -24, 1.0, NAN, -1.0):
        target = hot.repeat(3, 1)
        au, su = torch.full((3, 2), min(max(u, 0.0), 1 - 2 ** -24) if u == u else 0.0), torch.full((3,), u)
        v = _verify(target, tokens, None, [0, 3, 6], [3] * 3, au, su)
        ok()
        assert v.tokens.tolist() == [[4999, 17, 0], [4999, 17, -1], [4999, -1, -1]]
    g = torch.Generator().manual_seed(1)
    target = _probs(g, 4, 777)
    target[:, 700:] = 0.0
    target[:, :30] = 0.0
    for u in (0.0, 1.0 - 2.0 ** -24, 1.0, NAN):
        su = torch.full((4,), u)
        e = torch.zeros(4, 0)
        v = _verify(target, e.long(), None, [0, 1, 2, 3], [1] * 4, e, su)
        ok()
        _check_verify(v, target, e.long(), None, [0, 1, 2, 3], [1] * 4, e, su)
        assert v.tokens.flatten().tolist() == [30 if u != u or u == 0.0 else 699] * 4


def test_verify_odd_probabilities():
    """Negative, infinite and NaN values count as 0; a residual of nothing falls back to the target's row; a row of nothing gives -1."""
    g = torch.Generator().manual_seed(2)
    V = 300
    target, draft = _probs(g, 6, V), _probs(g, 3, 1, V)
    target[0, 5], target[1, 7], draft[0, 0, 9], draft[0, 0, 11] = NAN, math.inf, -3.0, NAN
    draft[1, 0] = target[2]          # p = q: nothing left where the draft is rejected all the same
    target[4] = 0.0                  # the third request's rejected draft: no probability at all
    tokens = torch.tensor([[5], [3], [8]])
    au, su = torch.tensor([[0.5], [1.0], [0.5]]), torch.tensor([0.3, 0.6, 0.2])
    v = _verify(target, tokens, draft, [0, 2, 4], [2, 2, 2], au, su)
    fails("without any positive")
    _check_verify(v, target, tokens, draft, [0, 2, 4], [2, 2, 2], au, su)
    assert v.tokens[2].tolist() == [-1, -1] and v.accepted.tolist() == [0, 0, 0]


def test_verify_refuses_bad_requests_alone():
    g = torch.Generator().manual_seed(5)
    target, draft = _probs(g, 9, 50), _probs(g, 3, 2, 50)
    tokens, au, su = torch.randint(0, 50, (3, 2), generator=g), torch.rand(3, 2, generator=g), torch.rand(3, generator=g)
    for start, q_len in (([0, 3, 6], [3, 4, 3]), ([0, 7, 6], [3, 3, 3]), ([0, -1, 6], [3, 3, 3]), ([0, 3, 6], [3, -1, 3])):
        v = _verify(target, tokens, draft, start, q_len, au, su, [20, 30, 40])
        fails("sequence length")
        assert v.tokens[1].tolist() == [-1] * 3 and int(v.accepted[1]) == 0 and int(v.keep_lens[1]) == 30
        for r in (0, 2):
            assert v.tokens[r].tolist()[0] >= 0
    for bad in (-1, 50, 1 << 40):
        t = tokens.clone()
        t[1, 0] = bad
        v = _verify(target, t, draft, [0, 3, 6], [3] * 3, au, su)
        fails("outside the vocabulary")
        assert int(v.accepted[1]) == 0
        _check_verify(v, target, t, draft, [0, 3, 6], [3] * 3, au, su)


def test_verify_strides():
    """Rows of a padded vocabulary, drafts stacked step by step, numbers out of wider tables."""
    g = torch.Generator().manual_seed(6)
    R, K, V = 5, 3, 999
    wide = torch.full((R * 4, 1024), 9.0)
    wide[:, :V] = _probs(g, R * 4, V)
    steps = _probs(g, K, R, V)
    toks = torch.randint(0, V, (R, 8), generator=g)
    au = torch.rand(R, 7, generator=g)
    start, q_len, su = [4 * r for r in range(R)], [4] * R, torch.rand(R, generator=g)
    wc, sc = wide.cuda(), steps.cuda()
    v = gpu_ops.verify_drafts(wc[:, :V], toks.cuda()[:, 2:5], sc.transpose(0, 1), i32(start), i32(q_len), au.cuda()[:, 1:4], su.cuda())
    ok()
    _check_verify(v, wide[:, :V], toks[:, 2:5], steps.transpose(0, 1), start, q_len, au[:, 1:4], su)


def test_verify_draws_by_the_probabilities():
    """The accepted and drawn first tokens of many requests follow the target, whatever the draft: 40000 draws over 8 tokens,
    each count within 5 standard deviations."""
    g = torch.Generator().manual_seed(7)
    R, V = 40000, 8
    p, q = _probs(g, V, spread=1.0), _probs(g, V, spread=1.0)
    tokens = torch.multinomial(q, R, replacement=True, generator=g).view(R, 1)
    v = _verify(p.expand(2 * R, V).contiguous(), tokens, q.expand(R, 1, V).contiguous(), [2 * r for r in range(R)], [2] * R,
                torch.rand(R, 1, generator=g), torch.rand(R, generator=g))
    ok()
    got = torch.bincount(v.tokens[:, 0].cpu(), minlength=V).double()
    assert bool(((got - R * p.double()).abs() <= 5 * (R * p * (1 - p)).double().sqrt()).all())


# ------------------------------------------------------------------ refusals that need a device's tensors


def test_calls_refuse_mismatched_tensors():
    pg = Paged([40, 50], 2, 16, 64, torch.float16, seed=1)
    stats, q = pg.stats(), torch.randn(2, 4, 64).half().cuda()
    lse, one = torch.zeros(4, 2, device="cuda"), i32([1, 1])

    def weights(**k):
        a = dict(q=q, tiers=pg.tiers, tier_split=pg.G, block_table=pg.table, q_start=i32([0, 1]), q_len=one, k_len=i32([40, 50]),
                 scale=0.125, lse=lse, stats=stats)
        a.update(k)
        gpu_ops.key_weights(**a)

    weights()
    ok()
    with pytest.raises(RuntimeError, match="lse"):
        weights(lse=lse.T)
    with pytest.raises(RuntimeError, match="lse"):
        weights(lse=lse.double())
    with pytest.raises(RuntimeError, match="q_len"):
        weights(q_len=one.long())
    with pytest.raises(RuntimeError, match="evicted"):
        weights(evicted=one[:1])
    with pytest.raises(RuntimeError, match="stats"):
        weights(stats=KeyStats.zeros(pg.G, 2, 8, dev()))
    with pytest.raises(RuntimeError, match="head size"):
        weights(q=q[..., :32])
    with pytest.raises(RuntimeError, match="workspace_buf"):
        weights(q=q.expand(2, 4, 64).repeat(1000, 1, 1), lse=torch.zeros(4, 2000, device="cuda"), max_q_len=0,
                workspace_buf=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    m = KeyMoves(2, 2, 30, dev())
    with pytest.raises(RuntimeError, match="keep_lens"):
        gpu_ops.select_keys(stats, pg.table, i32([40, 50]), i32([20]), m)
    with pytest.raises(RuntimeError, match="moves"):
        gpu_ops.select_keys(stats, pg.table, i32([40, 50]), i32([20, 20]), KeyMoves(1, 2, 30, dev()))
    with pytest.raises(RuntimeError, match="moves"):
        gpu_ops.move_keys(KeyMoves(2, 3, 30, dev()), pg.tiers, pg.G, pg.table)
    with pytest.raises(RuntimeError, match="at least one KV tier"):
        gpu_ops.move_keys(m, (None, None), pg.G, pg.table)
    with pytest.raises(RuntimeError, match="too small"):
        gpu_ops.trim_tables(i32([1, 1]), i32([40, 50]), pg.table, FreeBlocks(i32([0] * 9), None, i32([0, 0])), pg.G, 0, 16,
                            TrimTables(1, dev()))
    p, e = torch.rand(4, 10, device="cuda"), torch.zeros(2, 1, device="cuda")
    t, u = torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.zeros(2, device="cuda")
    for bad, match in (((p, t.int(), None, one, one, e, u), "draft_tokens"), ((p, t, torch.rand(2, 1, 11, device="cuda"), one, one, e, u), "draft_probs"),
                       ((p, t, torch.rand(2, 1, 10, device="cuda").half(), one, one, e, u), "draft_probs"),
                       ((p, t, None, one, one, e[:1], u), "accept_u"), ((p, t, None, one, one, e, u[:1]), "sample_u"),
                       ((p.T, t, None, one, one, e, u), "target_probs"), ((p, t, None, one[:1], one, e, u), "q_start")):
        with pytest.raises(RuntimeError, match=match):
            gpu_ops.verify_drafts(*bad)
    with pytest.raises(RuntimeError, match="DraftVerdict"):
        gpu_ops.verify_drafts(p, t, None, one, one, e, u, out=DraftVerdict(2, 2, dev()))


def test_default_buffers():
    """Calls without buffers of the caller's make their own."""
    lens, keep = [100, 90], [30, 90]
    _, stats, m, w, p, gone = _select(lens, keep)
    pg = Paged(lens, 2, 16, 8, torch.float32, seed=0)
    m2 = gpu_ops.select_keys(stats, pg.table, i32(lens), i32(keep), evicted=i32(gone), max_k_len=100)
    assert m2.room == 50 and torch.equal(m2.counts, m.counts)
    c = int(m.counts[0, 0])
    assert torch.equal(m2.src[0, 0, :c], m.src[0, 0, :c]) and torch.equal(m2.dst[0, 0, :c], m.dst[0, 0, :c])
    t = gpu_ops.trim_tables(i32(keep), i32(lens), pg.table, FreeBlocks(i32([0] * 20), None, i32([0, 0])), pg.G, 0, 16)
    assert t.seq_lens.tolist() == [30, 90] and t.counts.tolist() == [5, 0]
    ok()


# ------------------------------------------------------------------ places past 32 bits


def test_places_past_32_bits():
    """Block ids whose cache and stats offsets (in elements) pass 2^31."""
    KVH, BS, D = 8, 64, 128
    blocks = (1 << 31) // (KVH * BS * 2) + 7              # stats: [2^31 / 1024, 8, 64], cache: a view that strides far apart
    stats = KeyStats(torch.empty(2 * blocks, KVH, BS, device="cuda"), torch.empty(2 * blocks, KVH, BS, dtype=torch.int32, device="cuda"))
    few = 40
    far = (1 << 32) // (few - 1) // 8 * 8
    store = torch.empty(far * (few - 1) + KVH * BS * D, dtype=torch.bfloat16, device="cuda")
    k = store.as_strided((few, KVH, BS, D), (far, BS * D, D, 1))
    g = torch.Generator(device="cuda").manual_seed(1)
    k.copy_(torch.randn(few, KVH, BS, D, generator=g, device="cuda"))
    before = k.clone()
    top = 2 * blocks - few
    ids = [top + 37, top + 2, top + 39, top + 20]          # HBM ids: all below the split; the tier begins at id 0, so shift it
    base = KVTier(k, k)
    n, keep, H = 250, 100, 16
    q = torch.randn(3, H, D, generator=g, device="cuda").bfloat16()
    table = i32([[37, 2, 39, 20, 5]])
    keys = torch.cat([before[b].transpose(0, 1) for b in (37, 2, 39, 20)])[:n]
    lse = _lse(q, [keys], [3], D ** -0.5)
    stats.weights[:few].zero_()
    gpu_ops.key_weights(q, (base, None), few, table, i32([0]), i32([3]), i32([n]), D ** -0.5, lse, stats, max_q_len=3, max_k_len=n)
    ok()
    w, e = ref.key_weights(q, keys, lse, torch.zeros(KVH, n, device="cuda"), D ** -0.5)
    got = torch.stack([stats.weights[b] for b in (37, 2, 39, 20)], 1).flatten(1, 2)[:, :n].double()
    assert bool(((got - w).abs() <= e).all())
    # the same weights at the far end of the stats decide there
    for b, i in zip((37, 2, 39, 20), ids):
        stats.weights[i], stats.positions[i] = stats.weights[b], 5
    m = gpu_ops.select_keys(stats, i32([ids]), i32([n]), i32([keep]), KeyMoves(1, KVH, keep, dev()))
    ok()
    for h in range(KVH):
        a, b = ref.select(got[h].tolist(), [5] * n, n, keep, 0, 0, 0)
        c = int(m.counts[0, h])
        assert m.src[0, h, :c].tolist() == a and m.dst[0, h, :c].tolist() == b
    gpu_ops.move_keys(m, (base, None), few, table)
    ok()
    flat = lambda x, h: torch.cat([x[b, h] for b in (37, 2, 39, 20)])  # noqa: E731
    for h in range(KVH):
        c = int(m.counts[0, h])
        at = torch.arange(4 * BS, device="cuda")
        at[m.dst[0, h, :c].long()] = m.src[0, h, :c].long()
        assert torch.equal(flat(k, h), flat(before, h)[at])


# ------------------------------------------------------------------ streams and graphs


def _far_apart():
    """One call of each operator on buffers of its own; returns (call, results)."""
    pg = Paged([3000, 700], 4, 16, 128, torch.bfloat16, seed=21)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(800, 16, 128, generator=g).bfloat16().cuda()
    lse = _lse(q, pg.keys, [500, 300], 128 ** -0.5)
    stats = pg.stats(4)
    w0, p0 = stats.weights.clone(), stats.positions.clone()
    start, ql, kl, keep = i32([0, 500]), i32([500, 300]), i32([3000, 700]), i32([900, 100])
    m = KeyMoves(2, 4, 900, dev())
    st, ct = i32([[-1] * 300] * 2), i32([0, 0])
    tt = TrimTables(2, dev())
    tp, dp = _probs(g, 6, 5000).cuda(), _probs(g, 2, 2, 5000).cuda()
    toks, au, su = torch.randint(0, 5000, (2, 2), generator=g).cuda(), torch.rand(2, 2, generator=g).cuda(), torch.rand(2, generator=g).cuda()
    v = DraftVerdict(2, 2, dev())
    k0, v0 = pg.tiers[0].k.clone(), pg.tiers[0].v.clone()
    vs, vl = i32([0, 3]), i32([3, 3])

    def call():
        stats.weights.copy_(w0)
        stats.positions.copy_(p0)
        pg.tiers[0].k.copy_(k0)
        pg.tiers[0].v.copy_(v0)
        gpu_ops.key_weights(q, pg.tiers, pg.G, pg.table, start, ql, kl, 128 ** -0.5, lse, stats)
        gpu_ops.select_keys(stats, pg.table, kl, keep, m, recent=50)
        gpu_ops.move_keys(m, pg.tiers, pg.G, pg.table, stats)
        gpu_ops.trim_tables(keep, kl, pg.table, FreeBlocks(st[0], st[1], ct), pg.G, pg.C, 16, tt)
        gpu_ops.verify_drafts(tp, toks, dp, vs, vl, au, su, seq_lens=kl, out=v)

    return call, [stats.weights, stats.positions, pg.tiers[0].k, pg.tiers[0].v, m.src, m.dst, m.counts, st, tt.seq_lens, tt.counts, v.tokens,
                  v.accepted, v.keep_lens]


def _same(a, b):
    return all(torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x, y.view(torch.int16) if y.dtype == torch.bfloat16 else y)
               for x, y in zip(a, b))


def test_two_graphs_and_streams_do_not_share_anything():
    """Two captured graphs replayed on two streams at once, and eager calls on a third: all as the first eager call."""
    call, res = _far_apart()
    call()
    torch.cuda.synchronize()
    ok()
    want = [x.clone() for x in res]
    sides = []
    for _ in range(2):
        c, r = _far_apart()
        c()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c()
        sides.append((graph, r, torch.cuda.Stream()))
    third = torch.cuda.Stream()
    for _ in range(20):
        for graph, _, s in sides:
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(third):
            call()
    torch.cuda.synchronize()
    ok()
    assert _same(res, want) and all(_same(r, want) for _, r, _ in sides)


@pytest.mark.parametrize("keep", [1, 150, 299])
def test_select_s_bound_sizes_only_the_moves_that_it_makes(keep):
    """A bound that is too small: nothing, with moves given; a refusal where the call makes them itself."""
    lens = [300, 40]
    kept = [keep, 20]
    pg, stats, m, w, p, gone = _select(lens, kept, room=150, hint=10)
    ok()
    _check_select(m, lens, kept, w, p, gone, 0, 0)
    for bound in (0, 300):
        made = gpu_ops.select_keys(stats, pg.table, i32(lens), i32(kept), evicted=i32(gone), max_k_len=bound)
        ok()
        assert made.room >= 150 and made.counts.tolist() == m.counts.tolist()
        for r in range(2):
            for h in range(2):
                c = int(m.counts[r, h])
                assert torch.equal(made.src[r, h, :c], m.src[r, h, :c]) and torch.equal(made.dst[r, h, :c], m.dst[r, h, :c])
    small = gpu_ops.select_keys(stats, pg.table, i32(lens), i32(kept), evicted=i32(gone), max_k_len=40)
    if min(keep, 300 - keep) > 20:
        fails("sequence length")
        assert small.counts[0].tolist() == [0, 0]
    else:
        ok()
        assert small.counts[0].tolist() == m.counts[0].tolist()
    assert small.counts[1].tolist() == m.counts[1].tolist()


def test_a_trim_by_a_verdict_without_lengths_cuts_nothing():
    lens, block = [40, 33], 16
    table, stacks, counts, hbm, host = _trim(lens, lens, block, 0.5)
    g = torch.Generator().manual_seed(6)
    v = _verify(_probs(g, 6, 20), torch.zeros(2, 2, dtype=torch.int64), None, [0, 3], [3, 3], torch.ones(2, 2), torch.rand(2, generator=g))
    st, ct, ln = i32(stacks), i32(counts), i32(lens)
    out = gpu_ops.trim_tables(v.keep_lens, ln, i32(table), FreeBlocks(st[0], st[1], ct), hbm, host, block)
    ok()
    assert out.seq_lens.tolist() == lens and out.counts.tolist() == counts and st.tolist() == stacks


# ------------------------------------------------------------------ a run of them together


class Serving:
    """Requests whose drafted tokens are verified and whose caches are kept within a budget, one layer."""

    def __init__(self, seed, budget=48, over=8):
        self.R, self.K, self.KVH, self.H, self.D, self.BS, self.V = 4, 3, 2, 8, 64, 16, 50
        self.budget, self.over, self.sinks, self.recent = budget, over, 2, budget // 3
        self.G, self.C = 20, 24
        g = torch.Generator().manual_seed(seed)
        shape = (self.KVH, self.BS, self.D)
        cache = torch.zeros(self.G, *shape, dtype=torch.float16, device="cuda")
        host = [torch.zeros(self.C, *shape, dtype=torch.float16).pin_memory() for _ in range(2)]
        self.tiers = (KVTier(cache, cache.clone()), KVTier(*host))
        self.table = torch.zeros(self.R, 12, dtype=torch.int32, device="cuda")
        self.stack = torch.zeros(2, self.G + self.C, dtype=torch.int32, device="cuda")
        self.stack[0, :self.G] = torch.randperm(self.G, generator=g).int().cuda()
        self.stack[1, :self.C] = (torch.randperm(self.C, generator=g) + self.G).int().cuda()
        self.counts = i32([self.G, self.C])
        self.free = FreeBlocks(self.stack[0], self.stack[1], self.counts)
        self.lens, self.gone = i32([0] * self.R), i32([0] * self.R)
        self.T = self.R * 40
        self.t = StepTables(self.R, self.T, "cuda", seq_lens=self.lens, counts=self.counts)
        self.trim = TrimTables(self.R, "cuda", seq_lens=self.lens, counts=self.counts)
        self.stats = KeyStats.zeros(self.G + self.C, self.KVH, self.BS, "cuda")
        self.moves = KeyMoves(self.R, self.KVH, self.budget, "cuda")
        self.verdict = DraftVerdict(self.R, self.K, "cuda")
        ang = torch.outer(torch.arange(4096, dtype=torch.float64), 100.0 ** (-torch.arange(0, self.D, 2).double() / self.D))
        self.cos_sin = torch.cat([ang.cos(), ang.sin()], 1).float().cuda()
        z = lambda *n: torch.zeros(n, dtype=torch.float16, device="cuda")  # noqa: E731
        self.q, self.k, self.v = z(self.T, self.H, self.D), z(self.T, self.KVH, self.D), z(self.T, self.KVH, self.D)
        self.out, self.lse = z(self.T, self.H, self.D), torch.zeros(self.H, self.T, device="cuda")
        self.new, self.drafts = i32([0] * self.R), torch.zeros(self.R, self.K, dtype=torch.int64, device="cuda")
        self.target, self.probs = torch.zeros(self.T, self.V, device="cuda"), torch.zeros(self.R, self.K, self.V, device="cuda")
        self.au, self.su = torch.zeros(self.R, self.K, device="cuda"), torch.zeros(self.R, device="cuda")
        self.used, self.kept = i32([0] * self.R), i32([0] * self.R)

    def fill(self, step):
        g = torch.Generator().manual_seed(1000 + step)
        new = [30, 25, 0, 40] if step == 0 else [4, 0, 30, 4] if step == 1 else [4, -1, 2, 4] if step == 9 else [4, 3, 4, 1]
        if step == 10:
            new[1] = 35
        self.new.copy_(i32(new))
        for x in (self.q, self.k, self.v):
            x.copy_(torch.randn(x.shape, generator=g))
        p = _probs(g, self.T, self.V, spread=1.0)
        self.target.copy_(p)
        at = 0
        for r, n in enumerate(new):
            if 1 <= n <= self.K + 1:
                for d in range(n - 1):
                    self.probs[r, d] = (0.6 * p[at + d] + 0.4 * _probs(g, self.V, spread=1.0)).cuda()
            at += max(0, n)
        self.drafts.copy_(torch.randint(0, self.V, self.drafts.shape, generator=g))
        self.au.copy_(torch.rand(self.au.shape, generator=g) * 0.5)
        self.su.copy_(torch.rand(self.su.shape, generator=g))
        return new

    def attend(self):
        t = self.t
        gpu_ops.extend_tables(self.new, self.lens, self.table, self.free, self.G, self.C, self.BS, t, evicted=self.gone)
        gpu_ops.rope_store_kv(self.q, self.k, self.v, t.positions, self.cos_sin, t.slot_mapping, self.tiers, self.G)
        gpu_ops.chunk_attn(self.q, self.tiers, self.G, self.table, t.query_start_loc[:-1], t.query_lens, self.lens, self.D ** -0.5,
                           self.out, self.lse, max_q_len=40, max_k_len=180)

    def verify(self):
        # a prompt's step has no drafts: it samples from its last row
        ql, start = self.t.query_lens, self.t.query_start_loc[:-1]
        prompt = ql > self.K + 1
        first = torch.where(prompt, start + ql - 1, start)
        rows = torch.where(prompt, 1, ql)
        v = gpu_ops.verify_drafts(self.target, self.drafts, self.probs, first, rows, self.au, self.su, seq_lens=self.lens,
                                  out=self.verdict)
        self.used.copy_(torch.where(prompt | (ql == 0), ql, v.accepted + 1))
        gpu_ops.trim_tables(v.keep_lens, self.lens, self.table, self.free, self.G, self.C, self.BS, self.trim, max_cut=self.K)
        gpu_ops.key_weights(self.q, self.tiers, self.G, self.table, start, self.used, self.lens, self.D ** -0.5, self.lse, self.stats,
                            evicted=self.gone, max_q_len=40, max_k_len=180)

    def cut(self):
        self.kept.copy_(torch.where(self.lens > self.budget + self.over, self.budget, self.lens))
        gpu_ops.select_keys(self.stats, self.table, self.lens, self.kept, self.moves, sinks=self.sinks, recent=self.recent,
                            evicted=self.gone, max_k_len=180)
        gpu_ops.move_keys(self.moves, self.tiers, self.G, self.table, self.stats)
        gpu_ops.trim_tables(self.kept, self.lens, self.table, self.free, self.G, self.C, self.BS, self.trim, evicted=self.gone)

    def step(self):
        self.attend()
        self.verify()
        self.cut()

    def state(self):
        return [self.tiers[0].k, self.tiers[0].v, self.tiers[1].k, self.tiers[1].v, self.table, self.stack, self.counts, self.lens, self.gone,
                self.stats.weights, self.stats.positions, self.verdict.tokens, self.verdict.accepted, self.out, self.lse]

    def cached(self, r, n):
        """K, V [KVH, n, D], weights and positions [KVH, n] of request r."""
        torch.cuda.synchronize()
        ids = self.table[r].tolist()[:-(-n // self.BS)]
        blk = lambda t, u, b: t[b] if b < self.G else u[b - self.G].cuda()  # noqa: E731
        k, v = (torch.cat([blk(a, b, i) for i in ids], 1)[:, :n] if n else a[0][:, :0]
                for a, b in ((self.tiers[0].k, self.tiers[1].k), (self.tiers[0].v, self.tiers[1].v)))
        w, p = (torch.cat([x[i] for i in ids], 1)[:, :n] if n else x[0][:, :0] for x in (self.stats.weights, self.stats.positions))
        return k, v, w, p


@pytest.mark.parametrize("budget,over,least", [(48, 8, 2), (24, 0, 12)])
def test_serving_steps_against_lists(budget, over, least):
    """Twelve steps: attention over what stayed, accepted drafts, budgets, blocks; each against a plain account of every key."""
    s = Serving(3, budget, over)
    held = [[{} for _ in range(s.KVH)] for _ in range(s.R)]  # per head: position -> (k, v, weight)
    total = [0] * s.R                                        # tokens that a request has had
    cuts = 0
    for step in range(12):
        new = s.fill(step)
        s.attend()
        ok()
        s.t.read_header()
        for r in range(s.R):
            if new[r] < 0:
                held[r], total[r], new[r] = [{} for _ in range(s.KVH)], 0, 0
        start = [sum(new[:r]) for r in range(s.R)]
        assert s.t.positions.tolist()[:sum(new)] == [total[r] + i for r in range(s.R) for i in range(new[r])]
        n_before = s.lens.tolist()
        for r in range(s.R):
            n = n_before[r]
            assert n == len(held[r][0]) + new[r]
            if new[r] == 0:
                continue
            k, v, _, _ = s.cached(r, n)
            q = s.q[start[r]:start[r] + new[r]].double()
            for h in range(s.H):
                g = h // (s.H // s.KVH)
                old = [held[r][g][p] for p in sorted(held[r][g])]
                kk = torch.cat([torch.stack([x[0] for x in old]), k[g, n - new[r]:]]) if old else k[g]
                vv = torch.cat([torch.stack([x[1] for x in old]), v[g, n - new[r]:]]) if old else v[g]
                sc = q[:, h] @ kk.double().T * s.D ** -0.5
                sc = sc.masked_fill(torch.arange(n, device="cuda") > (n - new[r] + torch.arange(new[r], device="cuda"))[:, None], -math.inf)
                o = sc.softmax(-1) @ vv.double()
                # P and the result are rounded to fp16, half a step of 2^-11 each, of |v| below 5; scores in fp32
                assert float((s.out[start[r]:start[r] + new[r], h].double() - o).abs().max()) <= 2 * 2.0 ** -11 * 5 + 1e-4
                assert float((s.lse[h, start[r]:start[r] + new[r]].double() - sc.logsumexp(-1)).abs().max()) <= 1e-4
        fresh = [s.cached(r, n_before[r])[:2] for r in range(s.R)]
        s.verify()
        ok()
        t64, used = s.target.double().tolist(), s.used.tolist()
        for r in range(s.R):
            if new[r] == 0:
                assert s.verdict.tokens[r].tolist() == [-1] * (s.K + 1) and used[r] == 0
                continue
            prompt = new[r] > s.K + 1
            got, a = ref.verify(t64, s.drafts[r].tolist(), s.probs[r].double().tolist(), start[r] + new[r] - 1 if prompt else start[r],
                                1 if prompt else new[r], s.au[r].double().tolist(), float(s.su[r]))
            assert s.verdict.tokens[r].tolist() == got + [-1] * (s.K + 1 - len(got))
            assert used[r] == (new[r] if prompt else a + 1)
        lens = s.lens.tolist()
        for r in range(s.R):
            assert lens[r] == n_before[r] - new[r] + used[r]
            if used[r] == 0:
                continue
            k, v, w, p = s.cached(r, lens[r])
            for g in range(s.KVH):
                old = {x: held[r][g][x][2] for x in held[r][g]}
                pos = p[g].tolist()
                assert sorted(pos) == sorted(old) + [total[r] + i for i in range(used[r])]
                before = torch.tensor([old.get(x, 0.0) for x in pos], device="cuda")
                qh = s.q[start[r]:start[r] + used[r], g * 4:(g + 1) * 4]
                want, tol = ref.key_weights(qh, k[g][:, None], s.lse[g * 4:(g + 1) * 4, start[r]:start[r] + used[r]], before[None], s.D ** -0.5)
                assert bool(((w[g].double() - want[0]).abs() <= tol[0]).all())
                assert torch.equal(k[g, lens[r] - used[r]:], fresh[r][0][g, n_before[r] - new[r]:n_before[r] - new[r] + used[r]])
                held[r][g] = {x: (k[g, j].clone(), v[g, j].clone(), float(w[g, j])) for j, x in enumerate(pos)}
            total[r] += used[r]
        gone = s.gone.tolist()
        s.cut()
        ok()
        for r in range(s.R):
            n, keep = lens[r], s.budget if lens[r] > s.budget + s.over else lens[r]
            assert s.lens.tolist()[r] == keep and s.gone.tolist()[r] == gone[r] + n - keep == total[r] - keep
            cuts += keep < n
            k, v, w, p = s.cached(r, keep)
            for g in range(s.KVH):
                if keep < n:
                    guard = {x for x in held[r][g] if x < s.sinks or x >= total[r] - s.recent}
                    rest = sorted((x for x in held[r][g] if x not in guard), key=lambda x: -held[r][g][x][2])
                    ws = [held[r][g][x][2] for x in rest]
                    assert len(set(ws)) == len(ws)  # (no ties: which of two stays depends on their places)
                    held[r][g] = {x: held[r][g][x] for x in guard | set(rest[:keep - len(guard)])}
                pos = p[g].tolist()
                assert sorted(pos) == sorted(held[r][g])
                for j, x in enumerate(pos):
                    assert torch.equal(k[g, j], held[r][g][x][0]) and torch.equal(v[g, j], held[r][g][x][1])
                    assert float(w[g, j]) == held[r][g][x][2]
        # every block is on a stack or in a table once
        c = s.counts.tolist()
        used_ids = [b for r in range(s.R) for b in s.table[r].tolist()[:-(-s.lens.tolist()[r] // s.BS)]]
        assert sorted(used_ids + s.stack[0, :c[0]].tolist() + s.stack[1, :c[1]].tolist()) == list(range(s.G + s.C))
    assert cuts >= least


def test_serving_steps_in_one_graph():
    """The whole step captured once and replayed gives what eager steps give, bit for bit."""
    a, b = Serving(3), Serving(3)
    a.fill(0), b.fill(0)
    a.step(), b.step()  # (warm: lazy loading does not fall into the capture)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for step in range(1, 12):
        a.fill(step), b.fill(step)
        a.step()
        graph.replay()
        ok()
        for x, y in zip(a.state(), b.state()):
            assert torch.equal(x, y), step


# ------------------------------------------------------------------ the documented step


def _documented():
    """The documents' python blocks that verify drafts, by their file's name."""
    found = {}
    for path in sorted(Path(__file__).resolve().parents[1].glob("*.md")):
        for block in path.read_text().split("```python\n")[1:]:
            code = block.split("```")[0]
            if "verify_drafts(" in code:
                found[path.stem] = code
    return found


@pytest.mark.parametrize("where", sorted(_documented()) or ["none"])
def test_the_documented_step_of_prompts_and_drafts(where):
    """What the documents tell a user to run after the attention, on a step that mixes a long prompt, a prompt shorter
    than the drafts, drafts and a request without part."""
    code = _documented()[where]
    for new, prompt in (([4, 2, 30, 3], [False, True, True, False]), ([1, 0, 25, 4], [False, False, True, False])):
        s = Serving(3)
        s.fill(0)
        s.attend()
        s.verify()
        ok()
        s.fill(20)
        s.new.copy_(i32(new))
        total = s.lens.tolist()
        s.attend()
        ok()
        start = [sum(new[:r]) for r in range(s.R)]
        # one draft of each request that the target is sure of, so that some are accepted
        for r in range(s.R):
            if not prompt[r] and new[r] > 1:
                s.target[start[r]] = 0.0
                s.target[start[r], int(s.drafts[r, 0])] = 1.0
        w0, p0 = s.stats.weights.clone(), s.stats.positions.clone()
        ns = dict(torch=torch, gpu_ops=gpu_ops, R=s.R, K=s.K, KVH=s.KVH, G=s.G, C=s.C, BS=s.BS, device="cuda", counts=s.counts, free=s.free,
                  t=s.t, block_table=s.table, tiers=s.tiers, scale=s.D ** -0.5, q=s.q, lse=s.lse, target_probs=s.target, drafts=s.drafts,
                  draft_probs=s.probs, accept_u=s.au, sample_u=s.su, prompt=torch.tensor(prompt, device="cuda"), trim=s.trim, stats=s.stats,
                  moves=s.moves, room=s.budget, evicted=s.gone, layers=1, l=0, max_q=40, max_k=180, keep_lens=i32([-1] * s.R))
        exec(code, ns)
        ok()
        stats = ns["stats"]
        if isinstance(stats, list):  # made by the block itself
            stats, w0, p0 = stats[0], torch.zeros_like(w0), torch.zeros_like(p0)
        t64 = s.target.double().tolist()
        want_w, tol, want_p = w0.double(), torch.zeros_like(w0, dtype=torch.float64), p0.clone()
        accepted = 0
        for r in range(s.R):
            if new[r] == 0:
                used, got = 0, []
            else:
                first, rows = (start[r] + new[r] - 1, 1) if prompt[r] else (start[r], new[r])
                got, a = ref.verify(t64, s.drafts[r].tolist(), s.probs[r].double().tolist(), first, rows, s.au[r].double().tolist(),
                                    float(s.su[r]))
                used = new[r] if prompt[r] else a + 1
                accepted += 0 if prompt[r] else a
            assert ns["v"].tokens[r].tolist() == got + [-1] * (s.K + 1 - len(got))
            n = total[r] + used
            assert s.lens.tolist()[r] == n
            if used == 0:
                continue
            k = s.cached(r, n)[0]
            ids = torch.tensor(s.table[r].tolist(), device="cuda")
            j = torch.arange(n, device="cuda")
            blk, off = ids[j // s.BS], j % s.BS
            for g in range(s.KVH):
                qh = s.q[start[r]:start[r] + used, g * 4:(g + 1) * 4]
                w, e = ref.key_weights(qh, k[g][:, None], s.lse[g * 4:(g + 1) * 4, start[r]:start[r] + used], w0[blk, g, off][None], s.D ** -0.5)
                want_w[blk, g, off], tol[blk, g, off] = w[0], e[0]
                want_p[blk[total[r]:], g, off[total[r]:]] = j[total[r]:].int()
        assert accepted > 0
        assert bool(((stats.weights.double() - want_w).abs() <= tol).all())
        assert torch.equal(stats.positions, want_p)
