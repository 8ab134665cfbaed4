"""Plain 64-bit forms of the multi-token step's operators, for their tests."""

from __future__ import annotations

import torch


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, limit, scale):
    """One request: q [nq, H, D], k / v [nk, KVH, D], query i sees keys 0 ..
    limit[i].  Returns float64 o, lse [H, nq], A = sum p |v| / l (the scale of
    P.V's rounding) and the largest |q|.|k| scale (that of the scores')."""
    nq, H, D = q.shape
    nk, KVH = k.shape[0], k.shape[1]
    qd = q.double().transpose(0, 1)                                       # [H, nq, D]
    kd = k.double().transpose(0, 1).repeat_interleave(H // KVH, 0)        # [H, nk, D]
    vd = v.double().transpose(0, 1).repeat_interleave(H // KVH, 0)
    s = qd @ kd.transpose(1, 2) * scale
    seen = torch.arange(nk, device=q.device) <= limit[:, None]
    s = s.masked_fill(~seen, float("-inf"))
    lse = torch.logsumexp(s, -1) if nk else torch.full((H, nq), float("-inf"), dtype=torch.float64, device=q.device)
    p = torch.where(seen, (s - torch.where(lse.isinf(), 0.0, lse)[..., None]).exp(), 0.0)
    big = float((qd.abs() @ kd.abs().transpose(1, 2)).max()) * scale if nk and nq else 0.0
    return (p @ vd).transpose(0, 1), lse, (p @ vd.abs()).transpose(0, 1), big


def attn_bounds(dtype, o, A, big, nk, D, p_rounded):
    """How far o and lse may be off.  Scores: a sum of D products in fp32 is
    off by at most D 2^-24 of the sum of their sizes (big), scaled with two
    more roundings; the exponent's error is the relative error of p, in the
    numerator and in the sum; ex2 adds 2^-21 and sums of nk terms nk 2^-24,
    in as many again for the joins.  P is rounded to the type for P.V where
    `p_rounded`, the result once."""
    u = half_step(dtype)
    rel = 2 * ((D + 4) * 2.0 ** -24 * big + 2.0 ** -21 + (nk + 300) * 2.0 ** -24)
    return u * o.abs() + (rel + (u if p_rounded else 0.0)) * A + 2.0 ** -24, rel + 2.0 ** -22 * 20


def check_attn(out, lse, refs, q_start, q_len, dtype, D, p_rounded, untouched=True):
    """Compare every request's rows; rows of no request must still be NaN."""
    covered = torch.zeros(out.shape[0], dtype=torch.bool, device=out.device)
    for r, (o, l, A, big, nk) in enumerate(refs):
        a, b = int(q_start[r]), int(q_start[r]) + int(q_len[r])
        covered[a:b] = True
        if a == b:
            continue
        tol, tol_l = attn_bounds(dtype, o, A, big, nk, D, p_rounded)
        err = (out[a:b].double() - o).abs()
        assert bool((err <= tol).all()), (r, float((err - tol).max()), float(err.max()))
        if lse is not None:
            got, none = lse[:, a:b].double(), l.isinf()
            assert bool((got[none] == float("-inf")).all()), r
            e = (got - l)[~none].abs()
            assert bool((e <= tol_l).all()), (r, float(e.max()), tol_l)
    if untouched:
        assert bool(out[~covered].isnan().all())
        assert lse is None or bool(lse[:, ~covered].isnan().all())


def tables(new, prior, table, stacks, counts, num_gpu, block_size, max_tokens):
    """extend_tables on lists; None when the step cannot be applied."""
    table, stacks, counts = [list(r) for r in table], [list(s) for s in stacks], list(counts)
    W = len(table[0]) if table else 0
    for r, n in enumerate(new):
        if n == -1:
            for b in table[r][:-(-prior[r] // block_size)]:
                t = 0 if b < num_gpu else 1
                if counts[t] >= len(stacks[t]):
                    return None
                stacks[t][counts[t]] = b
                counts[t] += 1
    qsl, slots, pos, seq = [0], [], [], []
    for r, n in enumerate(new):
        if n < -1 or prior[r] < 0 or prior[r] + max(0, n) > W * block_size:
            return None
        for p in range(prior[r], prior[r] + max(0, n)):
            if p % block_size == 0:
                t = 0 if counts[0] else 1
                if not counts[t]:
                    return None
                counts[t] -= 1
                table[r][p // block_size] = stacks[t][counts[t]]
            slots.append(table[r][p // block_size] * block_size + p % block_size)
            pos.append(p)
        seq.append(0 if n < 0 else prior[r] + n)
        qsl.append(len(slots))
    if len(slots) > max_tokens:
        return None
    pad = max_tokens - len(slots)
    return table, stacks, counts, seq, qsl, slots + [-1] * pad, pos + [0] * pad


def rope(x, positions, cos_sin, axis, pairs):
    """x [T, heads, D] rotated in float64; axis: the axis of each pair."""
    rot = cos_sin.shape[1]
    half = rot // 2
    at = positions[torch.tensor(list(axis), device=x.device)].T             # [T, pairs]
    i = torch.arange(half, device=x.device)
    c, s = cos_sin.double()[at, i][:, None], cos_sin.double()[at, half + i][:, None]
    y = x.double().clone()
    f, g = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, half), slice(half, rot))
    a, b = x.double()[..., f], x.double()[..., g]
    y[..., f], y[..., g] = a * c - b * s, b * c + a * s
    return y
