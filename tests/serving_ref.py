"""Plain 64-bit and list forms of the operators behind a step's attention, for
their tests."""

from __future__ import annotations

import math

import torch


def key_weights(q, k, lse, old, scale):
    """One request: q [nq, H, D], k [nk, KVH, D], lse [H, nq]; query i sees keys
    0 .. nk - nq + i.  Returns in float64 the weights [KVH, nk] that the keys
    receive and how far a sum in fp32 may be off; `old` [KVH, nk]: what the
    older keys had.

    A score is a sum of D products in fp32, off by at most D 2^-23 of the sum
    of their sizes where each addition may be cut off instead of rounded; its
    scaling, the scaled lse and their difference are rounded once each (2^-24 of
    their sizes).  That error of the exponent is the relative error of its
    power, to which ex2 adds 2^-21; a sum of m terms adds m 2^-24, as does the
    addition to what the key had."""
    nq, H, D = q.shape
    nk, KVH = k.shape[0], k.shape[1]
    G = H // KVH
    qd = q.double().transpose(0, 1)
    kd = k.double().transpose(0, 1).repeat_interleave(G, 0)
    s = qd @ kd.transpose(1, 2) * scale                                     # [H, nq, nk]
    seen = torch.arange(nk, device=q.device) <= (nk - nq + torch.arange(nq, device=q.device))[:, None]
    ls = lse.double()[..., None]
    p = torch.where(seen & ~ls.isinf(), (s - ls).exp(), 0.0)
    size = qd.abs() @ kd.abs().transpose(1, 2) * scale
    err = p * (D * 2.0 ** -23 * size + 4 * 2.0 ** -24 * (size + ls.abs().nan_to_num(posinf=0.0)) + 2.0 ** -21)
    w, e = (x.sum(1).view(KVH, G, nk).sum(1) for x in (p, torch.where(p > 0, err, 0.0)))
    e = e + w * (nq * G + 16) * 2.0 ** -24
    new = torch.arange(nk, device=q.device) >= nk - nq
    w = torch.where(new, w, old.double() + w)
    return w, e + w.abs() * 2.0 ** -23 + 1e-37


def select(weights, positions, n, keep, gone, sinks, recent):
    """One request and kv head, on lists: (src, dst) of the moves."""
    if keep < 0 or keep >= n:
        return [], []
    guarded = [p < sinks or p >= n + gone - recent for p in positions]
    rank = [0.0 if g else (math.inf if math.isnan(w) else -w) for g, w in zip(guarded, weights)]
    order = sorted(range(n), key=lambda j: (not guarded[j], not guarded[j] and math.isnan(weights[j]), rank[j], j))
    stays = set(order[:keep])
    return [j for j in range(keep, n) if j in stays], [j for j in range(keep) if j not in stays]


def trim(keep, lens, table, stacks, counts, num_gpu, block_size):
    """trim_tables on lists; None when the call cannot be applied."""
    stacks, counts, left = [list(s) for s in stacks], list(counts), []
    for r, (b, n) in enumerate(zip(keep, lens)):
        if n < 0 or n > len(table[r]) * block_size:
            return None
        left.append(b if 0 <= b < n else n)
        for block in table[r][-(-left[r] // block_size):-(-n // block_size)]:
            t = 0 if block < num_gpu else 1
            if counts[t] >= len(stacks[t]):
                return None
            stacks[t][counts[t]] = block
            counts[t] += 1
    return stacks, counts, left


def _weight(x):
    return x if 0.0 < x < math.inf else 0.0


def verify(target, tokens, draft, start, q_len, accept_u, sample_u):
    """One request, value by value: target [T, V], tokens [K], draft [K, V] or
    None (lists of floats); (tokens, accepted)."""
    if q_len == 0:
        return [], 0
    got = []
    V = len(target[0])
    for d in range(q_len - 1):
        x = tokens[d]
        if not 0 <= x < V:
            break
        q = 1.0 if draft is None else _weight(draft[d][x])
        if not accept_u[d] * q < _weight(target[start + d][x]):
            break
        got.append(x)
    a = len(got)
    p = [_weight(x) for x in target[start + a]]
    w = p
    if a < q_len - 1 and draft is not None:
        w = [_weight(x - _weight(y)) for x, y in zip(target[start + a], draft[a])]
    elif a < q_len - 1:
        w = [0.0 if i == tokens[a] else x for i, x in enumerate(p)]
    if not sum(w) > 0.0:
        w = p
    if not sum(w) > 0.0:
        return got + [-1], a
    total = 0.0
    for x in w:
        total += x
    u = min(max(sample_u, 0.0), 1.0 - 2.0 ** -24) if sample_u == sample_u else 0.0
    run = 0.0
    for i, x in enumerate(w):
        run += x
        if run > u * total:
            break
    return got + [i], a
