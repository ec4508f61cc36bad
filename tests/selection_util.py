"""Plain 64-bit forms of the row-selection operators, and the error bounds
their tests hold the kernels to.

A result computed in precision u (2^-24 in fp32, 2^-53 in fp64) from n terms,
in any order, is within gamma = (n + 2) u of the exact one relative to the sum
of the terms' magnitudes (one rounding a product, n - 1 sums, the scale, and a
sum into what was there). Rounding it to the output's type adds half a step:
eps / 2 of the value, or half the smallest subnormal."""
from __future__ import annotations

import math

import torch

UNIT = {torch.float64: 2.0 ** -53}


def allowed(ref, magnitude, terms: int, dtype):
    u = UNIT.get(dtype, 2.0 ** -24)
    err = (terms + 2) * u / (1 - (terms + 2) * u) * magnitude
    f = torch.finfo(dtype)
    return err + f.eps / 2 * (ref.abs() + err) + f.smallest_normal * f.eps / 2


def check(got, ref, bound, label=""):
    got, ref = got.double().cpu(), ref.cpu()
    bound = bound.cpu() if torch.is_tensor(bound) else torch.full_like(ref, bound)
    assert got.shape == ref.shape
    bad = ~((got - ref).abs() <= bound)
    bad &= ~(torch.isnan(got) & torch.isnan(ref)) & (got != ref)
    assert not bad.any(), (f"{label}: {int(bad.sum())} of {bad.numel()} out of bound, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()!r} against {ref[bad][0].item()!r}, {bound[bad][0].item():.3g} allowed")


def rows_at(X, idx):
    """X's rows in 64 bits, zeros where idx is negative."""
    idx = idx.long()
    return torch.where((idx >= 0).unsqueeze(-1), X.double()[idx.clamp(min=0)], 0.0)


def grad_rows(tokens, dout, rows):
    """(sums, sums of magnitudes, most terms) of dout's rows by token."""
    keep = tokens >= 0
    at, d = tokens[keep].long(), dout.double()[keep]
    zero = torch.zeros(rows, dout.shape[1], dtype=torch.float64, device=dout.device)
    most = int(torch.bincount(at, minlength=1).max()) if at.numel() else 0
    return zero.index_add(0, at, d), zero.index_add(0, at, d.abs()), most


def scores(logits, score):
    l = logits.double()
    if score == "sigmoid":
        return torch.sigmoid(l)
    out = torch.zeros_like(l)
    for t, row in enumerate(l):
        if not torch.isnan(row).any() and row.max() < math.inf and row.max() > -math.inf:
            out[t] = torch.softmax(row, 0)
    return out


def choose(logits, bias, k, score, groups=1, groups_kept=1, group_top=1):
    """The chosen experts of every row, one row and one choice at a time."""
    value = scores(logits, score)
    logits = logits.double()
    picks = torch.full((logits.shape[0], k), -1, dtype=torch.int32)
    experts = logits.shape[1]
    per = experts // groups
    for t in range(logits.shape[0]):
        l = logits[t].tolist()
        if score == "softmax" and any(math.isnan(x) or x == math.inf for x in l):
            continue
        s = value[t].tolist()
        rank = l if bias is None else [a + float(b) for a, b in zip(s, bias)]
        open_ = [e for e in range(experts) if l[e] > -math.inf and rank[e] > -math.inf]
        if groups > 1:
            level = []
            for g in range(groups):
                inside = [e for e in open_ if e // per == g]
                worth = [rank[e] if bias is not None or group_top == 1 else s[e] for e in inside]
                worth = sorted(worth, reverse=True)[:group_top]
                level.append(sum(worth) if worth else -math.inf)
            kept = sorted(range(groups), key=lambda g: (-level[g], g))[:groups_kept]
            open_ = [e for e in open_ if e // per in kept]
        for j, e in enumerate(sorted(open_, key=lambda e: (-rank[e], e))[:k]):
            picks[t, j] = e
    return picks


def weights_of(logits, picks, score, renormalise, scale):
    """The weights of a choice, from the logarithms of the scores, in 64 bits
    (differentiable in logits)."""
    l = logits.double()
    there = picks >= 0
    at = picks.long().clamp(min=0)
    # log_softmax and softmax take the largest logit off first: the lowest finite value of a type is an ordinary logit.
    if score == "sigmoid":
        log = torch.nn.functional.logsigmoid(l).gather(1, at)
    else:
        log = (l if renormalise else torch.log_softmax(l, 1)).gather(1, at)
    if renormalise:
        share = torch.softmax(torch.where(there, log, -math.inf), 1)
    else:
        share = torch.exp(torch.where(there, log, 0.0))
    return torch.where(there, share, 0.0) * scale


def plan_of(picks, experts):
    """(offsets, order, position) of a choice, entry by entry."""
    flat = picks.reshape(-1).tolist()
    by = [[i for i, e in enumerate(flat) if e == x] for x in range(experts)] if len(flat) < 4000 else None
    if by is None:
        by = [[] for _ in range(experts)]
        for i, e in enumerate(flat):
            if 0 <= e < experts:
                by[e].append(i)
    offsets, order, position = [0], [], [-1] * len(flat)
    for rows in by:
        for i in rows:
            position[i] = len(order)
            order.append(i)
        offsets.append(len(order))
    return offsets, order, position
