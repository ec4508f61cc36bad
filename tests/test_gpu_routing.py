"""Routing where the choice and its weights are hardest to get right, against
the 64-bit forms of tests/selection_util.py: groups whose scores saturate, and
rows that share a warp (a training batch), in every type."""
from __future__ import annotations

import math

import pytest
import torch

import spmvbench_b200 as S
from selection_util import check, choose, plan_of, weights_of

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def route(ctx, logits, k, bias=None, **spec):
    """(indices, weights) of the kernel, on the CPU."""
    tokens, experts = logits.shape
    R = S.Router(ctx, experts, k, max_tokens=tokens, **spec)
    indices = torch.full((tokens, k), 77, dtype=torch.int32, device=DEV)
    weights = torch.full((tokens, k), 77.0, device=DEV)
    R.route(logits.to(DEV), indices, weights, bias=None if bias is None else bias.to(DEV))
    ctx.check()
    return indices.cpu(), weights.cpu()


# ---- groups by their best logit --------------------------------------------------

@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_groups_by_their_best_logit_where_scores_are_equal(ctx, dtype, score):
    """Without a bias and with group_top = 1 a group's value is its best
    logit: sigmoids of 40 and 50 are both 1 in 64 bits, softmax scores of
    e^-800 and e^-900 both 0, and tiny logits' sigmoids all 1/2."""
    nan, inf, low = math.nan, math.inf, torch.finfo(dtype).min
    rows = torch.tensor([[40, 0, 50, nan], [40, 0, 50, inf], [40, 0, 50, low], [40, 0, 50, -1e9], [40, 0, 50, -inf],
                         [nan, 44, 41, 45], [1e-7, 0, 2e-7, nan], [1e-7, 0, 2e-7, -60000], [-900, -1000, -800, 0],
                         [-900, nan, -800, -2000], [-900, low, -800, -2000]]).to(dtype)
    for kept in (1, 2):
        indices, _ = route(ctx, rows, 1, score=score, groups=2, groups_kept=kept)
        assert torch.equal(indices, choose(rows, None, 1, score, 2, kept, 1))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("experts,k,groups,kept", [(32, 3, 4, 2), (64, 6, 8, 3), (60, 4, 5, 2), (256, 8, 8, 4), (34, 2, 17, 1)])
@pytest.mark.parametrize("tokens", [40, 1210])
def test_groups_of_saturated_scores(ctx, tokens, experts, k, groups, kept, score, dtype):
    """Rows of logits past 37 (sigmoid 1) or far below the row's largest
    (softmax 0), with NaN, infinities, the type's least value and -1e9 put in
    at random."""
    g = torch.Generator().manual_seed(experts + tokens)
    l = torch.rand(tokens, experts, generator=g) * 40 + 37
    if score == "softmax":
        l = -l * 20
        l[:, 0] = torch.where(torch.rand(tokens, generator=g) < 0.5, 0.0, l[:, 0])
    special = [-1e9, torch.finfo(dtype).min, -math.inf]
    special += [math.nan, math.inf] if score == "sigmoid" else []
    for v in special:
        hit = (torch.rand(tokens, experts, generator=g) < 1.0 / experts) & (torch.rand(tokens, 1, generator=g) < 0.4)
        l = torch.where(hit, v, l)
    l = l.to(dtype)
    indices, _ = route(ctx, l, k, score=score, groups=groups, groups_kept=kept)
    assert torch.equal(indices, choose(l, None, k, score, groups, kept, 1))


# ---- a lone choice ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("tokens", [150, 3000])
def test_a_lone_choice_has_the_whole_weight(ctx, tokens, score, dtype):
    """k = 1, renormalised: x / x is 1, so the weight is the scale and does not
    depend on the logits; the same where masks leave one expert of many."""
    g = torch.Generator().manual_seed(tokens)
    l = (torch.randn(tokens, 64, generator=g) * 3).to(dtype)
    lone = torch.full_like(l, -math.inf).scatter_(1, torch.randint(0, 64, (tokens, 1), generator=g), l[:, :1])
    for logits, k in ((l, 1), (lone, 5)):
        indices, weights = route(ctx, logits, k, score=score, scale=2.5)
        assert (indices[:, 0] >= 0).all() and (indices[:, 1:] == -1).all()
        assert (weights[:, 0] == 2.5).all() and not weights[:, 1:].any()
        d = torch.full((tokens, 64), 7.0, device=DEV, dtype=dtype)
        R = S.Router(ctx, 64, k, max_tokens=tokens, score=score, scale=2.5)
        R.route_grad(logits.to(DEV), indices.to(DEV), torch.randn(tokens, k, generator=g).to(DEV), d)
        assert not d.any()


# ---- rows that share a warp ------------------------------------------------------

def weight_error(logits, picks, score, renormalise, experts):
    """fp32's error of a row's weights, relative, u = 2^-24 a rounding. exp has
    2 u and u a unit of its argument (a difference of two logits, `reach` at
    most); a quotient 4 u; a scale 1 u.
    - renormalised: two such exps, under the sigmoid each over 1 + exp (5 + 4
      u), up to 32 values summed in a tree (5 u), a quotient, the scale.
    - sigmoid: exp, 1 +, quotient, scale.
    - softmax: exp over the row's sum, whose exps are rougher (4 u, and 2 u a
      unit: the argument times log2 e) and are added 64 one after the other at
      most and 5 in a tree."""
    l = logits.double()
    if renormalise:
        l = torch.where(picks >= 0, l.gather(1, picks.clamp(min=0).long()), math.nan)
        if score == "sigmoid":
            l = l.clamp(max=0)
    elif score == "sigmoid":
        return torch.full((l.shape[0], 1), 12 * 2.0 ** -24, dtype=torch.float64)
    there = (l > -math.inf) & (l < math.inf)
    reach = torch.where(there, l, -1e30).amax(1, keepdim=True) - torch.where(there, l, 1e30).amin(1, keepdim=True)
    # Past 120 below the largest a weight is 0 in fp32, and its error absolute.
    reach = torch.where(there.any(1, keepdim=True), reach, 0.0).clamp(0, 120)
    return (2 * reach + 24 if renormalise else 3 * reach + 16 + experts / 8) * 2.0 ** -24


SHARED = [
    # experts, k, score, renormalise, groups, kept, top, bias
    (16, 2, "softmax", True, 1, 1, 1, False), (16, 8, "sigmoid", False, 4, 2, 2, True), (60, 4, "softmax", False, 1, 1, 1, False),
    (60, 4, "sigmoid", True, 5, 3, 1, False), (64, 8, "softmax", True, 1, 1, 1, False), (64, 6, "sigmoid", True, 8, 3, 2, True),
    (64, 2, "softmax", False, 8, 2, 1, False), (64, 8, "softmax", False, 8, 4, 2, False), (100, 10, "softmax", True, 1, 1, 1, True),
    (100, 6, "sigmoid", False, 4, 2, 2, False), (128, 16, "sigmoid", True, 16, 8, 2, True), (128, 8, "softmax", False, 1, 1, 1, False),
    (96, 12, "softmax", True, 4, 2, 1, False), (3, 1, "sigmoid", False, 1, 1, 1, False), (256, 8, "sigmoid", True, 8, 4, 2, True)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("experts,k,score,renormalise,groups,kept,top,bias", SHARED)
def test_rows_that_share_a_warp(ctx, experts, k, score, renormalise, groups, kept, top, bias, dtype):
    """A training batch (1,301 rows, of which four or two share a warp):
    choices, weights and plan, with masks, equal logits, and rows of NaN and
    infinities beside ordinary ones."""
    tokens = 1301
    g = torch.Generator().manual_seed(experts * 3 + k)
    l = torch.randn(tokens, experts, generator=g) * 2
    l = torch.where(torch.rand(tokens, 1, generator=g) < 0.3, (l * 2).round() / 2, l)
    l = torch.where(torch.rand(tokens, experts, generator=g) < 0.1, -math.inf, l)
    l[torch.rand(tokens, generator=g) < 0.05] = -math.inf
    for v in (math.nan, math.inf, torch.finfo(dtype).min):
        l = torch.where((torch.rand(tokens, experts, generator=g) < 0.3) & (torch.rand(tokens, 1, generator=g) < 0.04), v, l)
    l[7] = math.nan
    l = l.to(dtype)
    b = (torch.randn(experts, generator=g) * 0.1) if bias else None
    spec = dict(score=score, renormalise=renormalise, scale=2.5, groups=groups, groups_kept=kept, group_top=top)
    R = S.Router(ctx, experts, k, max_tokens=tokens, **spec)
    i32 = dict(dtype=torch.int32, device=DEV)
    indices, weights = torch.full((tokens, k), 77, **i32), torch.full((tokens, k), 77.0, device=DEV)
    offsets, order, position = torch.full((experts + 1,), 77, **i32), torch.full((tokens * k,), -77, **i32), torch.full((tokens, k), 77, **i32)
    wide = torch.full((tokens, experts + 3), math.nan, device=DEV, dtype=dtype)
    wide[:, :experts] = l.to(DEV)
    picks = choose(l, b, k, score, groups, kept, top)
    none = (torch.isnan(l) | (l == math.inf)).any(1, keepdim=True) if score == "softmax" else torch.zeros(tokens, 1, dtype=torch.bool)
    ref = torch.where(none, math.nan, weights_of(l, picks, score, renormalise, 2.5))
    bound = ref.nan_to_num().abs() * weight_error(l, picks, score, renormalise, experts) + 2.0 ** -120
    # Rows of a wider buffer, then rows that 16-byte words fit; with the plan, then without.
    for logits in (wide[:, :experts], l.to(DEV)):
        R.route(logits, indices, weights, bias=None if b is None else b.to(DEV), offsets=offsets, order=order, position=position)
        assert torch.equal(indices.cpu(), picks)
        check(weights, ref, bound, "weights")
        o, by, at = plan_of(picks, experts)
        assert offsets.tolist() == o and position.flatten().tolist() == at and order[:len(by)].tolist() == by
        again, w2 = route(ctx, logits, k, bias=b, **spec)
        assert torch.equal(again, picks) and torch.equal(w2.view(torch.int32), weights.cpu().view(torch.int32))
    # Every row alone chooses the same.
    some = list(range(0, tokens, 37)) + [7]
    for t in some:
        i, w = route(ctx, l[t:t + 1], k, bias=b, **spec)
        assert torch.equal(i[0], picks[t])
        check(w, ref[t:t + 1], bound[t:t + 1], "weights of a row alone")
    ctx.check()
