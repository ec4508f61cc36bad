"""Routing where the choice and its weights are hardest to get right, against
the 64-bit forms of tests/selection_util.py: groups whose scores saturate, and
rows that share a warp (a training batch), in every type."""
from __future__ import annotations

import math

import pytest
import torch

import spmvbench_b200 as S
from selection_util import choose

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
