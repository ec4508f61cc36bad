"""The exchange with the experts where every row begins and ends on a 16-byte
word, for every number of choices: one, up to eight (rows in shared memory) and
up to 32 (rows in registers). Against 64 bits; bounds in
tests/selection_util.py."""
from __future__ import annotations

import pytest
import torch

import spmvbench_b200 as S
from selection_util import allowed, check, rows_at

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def rows_of(rows, width, dtype, pad, g):
    base = torch.full((rows, width + pad), float("nan"), device=DEV, dtype=dtype)
    base[:, :width] = torch.randn(rows, width, generator=g, device=DEV).to(dtype)
    return base[:, :width], base


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("k", [1, 2, 8, 9, 10, 17, 31, 32])
@pytest.mark.parametrize("tokens,width,pad", [(37, 8, 0), (5, 128, 8), (37, 1000, 16), (3, 2056, 0), (130, 4096, 0), (2, 8200, 8)])
def test_exchange_of_aligned_rows(ctx, tokens, width, pad, k, dtype):
    g = torch.Generator(device=DEV).manual_seed(tokens + 40 * k + width)
    rows = tokens * k + 3
    R = S.Router(ctx, 32, k, max_tokens=tokens)
    position = torch.randperm(rows, generator=g, device=DEV)[:tokens * k].view(tokens, k).int()
    position[torch.rand(tokens, k, generator=g, device=DEV) < 0.2] = -1
    position[0] = -1  # a token without experts
    w = torch.rand(tokens, k, generator=g, device=DEV) - 0.3
    X, _ = rows_of(tokens, width, dtype, pad, g)
    Y, _ = rows_of(rows, width, dtype, pad, g)
    there = position >= 0
    named = torch.zeros(rows, dtype=torch.bool, device=DEV)
    named[position[there].long()] = True

    def rows_named_alone(got, base, before):
        assert torch.equal(got[~named], before[~named]), "a row that no position names was written"
        assert torch.isnan(base[:, width:]).all(), "written beside the rows"

    xs, base = rows_of(rows, width, dtype, pad, g)
    before = xs.clone()
    R.dispatch(position, X, xs)
    rows_named_alone(xs, base, before)
    ref = before.clone()
    ref[position[there].long()] = X.repeat_interleave(k, 0)[there.flatten()]
    assert torch.equal(xs, ref)

    out, base = rows_of(tokens, width, dtype, pad, g)
    terms = rows_at(Y, position) * w.double().unsqueeze(-1)
    R.combine(position, w, Y, out)
    check(out, terms.sum(1), allowed(terms.sum(1), terms.abs().sum(1), k, dtype), "combine")
    terms = rows_at(Y, position)
    R.dispatch_grad(position, Y, out)
    check(out, terms.sum(1), allowed(terms.sum(1), terms.abs().sum(1), k, dtype), "dispatch_grad")
    assert not out[0].any() and (pad == 0 or torch.isnan(base[:, width:]).all())

    dY, base = rows_of(rows, width, dtype, pad, g)
    before = dY.clone()
    dw = torch.full((tokens, k), 7.0, device=DEV)
    R.combine_grad(position, w, Y, X, dY, dw)
    rows_named_alone(dY, base, before)
    ref = before.double()
    ref[position[there].long()] = (X.double().unsqueeze(1) * w.double().unsqueeze(-1))[there]
    check(dY, ref, allowed(ref, ref.abs(), 1, dtype), "dY")
    terms = rows_at(Y, position) * X.double().unsqueeze(1)
    check(dw, terms.sum(2), allowed(terms.sum(2), terms.abs().sum(2), width, torch.float32), "dweights")
    assert not dw[~there].any()
    ctx.check()
