"""Row-selection operators on the GPU against plain 64-bit forms: embedding
lookup and gradient, routing, the experts' plan and exchange, and all of them
together. Bounds: tests/selection_util.py."""
from __future__ import annotations

import math

import pytest
import torch

import spmvbench_b200 as S
from selection_util import allowed, check, choose, grad_rows, plan_of, rows_at, weights_of

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]
ALL = FLOATS + [torch.float64]
DEV = "cuda:0"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, g, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def tokens_of(count, rows, g, empty=0.1):
    t = torch.randint(0, rows, (count,), generator=g, device=DEV, dtype=torch.int32)
    return torch.where(torch.rand(count, generator=g, device=DEV) < empty, -1, t).int()


def strided(rows, width, dtype, pad=0, shift=0, fill=float("nan")):
    """A rows x width view with `pad` extra columns a row, `shift` elements
    into its storage; returns (view, everything around it)."""
    base = torch.full((rows * (width + pad) + shift,), fill, device=DEV, dtype=dtype)
    return base[shift:].view(rows, width + pad)[:, :width], base


def outside_untouched(base, view):
    """Nothing but the view was written in its storage (filled with NaN)."""
    kept = base.clone()
    torch.as_strided(kept, view.shape, view.stride(), view.storage_offset()).fill_(float("nan"))
    assert torch.isnan(kept).all(), "written outside the rows"


# ---- embedding ----------------------------------------------------------------

@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("count,rows,width,pad,shift", [
    (1, 1, 1, 0, 0), (1, 5, 64, 0, 0), (3, 7, 7, 2, 1), (33, 100, 8, 0, 0), (130, 50, 1000, 24, 8), (65, 300, 1001, 3, 1),
    (40, 1000, 4096, 0, 0), (17, 9, 2052, 4, 4), (5, 3, 12, 0, 2), (0, 4, 16, 0, 0)])
def test_lookup(ctx, dtype, count, rows, width, pad, shift):
    g = gen(count * 31 + width)
    tokens = tokens_of(count, rows, g)
    table, tbase = strided(rows, width, dtype, pad, shift)
    table.copy_(randn(rows, width, g=g))
    out, base = strided(count, width, dtype, pad, shift)
    E = S.Embedding(ctx, rows, width, max_tokens=0)
    E.lookup(tokens, table, out, scale=1.75)
    ref = rows_at(table, tokens) * 1.75
    check(out, ref, allowed(ref, ref.abs(), 1, dtype), "lookup")
    if count:
        outside_untouched(base, out)
    ctx.check()


def test_lookup_of_scale_one_is_a_copy_and_matches_the_sparse_product(ctx):
    """scale 1 returns the rows bit for bit: the product of the CSR matrix
    with one 1 per row and the table, as DeviceMatrix.spmm computes it."""
    import numpy as np
    g = gen(5)
    rows, width, count = 300, 64, 500
    tokens = tokens_of(count, rows, g, empty=0.2)
    table = randn(rows, width, g=g)
    out = torch.empty(count, width, device=DEV)
    S.Embedding(ctx, rows, width, max_tokens=0).lookup(tokens, table, out)
    there = (tokens >= 0).cpu().numpy()
    rowptr = np.concatenate([[0], np.cumsum(there)]).astype(np.int32)
    A = S.CsrMatrix(count, rows, rowptr, tokens.cpu().numpy()[there], np.ones(int(there.sum())))
    M = S.DeviceMatrix(ctx, A, S.F32)
    Y = torch.empty(count, width, device=DEV)
    M.spmm(table, Y, width, tile=64)
    assert torch.equal(out, Y)
    M.close()


@pytest.mark.parametrize("grad32", [False, True])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("count,rows,width,pad,shift", [
    (1, 1, 1, 0, 0), (1, 4, 64, 0, 0), (16, 1, 33, 0, 0), (17, 2, 8, 3, 1), (100, 40, 1000, 24, 8), (300, 600000, 16, 0, 0),
    (1500, 3, 257, 0, 1), (5000, 1200, 72, 8, 8), (0, 6, 16, 0, 0), (64, 8, 4096, 0, 0)])
def test_lookup_grad(ctx, dtype, count, rows, width, pad, shift, accumulate, grad32):
    if grad32 and dtype in (torch.float32, torch.float64):
        pytest.skip("the gradient has the rows' type already")
    g = gen(count + width)
    tokens = tokens_of(count, rows, g)
    dout, _ = strided(count, width, dtype, pad, shift)
    dout.copy_(randn(count, width, g=g))
    kind = torch.float32 if grad32 else dtype
    dtable, base = strided(rows, width, kind, pad, shift)
    before = randn(rows, width, g=g).to(kind) if accumulate else torch.full_like(dtable, float("nan"))
    dtable.copy_(before)
    E = S.Embedding(ctx, rows, width, max_tokens=count + 3)
    E.lookup_grad(tokens, dout, dtable, scale=0.75, accumulate=accumulate)
    total, size, most = grad_rows(tokens, dout, rows)
    ref, size = total * 0.75, size * 0.75
    if accumulate:
        ref, size = ref + before.double(), size + before.double().abs()
    check(dtable, ref, allowed(ref, size, most + 1, kind), "lookup_grad")
    outside_untouched(base, dtable)
    if accumulate:
        named = torch.zeros(rows, dtype=torch.bool, device=DEV)
        named[tokens[tokens >= 0].long()] = True
        assert torch.equal(dtable[~named], before[~named])
    ctx.check()


@pytest.mark.parametrize("runs", [[16, 16, 16], [15, 1, 17, 31, 2], [1, 200, 3], [4096], [5, 16, 11, 16, 160, 1]])
def test_lookup_grad_runs_that_meet_chunk_edges(ctx, runs):
    """Rows named by runs of tokens of every alignment, in shuffled order,
    with integers whose sums fp32 holds exactly: the result is exact."""
    g = gen(sum(runs))
    tokens = torch.repeat_interleave(torch.arange(len(runs)) * 3, torch.tensor(runs)).int()
    tokens = tokens[torch.randperm(tokens.numel(), generator=torch.Generator().manual_seed(1))].to(DEV)
    dout = torch.randint(-64, 65, (tokens.numel(), 40), generator=g, device=DEV).float()
    dtable = torch.full((3 * len(runs), 40), 9.0, device=DEV)
    E = S.Embedding(ctx, 3 * len(runs), 40, max_tokens=5000)
    E.lookup_grad(tokens, dout, dtable)
    assert torch.equal(dtable.double(), grad_rows(tokens, dout, 3 * len(runs))[0])


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("count,rows,hot", [
    (256, 40, 0.0), (257, 40, 0.3), (2048, 3000, 0.1), (2049, 3000, 0.1), (9000, 2000, 0.5), (16384, 131072, 0.02),
    (16384, 7, 1.0), (16385, 50000, 0.3), (70000, 300, 0.2), (140000, 600000, 0.0), (600, 9_000_000, 0.2), (30, 9_000_000, 0.0),
    (3000, 1_000_000, 0.0)])
def test_lookup_grad_of_every_way_to_sort(ctx, count, rows, hot, accumulate):
    """Every number of tokens that is sorted in its own way, with a token that
    is most of a block's; two calls in a row (the scratch is left as it was
    found), integers: exact."""
    g = gen(count + rows)
    tokens = tokens_of(count, rows, g, empty=0.05)
    tokens = torch.where(torch.rand(count, generator=g, device=DEV) < hot, rows - 1, tokens).int()
    E = S.Embedding(ctx, rows, 8, max_tokens=count)
    for turn in range(2):
        dout = torch.randint(-16, 17, (count, 8), generator=g, device=DEV).float()
        dtable = torch.randint(-4, 5, (rows, 8), generator=g, device=DEV).float()
        want = grad_rows(tokens, dout, rows)[0] + (dtable.double() if accumulate else 0)
        E.lookup_grad(tokens, dout, dtable, accumulate=accumulate)
        assert torch.equal(dtable.double(), want), turn
        tokens = tokens.flip(0).contiguous()
    ctx.check()


@pytest.mark.parametrize("width", [8, 600, 4096])
@pytest.mark.parametrize("runs", [
    [188, 189, 190, 191, 192, 193, 194, 195, 196], [3, 752, 1, 767, 768, 769, 784], [1024, 16, 1023, 1025],
    [12, 4096, 4, 2049, 7000], [1, 16383], [16384], [5, 20000, 64, 8192], [700] * 20])
def test_lookup_grad_runs_over_many_chunks(ctx, runs, width):
    """Rows that so many tokens name that their parts are added in steps: runs
    of every place against those steps, beside each other. Integers, exact;
    twice, with other tokens between."""
    count, rows = sum(runs), 2 * len(runs) + 1
    g = gen(count + width)
    tokens = (2 * torch.repeat_interleave(torch.arange(len(runs)), torch.tensor(runs)) + 1).int().to(DEV)
    E = S.Embedding(ctx, rows, width, max_tokens=count)
    for turn in range(3):
        use = tokens if turn != 1 else tokens[torch.randperm(count, generator=g, device=DEV)[: count // 2 + 1]]
        dout = torch.randint(-8, 9, (use.numel(), width), generator=g, device=DEV).float()
        dtable = torch.full((rows, width), 9.0, device=DEV)
        E.lookup_grad(use, dout, dtable)
        assert torch.equal(dtable.double(), grad_rows(use, dout, rows)[0]), turn
    ctx.check()


@pytest.mark.parametrize("rows", [3000, 100000])
@pytest.mark.parametrize("share", [[0.5], [0.97], [0.2, 0.2, 0.2], [0.1, 0.05, 0.03, 0.02]])
def test_lookup_grad_adds_in_token_order(ctx, share, rows):
    """The order of a sum is the tokens' own: values whose fp32 sum depends on
    it, as bits, for frequent rows in the middle, at the end and at the
    beginning of the table."""
    count, width = 9001, 4
    g = gen(rows + len(share))
    tokens = tokens_of(count, rows, g, empty=0.05)
    u = torch.rand(count, generator=g, device=DEV)
    for q, part in enumerate(share):
        row = (rows // 2, rows - 1, 0, 7)[q]
        tokens = torch.where((u >= 0) & (u < part), row, tokens).int()
        u = u - part
    dout = randn(count, width, g=g).float()
    few = S.Embedding(ctx, rows, width, max_tokens=count)
    dtable = torch.empty(rows, width, device=DEV)
    few.lookup_grad(tokens, dout, dtable)
    # The same tokens, sorted beforehand by a stable sort, with their rows:
    # the same runs in the same places.
    order = torch.argsort(torch.where(tokens < 0, rows, tokens), stable=True)
    again = torch.empty_like(dtable)
    few.lookup_grad(tokens[order].contiguous(), dout[order].contiguous(), again)
    assert torch.equal(dtable, again)
    ctx.check()


def test_rows_of_any_alignment(ctx):
    """Widths, strides and offsets of every remainder of a 16-byte word, for
    each operator that moves rows; nothing beside the rows is written."""
    g = gen(21)
    for dtype in (torch.bfloat16, torch.float32):
        for width in (1, 2, 3, 5, 7, 8, 9, 15, 16, 17, 23, 31, 64, 65):
            for pad, shift in ((0, 0), (1, 0), (0, 1), (3, 5), (8, 4), (7, 8)):
                rows = 11
                X, xb = strided(rows, width, dtype, pad, shift)
                X.copy_(randn(rows, width, g=g))
                tokens = torch.tensor([3, -1, 10, 0, 10], dtype=torch.int32, device=DEV)
                out, ob = strided(5, width, dtype, (pad + 3) % 9, (shift + 1) % 9)
                E = S.Embedding(ctx, rows, width, max_tokens=5)
                E.lookup(tokens, X, out)
                assert torch.equal(out, rows_at(X, tokens).to(dtype))
                outside_untouched(ob, out)
                grad, gb = strided(rows, width, dtype, pad, (shift + 3) % 9)
                E.lookup_grad(tokens[:4], out[:4], grad)
                assert torch.equal(grad, grad_rows(tokens[:4], out[:4], rows)[0].to(dtype))
                outside_untouched(gb, grad)
                R = S.Router(ctx, 4, 2, max_tokens=5)
                position = torch.tensor([[0, 7], [2, -1], [9, 4], [-1, -1], [1, 3]], dtype=torch.int32, device=DEV)
                xs, sb = strided(rows, width, dtype, (pad + 1) % 9, (shift + 2) % 9)
                R.dispatch(position, out, xs)
                for t, j in ((0, 0), (0, 1), (1, 0), (2, 0), (2, 1), (4, 0), (4, 1)):
                    assert torch.equal(xs[position[t, j]], out[t])
                outside_untouched(sb, xs)
                back, bb = strided(5, width, dtype, pad, (shift + 5) % 9)
                one = torch.ones(5, 2, device=DEV)
                R.combine(position, one, xs, back)
                assert torch.equal(back, rows_at(xs, position).sum(1).to(dtype))
                outside_untouched(bb, back)
                dY, yb = strided(rows, width, dtype, pad, (shift + 7) % 9)
                dw = torch.empty(5, 2, device=DEV)
                R.combine_grad(position, one, xs, out, dY, dw)
                assert torch.equal(dY[7], out[0]) and torch.equal(dY[2], out[1])
                outside_untouched(yb, dY)
    ctx.check()


def test_lookup_and_its_gradient_are_adjoint(ctx):
    """<lookup(X), G> = <X, lookup_grad(G)>: exact in integers."""
    g = gen(8)
    tokens = tokens_of(700, 90, g)
    X = torch.randint(-8, 9, (90, 50), generator=g, device=DEV).float()
    G = torch.randint(-8, 9, (700, 50), generator=g, device=DEV).float()
    E = S.Embedding(ctx, 90, 50, max_tokens=700)
    out, dX = torch.empty_like(G), torch.empty_like(X)
    E.lookup(tokens, X, out, scale=2.0)
    E.lookup_grad(tokens, G, dX, scale=2.0)
    assert (out.double() * G.double()).sum() == (X.double() * dX.double()).sum()


def test_offsets_past_32_bits(ctx):
    """The last rows of a table of over 2^31 elements."""
    rows, width = 530000, 4104
    assert rows * width > 2 ** 31
    table = torch.empty(rows, width, device=DEV, dtype=torch.bfloat16)
    table[-3:] = torch.randn(3, width, device=DEV)
    tokens = torch.tensor([rows - 1, -1, rows - 3, rows - 1], dtype=torch.int32, device=DEV)
    out = torch.empty(4, width, device=DEV, dtype=torch.bfloat16)
    E = S.Embedding(ctx, rows, width, max_tokens=4)
    E.lookup(tokens, table, out)
    assert torch.equal(out[[0, 2, 3]], table[[-1, -3, -1]]) and not out[1].any()
    E.lookup_grad(tokens, out, table, accumulate=False)
    assert torch.equal(table[-1], (2 * out[0].float()).bfloat16()) and torch.equal(table[-3], out[2])
    assert not table[-2].any() and not table[0].any() and not table[rows // 2].any()


def test_tokens_past_the_table_are_left_out_and_reported(ctx):
    tokens = torch.tensor([0, 7, 3, 2 ** 31 - 1, -2 ** 31, 2], dtype=torch.int32, device=DEV)
    table = torch.ones(4, 24, device=DEV)
    out = torch.full((6, 24), 5.0, device=DEV)
    E = S.Embedding(ctx, 4, 24, max_tokens=6)
    E.lookup(tokens, table, out)
    assert out[:, 0].tolist() == [1, 0, 1, 0, 0, 1]
    with pytest.raises(S.SpmvbError) as e:
        ctx.check()
    assert e.value.status == 1 and "out of range" in str(e.value)
    ctx.check()  # cleared
    grad = torch.empty(4, 24, device=DEV)
    E.lookup_grad(tokens, torch.ones(6, 24, device=DEV), grad)
    assert grad[:, 0].tolist() == [1, 0, 1, 1]
    with pytest.raises(S.SpmvbError):
        ctx.check()


# ---- routing --------------------------------------------------------------------

ROUTES = [
    # experts, k, score, renormalise, groups, kept, top, bias
    (1, 1, "softmax", True, 1, 1, 1, False), (2, 2, "sigmoid", False, 1, 1, 1, True), (8, 2, "softmax", True, 1, 1, 1, False),
    (60, 4, "softmax", False, 1, 1, 1, False), (64, 6, "softmax", False, 8, 3, 1, False),
    (160, 6, "softmax", True, 8, 3, 2, True), (256, 8, "sigmoid", True, 8, 4, 2, True), (256, 8, "sigmoid", False, 8, 4, 2, False),
    (96, 32, "sigmoid", True, 32, 16, 2, True), (33, 10, "softmax", True, 3, 2, 2, False), (500, 5, "softmax", False, 5, 5, 1, True),
    (1024, 32, "sigmoid", True, 2, 1, 1, True), (24, 24, "softmax", True, 1, 1, 1, True), (128, 1, "softmax", True, 1, 1, 1, False),
    (1020, 8, "sigmoid", True, 17, 5, 2, True), (330, 5, "softmax", False, 11, 4, 1, False)]


def route_case(tokens, experts, bias, dtype, seed, masks=True, ties=True):
    g = gen(seed)
    l = randn(tokens, experts, g=g) * 2
    if ties:  # logits on a coarse grid: many equal ones
        l = torch.where(torch.rand(tokens, 1, generator=g, device=DEV) < 0.3, (l * 2).round() / 2, l)
    if masks:
        l = torch.where(torch.rand(tokens, experts, generator=g, device=DEV) < 0.2, -math.inf, l)
        l[torch.rand(tokens, generator=g, device=DEV) < 0.1] = -math.inf
        if tokens > 3:
            l[1] = torch.finfo(dtype).min
            l[2, 1:] = -math.inf
    b = randn(experts, g=g) * 0.1 if bias else None
    return l.to(dtype), b


def weight_bound(logits, ref, experts):
    """fp32: the difference to the row's largest logit (half a step of up to
    `reach`), exp (2 steps), up to experts / 32 + 5 sums, a quotient and a
    product (2 steps), twice over for a quotient of two such values."""
    l = logits.double().cpu()
    fine = torch.isfinite(l)
    reach = torch.where(fine & (l.abs() < 200), l.abs(), 0.0).max().item() * 2
    return ref.abs() * 2 * (reach + experts / 32 + 16) * 2.0 ** -24 + 2.0 ** -140


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("experts,k,score,renormalise,groups,kept,top,bias", ROUTES)
@pytest.mark.parametrize("tokens", [1, 5, 131])
def test_route(ctx, tokens, experts, k, score, renormalise, groups, kept, top, bias, dtype):
    logits, b = route_case(tokens, experts, bias, dtype, experts * 7 + tokens)
    R = S.Router(ctx, experts, k, max_tokens=tokens, score=score, renormalise=renormalise, scale=2.5, groups=groups,
                 groups_kept=kept, group_top=top)
    indices = torch.full((tokens, k), 77, dtype=torch.int32, device=DEV)
    weights = torch.full((tokens, k), 77.0, device=DEV)
    offsets = torch.full((experts + 1,), 77, dtype=torch.int32, device=DEV)
    order = torch.full((tokens * k,), -77, dtype=torch.int32, device=DEV)
    position = torch.full((tokens, k), 77, dtype=torch.int32, device=DEV)
    wide = torch.full((tokens, experts + 5), float("nan"), device=DEV, dtype=dtype)
    wide[:, :experts] = logits
    R.route(wide[:, :experts], indices, weights, bias=b, offsets=offsets, order=order, position=position)
    picks = choose(logits.cpu(), None if b is None else b.cpu(), k, score, groups, kept, top)
    assert torch.equal(indices.cpu(), picks)
    ref = weights_of(logits.cpu(), picks, score, renormalise, 2.5)
    check(weights, ref, weight_bound(logits, ref, experts), "weights")
    o, by, at = plan_of(picks, experts)
    assert offsets.tolist() == o and position.flatten().tolist() == at
    assert order.tolist() == by + [-77] * (tokens * k - len(by))  # rows behind the last are left
    ctx.check()
    # The choice alone, without its plan.
    again, w2 = torch.empty_like(indices), torch.empty_like(weights)
    R.route(logits, again, w2, bias=b)
    assert torch.equal(again, indices) and torch.equal(w2.view(torch.int32), weights.view(torch.int32))


@pytest.mark.parametrize("score,bias", [("softmax", True), ("sigmoid", True)])
def test_route_between_scores_that_fp32_does_not_tell_apart(ctx, score, bias):
    """score + bias of the best two differ by about 2^-40 of a score: the
    larger one is chosen first, as in 64 bits."""
    experts, tokens = 64, 400
    g = gen(3)
    l = randn(tokens, experts, g=g).cpu()
    b = torch.zeros(experts)
    # A bias that fp32 holds, and a logit chosen so that the sums nearly meet.
    b[1::2] = 0.125
    if score == "sigmoid":
        s = torch.sigmoid(l.double())
        meet = (s[:, 1::2] + 0.125).clamp(0.2, 0.95)
        l[:, 0::2] = torch.log(meet / (1 - meet)).float()
        l[:, 1::2] = torch.log((meet - 0.125) / (1 - meet + 0.125)).float()
    R = S.Router(ctx, experts, 8, max_tokens=tokens, score=score)
    indices = torch.empty(tokens, 8, dtype=torch.int32, device=DEV)
    weights = torch.empty(tokens, 8, device=DEV)
    R.route(l.to(DEV), indices, weights, bias=b.to(DEV))
    assert torch.equal(indices.cpu(), choose(l, b, 8, score))


@pytest.mark.parametrize("experts,k,score,groups,kept,top", [
    (256, 8, "sigmoid", 8, 4, 2), (256, 8, "softmax", 1, 1, 1), (60, 4, "softmax", 1, 1, 1), (64, 8, "sigmoid", 8, 3, 1),
    (96, 32, "sigmoid", 32, 16, 2), (1020, 8, "sigmoid", 17, 5, 2)])
@pytest.mark.parametrize("levels,bias", [(1, True), (3, True), (3, False), (40, True)])
def test_route_of_equal_scores(ctx, experts, k, score, groups, kept, top, levels, bias):
    """Logits of few values, as of a router that begins at zero: every choice
    is among equals, and goes to the lowest index."""
    tokens = 1500  # enough for rows to share a warp
    g = gen(experts + levels)
    logits = torch.randint(0, levels, (tokens, experts), generator=g, device=DEV).float() / 8
    b = torch.randint(0, levels, (experts,), generator=g, device=DEV).float() / 16 if bias else None
    R = S.Router(ctx, experts, k, max_tokens=tokens, score=score, groups=groups, groups_kept=kept, group_top=top)
    indices = torch.empty(tokens, k, dtype=torch.int32, device=DEV)
    weights = torch.empty(tokens, k, device=DEV)
    R.route(logits, indices, weights, bias=b)
    some = slice(0, 150)
    assert torch.equal(indices[some].cpu(), choose(logits[some].cpu(), None if b is None else b.cpu(), k, score, groups, kept, top))


def test_route_many_tokens_is_route_few_tokens(ctx):
    """Rows that share a warp choose as rows that have one, ragged ends and
    all; both with their plans."""
    for experts, k, bias in ((64, 8, False), (100, 6, True), (16, 2, True), (128, 16, False)):
        logits, b = route_case(1300, experts, bias, torch.float32, experts)
        R = S.Router(ctx, experts, k, max_tokens=1300, score="sigmoid")
        whole = [torch.empty(1300, k, dtype=torch.int32, device=DEV), torch.empty(1300, k, device=DEV)]
        part = [torch.empty_like(t) for t in whole]
        R.route(logits, *whole, bias=b)
        for a in range(0, 1300, 433):
            R.route(logits[a:a + 433], part[0][a:a + 433], part[1][a:a + 433], bias=b)
        assert torch.equal(whole[0], part[0])
        check(whole[1], part[1].double(), weight_bound(logits, part[1].double(), experts), "weights")


def test_route_no_tokens(ctx):
    R = S.Router(ctx, 12, 3, max_tokens=0)
    none = dict(device=DEV, dtype=torch.int32)
    offsets = torch.full((13,), 5, **none)
    R.route(torch.empty(0, 12, device=DEV), torch.empty(0, 3, **none), torch.empty(0, 3, device=DEV), offsets=offsets,
            order=torch.empty(0, **none), position=torch.empty(0, 3, **none))
    assert not offsets.any()
    R.route_grad(torch.empty(0, 12, device=DEV), torch.empty(0, 3, **none), torch.empty(0, 3, device=DEV),
                 torch.empty(0, 12, device=DEV))


def test_first_calls_on_a_stream_of_their_own(ctx):
    """A handle's scratch is ready when create returns, also for a stream that
    does not wait for the default one."""
    g = gen(33)
    tokens = tokens_of(9000, 700, g)
    dout = torch.randint(-8, 9, (9000, 16), generator=g, device=DEV).float()
    want = grad_rows(tokens, dout, 700)[0]
    idx = torch.randint(0, 500, (9000, 4), generator=g, device=DEV, dtype=torch.int32)
    o, by, at = plan_of(idx, 500)
    side = torch.cuda.Stream()
    dtable = torch.empty(700, 16, device=DEV)
    plan = [torch.empty(n, dtype=torch.int32, device=DEV) for n in (501, 36000, 36000)]
    torch.cuda.synchronize()
    for turn in range(5):
        E, R = S.Embedding(ctx, 700, 16, max_tokens=9000), S.Router(ctx, 500, 4, max_tokens=9000)
        E.lookup_grad(tokens, dout, dtable, stream=side)
        R.plan(idx, *plan, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(dtable.double(), want)
        assert plan[0].tolist() == o and plan[1].tolist() == by and plan[2].tolist() == at


def test_route_rows_without_scores(ctx):
    """NaN and infinities: an unavailable expert under the sigmoid, a row
    without scores under the softmax."""
    nan, inf = math.nan, math.inf
    rows = torch.tensor([[nan, 1, 2, 0], [inf, 1, 2, 0], [-inf, -inf, -inf, -inf], [nan] * 4, [-inf, 3, -inf, nan],
                         [0.0, -0.0, 0.0, -0.0]], device=DEV)
    for bias in (None, torch.tensor([0.0, -inf, 0.5, nan], device=DEV)):
        for score in ("softmax", "sigmoid"):
            R = S.Router(ctx, 4, 2, max_tokens=6, score=score)
            indices = torch.empty(6, 2, dtype=torch.int32, device=DEV)
            weights = torch.empty(6, 2, device=DEV)
            R.route(rows, indices, weights, bias=bias)
            picks = choose(rows.cpu(), None if bias is None else bias.cpu(), 2, score)
            assert torch.equal(indices.cpu(), picks), (score, bias)
            w = weights.cpu()
            for t in range(6):
                if score == "softmax" and (torch.isnan(rows[t]).any() or (rows[t] == inf).any()):
                    assert torch.isnan(w[t]).all() and (picks[t] == -1).all()
                elif (picks[t] >= 0).any():
                    assert abs(w[t].sum().item() - 1) < 1e-6
                else:
                    assert not w[t].any()
    # dlogits: NaN where the row has no scores, 0 where nothing is chosen.
    for score, expect in (("softmax", [True, True, False, True, True, False]), ("sigmoid", [False] * 6)):
        R = S.Router(ctx, 4, 2, max_tokens=6, score=score)
        R.route(rows, indices, weights)
        d = torch.empty_like(rows)
        R.route_grad(rows, indices, torch.ones(6, 2, device=DEV), d)
        assert torch.isnan(d).all(1).tolist() == expect and not d[2].any()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("experts,k,score,renormalise,groups,kept,top,bias", ROUTES)
def test_route_grad(ctx, experts, k, score, renormalise, groups, kept, top, bias, dtype):
    tokens = 67
    logits, b = route_case(tokens, experts, bias, dtype, experts * 11)
    R = S.Router(ctx, experts, k, max_tokens=tokens, score=score, renormalise=renormalise, scale=2.5, groups=groups,
                 groups_kept=kept, group_top=top)
    picks = choose(logits.cpu(), None if b is None else b.cpu(), k, score, groups, kept, top)
    dw = randn(tokens, k, g=gen(2))
    base = torch.full((tokens, experts + 3), float("nan"), device=DEV, dtype=dtype)
    R.route_grad(logits, picks.to(DEV), dw, base[:, :experts])
    assert torch.isnan(base[:, experts:]).all()
    # d weights / d logits by automatic differentiation of the 64-bit formula; masked logits far below the rest.
    l = torch.where(torch.isfinite(logits.cpu()), logits.cpu().double(), -1e4).requires_grad_()
    weights_of(l, picks, score, renormalise, 2.5).backward(dw.cpu().double())
    ref = torch.where(torch.isfinite(logits.cpu()), l.grad, 0.0)
    # Each entry is a share (at most 1, relative error as of a weight) times differences of dw, all in fp32.
    size = 2.5 * dw.abs().sum(1, keepdim=True).cpu().double() * torch.ones_like(ref)
    share = torch.where(torch.isfinite(logits.cpu()), torch.ones_like(ref), 0.0)
    bound = weight_bound(logits, share, experts) * size
    f = torch.finfo(dtype)
    check(base[:, :experts], ref, bound + f.eps / 2 * (ref.abs() + bound) + f.smallest_normal * f.eps / 2, "route_grad")
    ctx.check()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_route_grad_against_differences(ctx, score, renormalise):
    """(w(l + h d) - w(l - h d)) / 2h along a direction d, from the kernel's
    own weights. With |d|_inf <= 1, h = 2^-6 and weights of at most 1, the third
    derivative along d is below 8 (a softmax's or sigmoid's derivatives are
    bounded by 1, its three factors by 8 together): h^2 / 6 * 8 = 3.3e-4 of
    truncation, 2^-20 / 2h of rounding."""
    tokens, experts, k = 50, 6, 6
    g = gen(12)
    logits = randn(tokens, experts, g=g)
    d = torch.rand(tokens, experts, generator=g, device=DEV) * 2 - 1
    R = S.Router(ctx, experts, k, max_tokens=tokens, score=score, renormalise=renormalise)

    def weights_by_expert(l):
        indices = torch.empty(tokens, k, dtype=torch.int32, device=DEV)
        w = torch.empty(tokens, k, device=DEV)
        R.route(l, indices, w)
        return indices, w, torch.zeros(tokens, experts, device=DEV).scatter_(1, indices.long(), w).double()

    h = 2.0 ** -6
    indices, _, _ = weights_by_expert(logits)
    slope = (weights_by_expert(logits + h * d)[2] - weights_by_expert(logits - h * d)[2]) / (2 * h)
    dw = randn(tokens, k, g=g)
    dl = torch.empty_like(logits)
    R.route_grad(logits, indices, dw, dl)
    along = (dl.double() * d.double()).sum(1)
    expect = (slope.gather(1, indices.long()) * dw.double()).sum(1)
    assert ((along - expect).abs() <= (3.4e-4 + 2.0 ** -20 / (2 * h) + 1e-5) * dw.abs().sum(1)).all()


@pytest.mark.parametrize("experts,k,tokens,skew", [(1, 1, 1, 0), (8, 2, 3, 0), (256, 8, 700, 3), (1024, 4, 3000, 0),
                                                   (511, 3, 1500, 1), (512, 3, 1500, 1), (4, 32, 2100, 0), (64, 8, 0, 0),
                                                   (100, 8, 33000, 2), (257, 4, 70000, 0), (1024, 1, 5000, 1)])
def test_plan(ctx, experts, k, tokens, skew):
    """Any indices: absent, repeated in a row, all one expert's."""
    g = gen(experts + tokens)
    u = torch.rand(tokens, k, generator=g, device=DEV)
    idx = (u ** (1 + skew) * experts).int().clamp(max=experts - 1)
    idx[torch.rand(tokens, k, generator=g, device=DEV) < 0.15] = -1
    R = S.Router(ctx, max(experts, k), k, max_tokens=tokens + 1)
    offsets = torch.full((R.experts + 1,), 9, dtype=torch.int32, device=DEV)
    order = torch.full((tokens * k,), -9, dtype=torch.int32, device=DEV)
    position = torch.full((tokens, k), 9, dtype=torch.int32, device=DEV)
    for turn in range(2):  # the scratch is left as it was found
        R.plan(idx, offsets, order, position)
        o, by, at = plan_of(idx, R.experts)
        assert offsets.tolist() == o and position.flatten().tolist() == at
        assert order[:len(by)].tolist() == by and (order[len(by):] == -9).all()
        idx = idx.flip(0).contiguous() if turn == 0 else idx
        order.fill_(-9)
    ctx.check()


# ---- exchange ----------------------------------------------------------------------

EXCHANGES = [(1, 1, 1, 0, 0), (1, 4, 2048, 0, 0), (7, 2, 33, 3, 1), (50, 8, 1000, 8, 8), (33, 3, 4096, 0, 0), (200, 6, 16, 0, 0),
             (0, 2, 64, 0, 0), (9, 32, 129, 0, 2)]


def exchange_case(ctx, tokens, k, seed):
    g = gen(seed)
    R = S.Router(ctx, 40, k, max_tokens=tokens)
    idx = torch.rand(tokens, 40, generator=g, device=DEV).argsort(1)[:, :k].int().contiguous()
    idx[torch.rand(tokens, k, generator=g, device=DEV) < 0.2] = -1
    offsets = torch.empty(41, dtype=torch.int32, device=DEV)
    order = torch.empty(tokens * k, dtype=torch.int32, device=DEV)
    position = torch.empty(tokens, k, dtype=torch.int32, device=DEV)
    R.plan(idx, offsets, order, position)
    return R, position, torch.rand(tokens, k, generator=g, device=DEV), g


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("tokens,k,width,pad,shift", EXCHANGES)
def test_dispatch_and_combine(ctx, dtype, tokens, k, width, pad, shift):
    R, position, w, g = exchange_case(ctx, tokens, k, tokens + k)
    rows = tokens * k + 2
    X, _ = strided(tokens, width, dtype, pad, shift)
    X.copy_(randn(tokens, width, g=g))
    out, base = strided(rows, width, dtype, pad, shift)
    R.dispatch(position, X, out)
    there = position >= 0
    ref = torch.full((rows, width), float("nan"), device=DEV, dtype=dtype)
    ref[position[there].long()] = X.repeat_interleave(k, 0)[there.flatten()]
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out.nan_to_num(), ref.nan_to_num())
    outside_untouched(base, out)

    Y, _ = strided(rows, width, dtype, pad, shift, fill=0.0)
    Y.copy_(randn(rows, width, g=g))
    y, ybase = strided(tokens, width, dtype, pad, shift)
    R.combine(position, w, Y, y)
    terms = rows_at(Y, position) * w.double().unsqueeze(-1)
    ref = terms.sum(1)
    check(y, ref, allowed(ref, terms.abs().sum(1), k, dtype), "combine")
    outside_untouched(ybase, y)
    R.dispatch_grad(position, Y, y)
    ref = rows_at(Y, position).sum(1)
    check(y, ref, allowed(ref, rows_at(Y, position).abs().sum(1), k, dtype), "dispatch_grad")
    ctx.check()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("tokens,k,width,pad,shift", EXCHANGES)
def test_combine_grad(ctx, dtype, tokens, k, width, pad, shift):
    R, position, w, g = exchange_case(ctx, tokens, k, tokens + k)
    rows = tokens * k + 2
    Y, _ = strided(rows, width, dtype, pad, shift)
    Y.copy_(randn(rows, width, g=g))
    dout, _ = strided(tokens, width, dtype, pad, shift)
    dout.copy_(randn(tokens, width, g=g))
    dY, base = strided(rows, width, dtype, pad, shift)
    dw = torch.full((tokens, k), 7.0, device=DEV)
    R.combine_grad(position, w, Y, dout, dY, dw)
    there = position >= 0
    ref = torch.full((rows, width), float("nan"), device=DEV, dtype=torch.float64)
    ref[position[there].long()] = (dout.double().unsqueeze(1) * w.double().unsqueeze(-1))[there]
    check(dY, ref, allowed(ref, ref.abs(), 1, dtype), "dY")
    outside_untouched(base, dY)
    terms = rows_at(Y, position) * dout.double().unsqueeze(1)
    check(dw, terms.sum(2), allowed(terms.sum(2), terms.abs().sum(2), width, torch.float32), "dweights")
    ctx.check()


def test_combine_matches_the_sparse_product(ctx):
    """combine is Y times the k-per-row matrix of the weights, as
    DeviceMatrix.spmm computes it (within the bound of both)."""
    import numpy as np
    R, position, w, g = exchange_case(ctx, 300, 4, 9)
    Y = randn(1200, 64, g=g)
    out = torch.empty(300, 64, device=DEV)
    R.combine(position, w, Y, out)
    there = (position >= 0).cpu().numpy()
    rowptr = np.concatenate([[0], np.cumsum(there.sum(1))]).astype(np.int32)
    A = S.CsrMatrix(300, 1200, rowptr, position.cpu().numpy()[there], w.cpu().double().numpy()[there])
    M = S.DeviceMatrix(ctx, A, S.F32)
    ref = torch.empty(300, 64, device=DEV)
    M.spmm(Y, ref, 64, tile=64)
    size = (rows_at(Y, position) * w.double().unsqueeze(-1)).abs().sum(1)
    check(out, ref.double(), 2 * allowed(ref.double(), size, 4, torch.float32))
    M.close()


def test_positions_past_the_rows_are_left_out_and_reported(ctx):
    R = S.Router(ctx, 4, 2, max_tokens=2)
    position = torch.tensor([[0, 9], [-5, 2]], dtype=torch.int32, device=DEV)
    X, w = torch.ones(2, 8, device=DEV), torch.ones(2, 2, device=DEV)
    rows = torch.zeros(3, 8, device=DEV)
    for call in (lambda: R.dispatch(position, X, rows), lambda: R.combine(position, w, rows, torch.empty(2, 8, device=DEV)),
                 lambda: R.dispatch_grad(position, rows, torch.empty(2, 8, device=DEV)),
                 lambda: R.combine_grad(position, w, rows, X, torch.empty(3, 8, device=DEV), torch.empty(2, 2, device=DEV)),
                 lambda: R.plan(position, torch.empty(5, dtype=torch.int32, device=DEV),
                                torch.empty(4, dtype=torch.int32, device=DEV),
                                torch.empty(2, 2, dtype=torch.int32, device=DEV))):
        call()
        with pytest.raises(S.SpmvbError):
            ctx.check()
    assert rows[:, 0].tolist() == [1, 0, 1]


# ---- streams, graphs, repetition -----------------------------------------------------

def step(ctx, E, R, C, st, stream=None):
    """One training step of a router with experts gain[e] * tanh(x); every
    output is in `st`. The dense parts are torch's."""
    dense = lambda: torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream())  # noqa: E731
    E.lookup(st["tokens"], st["table"], st["x"], scale=2.0, stream=stream)
    with dense():
        torch.mm(st["x"], st["wr"], out=st["logits"])
    R.route(st["logits"], st["indices"], st["weights"], offsets=st["offsets"], order=st["order"], position=st["position"],
            stream=stream)
    R.dispatch(st["position"], st["x"], st["xs"], stream=stream)
    with dense():
        expert = torch.bucketize(st["rows"], st["offsets"][1:], right=True).clamp(max=st["gain"].numel() - 1)
        gain = st["gain"][expert].unsqueeze(1)
        torch.mul(torch.tanh(st["xs"]), gain, out=st["ys"])
    R.combine(st["position"], st["weights"], st["ys"], st["out"], stream=stream)
    # Loss = <out, target>: its gradient in `out` is the target.
    R.combine_grad(st["position"], st["weights"], st["ys"], st["target"], st["dys"], st["dweights"], stream=stream)
    R.route_grad(st["logits"], st["indices"], st["dweights"], st["dlogits"], stream=stream)
    with dense():
        torch.mul(st["dys"], gain * (1 - torch.tanh(st["xs"]).square()), out=st["dxs"])
    R.dispatch_grad(st["position"], st["dxs"], st["dx"], stream=stream)
    with dense():
        st["dx"].addmm_(st["dlogits"], st["wr"].t())
        torch.mm(st["x"].t(), st["dlogits"], out=st["dwr"])
    E.lookup_grad(st["tokens"], st["dx"], st["dtable"], scale=2.0, stream=stream)
    C.clip(0.5, st["norm"], stream=stream)


def step_state(ctx, seed, tokens=150, rows=70, width=48, experts=12, k=3):
    g = gen(seed)
    f = dict(device=DEV, dtype=torch.float32)
    i = dict(device=DEV, dtype=torch.int32)
    st = {"tokens": tokens_of(tokens, rows, g), "table": randn(rows, width, g=g), "wr": randn(width, experts, g=g) * 0.2,
          "target": randn(tokens, width, g=g),
          "gain": torch.linspace(-1.0, 2.0, experts, device=DEV), "rows": torch.arange(tokens * k, **i), "x": torch.empty(tokens, width, **f), "logits": torch.empty(tokens, experts, **f),
          "indices": torch.empty(tokens, k, **i), "weights": torch.empty(tokens, k, **f),
          "offsets": torch.empty(experts + 1, **i), "order": torch.zeros(tokens * k, **i), "position": torch.empty(tokens, k, **i)}
    for n in ("xs", "ys", "dys", "dxs"):
        st[n] = torch.zeros(tokens * k, width, **f)
    for n in ("out", "dx"):
        st[n] = torch.empty(tokens, width, **f)
    st |= {"dweights": torch.empty(tokens, k, **f), "dlogits": torch.empty(tokens, experts, **f),
           "dtable": torch.empty(rows, width, **f), "dwr": torch.empty(width, experts, **f), "norm": torch.empty(1, **f)}
    E = S.Embedding(ctx, rows, width, max_tokens=tokens)
    R = S.Router(ctx, experts, k, max_tokens=tokens, score="softmax")
    return st, E, R, S.GradClip(ctx, [st["dtable"], st["dwr"]])


def test_a_training_step_against_automatic_differentiation(ctx):
    """Lookup, router, exchange, their gradients and the clipping, together,
    against the same step in 64 bits differentiated by torch. The fp32 chain
    has fewer than 2,000 roundings of terms of order 10 into gradients of
    order 1 to 100: 2^-24 * 2000 = 1.2e-4 of a tensor's largest magnitude."""
    st, E, R, C = step_state(ctx, 4)
    allow = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        step(ctx, E, R, C, st)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = allow
    table, wr = st["table"].double().cpu().requires_grad_(), st["wr"].double().cpu().requires_grad_()
    tokens, picks = st["tokens"].cpu().long(), st["indices"].cpu()
    x = torch.where((tokens >= 0)[:, None], table[tokens.clamp(min=0)], 0.0) * 2.0
    w = weights_of(x @ wr, picks, "softmax", True, 1.0)
    out = torch.tanh(x) * (w * st["gain"].double().cpu()[picks.long()]).sum(1, keepdim=True)
    (out * st["target"].double().cpu()).sum().backward()
    assert torch.equal(picks, choose(st["logits"].cpu(), None, 3, "softmax"))
    norm = math.sqrt(table.grad.square().sum() + wr.grad.square().sum())
    factor = min(1.0, 0.5 / (norm + 1e-6))
    assert abs(st["norm"].item() - norm) <= 1.2e-4 * norm
    for got, ref in ((st["out"], out.detach()), (st["dtable"], table.grad * factor), (st["dwr"], wr.grad * factor)):
        assert (got.double().cpu() - ref).abs().max() <= 1.2e-4 * ref.abs().max()
    ctx.check()


def test_graph_replays_and_other_streams_give_the_same_bits(ctx):
    st, E, R, C = step_state(ctx, 6)
    step(ctx, E, R, C, st)
    torch.cuda.synchronize()
    want = {n: t.clone() for n, t in st.items()}
    side = torch.cuda.Stream()
    for n in ("dtable", "out", "dlogits", "norm", "order"):
        st[n].zero_()
    torch.cuda.synchronize()
    step(ctx, E, R, C, st, stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(st[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(ctx, E, R, C, st)
    other, *_ = step_state(ctx, 7)
    for n in ("tokens", "table", "target"):
        st[n].copy_(other[n])
    graph.replay()
    torch.cuda.synchronize()
    mid = {n: t.clone() for n, t in st.items()}
    for n in ("dtable", "out", "dlogits", "norm"):
        st[n].zero_()
    step(ctx, E, R, C, st)
    torch.cuda.synchronize()
    assert all(torch.equal(st[n], mid[n]) for n in st)
    assert not torch.equal(mid["dtable"], want["dtable"])


# ---- refusals ------------------------------------------------------------------------

def test_refusals(ctx):
    f32 = dict(device=DEV)
    tok = torch.zeros(4, dtype=torch.int32, **f32)
    E = S.Embedding(ctx, 8, 16, max_tokens=4)
    table, out = torch.zeros(8, 16, **f32), torch.zeros(4, 16, **f32)
    big = torch.zeros(12, 16, **f32)
    bad = [
        lambda: E.lookup(tok.long(), table, out), lambda: E.lookup(tok.cpu(), table, out),
        lambda: E.lookup(tok, table.half(), out), lambda: E.lookup(tok, table[:, ::2], out),
        lambda: E.lookup(tok, table[:7], out), lambda: E.lookup(tok, table, out[:3]),
        lambda: E.lookup(tok, table.t(), out), lambda: E.lookup(tok, table.int(), out),
        lambda: E.lookup(tok, table, torch.zeros(1, 16, **f32).expand(4, 16)),
        lambda: E.lookup(torch.zeros(8, dtype=torch.int32, **f32)[::2], table, out),
        lambda: E.lookup_grad(tok, out, table.half()), lambda: E.lookup_grad(tok, out, table.double()),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    five = torch.zeros(5, dtype=torch.int32, **f32)
    R = S.Router(ctx, 8, 2, max_tokens=4)
    idx = torch.zeros(4, 2, dtype=torch.int32, **f32)
    w = torch.zeros(4, 2, **f32)
    logits = torch.zeros(4, 8, **f32)
    status = [
        lambda: E.lookup(tok, big[:8], big[6:10]),                            # out overlaps the table
        lambda: E.lookup_grad(five, torch.zeros(5, 16, **f32), table),        # more than max_tokens
        lambda: R.route(logits, idx, idx.view(torch.float32)),                # outputs share memory
        lambda: R.plan(torch.zeros(5, 2, dtype=torch.int32, **f32), torch.zeros(9, dtype=torch.int32, **f32),
                       torch.zeros(10, dtype=torch.int32, **f32), torch.zeros(10, dtype=torch.int32, **f32)),
        lambda: R.combine(idx, w, big[:8], big[4:8]),
        lambda: S.Router(ctx, 8, 9, max_tokens=1), lambda: S.Router(ctx, 8, 2, max_tokens=-1),
        lambda: S.Embedding(ctx, 0, 4, max_tokens=1), lambda: S.Embedding(ctx, 4, 4, max_tokens=-1),
    ]
    for call in status:
        with pytest.raises(S.SpmvbError) as e:
            call()
        assert e.value.status == 1
    for call in [lambda: R.route(logits, idx, w, offsets=torch.zeros(9, dtype=torch.int32, **f32)),
                 lambda: R.route(logits.double(), idx, w), lambda: R.route(logits, idx[:3], w),
                 lambda: R.route(logits, idx, w, bias=torch.zeros(7, **f32)),
                 lambda: R.dispatch(idx, torch.zeros(4, 8, **f32), torch.zeros(9, 16, **f32)),
                 lambda: R.dispatch(idx[:3], torch.zeros(4, 8, **f32), torch.zeros(9, 8, **f32)),
                 lambda: R.combine(idx, w.half(), big[:8], out)]:
        with pytest.raises(ValueError):
            call()
    # Column ranges of one buffer do not overlap.
    both = torch.zeros(8, 32, **f32)
    E.lookup(torch.arange(8, dtype=torch.int32, **f32), both[:, :16], both[:, 16:])
    torch.cuda.synchronize()
