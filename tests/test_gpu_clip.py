"""The global gradient norm and clipping against 64 bits. The squares are
summed in fp64: the norm is its fp32 rounding (half a step, and 1e-12 for the
sums); a clipped value is one fp32 product with a factor rounded to fp32,
rounded to the tensor's type."""
from __future__ import annotations

import math

import pytest
import torch

import spmvbench_b200 as S
from selection_util import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def norm_of(tensors):
    return math.sqrt(sum(t.double().square().sum().item() for t in tensors))


def expected(before, factor):
    """(values, bound) of a scaled tensor."""
    ref = before.double() * factor
    f = torch.finfo(before.dtype)
    u = 2.0 ** -53 if before.dtype == torch.float64 else 2.0 ** -24
    err = ref.abs() * 3 * u + (1e-12 * ref.abs() if before.dtype == torch.float64 else 0)
    return ref, err + f.eps / 2 * (ref.abs() + err) + f.smallest_normal * f.eps / 2


@pytest.mark.parametrize("sizes", [[1], [1, 2, 3], [16384], [16385, 7, 40000], [100] * 300, [0, 5, 0], [3_000_001, 12]])
@pytest.mark.parametrize("kinds", [[torch.float32], [torch.bfloat16], [torch.float16], [torch.float64],
                                   [torch.float32, torch.bfloat16, torch.float16, torch.float64]])
@pytest.mark.parametrize("shift", [0, 1])
def test_clip(ctx, sizes, kinds, shift):
    g = torch.Generator(device=DEV).manual_seed(len(sizes))
    tensors = [torch.randn(n + shift, generator=g, device=DEV).to(kinds[i % len(kinds)])[shift:] for i, n in enumerate(sizes)]
    before = [t.clone() for t in tensors]
    n = norm_of(before)
    C = S.GradClip(ctx, tensors)
    norm = torch.full((1,), -1.0, device=DEV)
    C.norm(norm)
    assert abs(norm.item() - n) <= n * (2.0 ** -24 + 1e-12)
    assert all(torch.equal(a, b) for a, b in zip(tensors, before))
    C.clip(2 * n + 1, norm)  # below the limit: unchanged
    assert all(torch.equal(a, b) for a, b in zip(tensors, before))
    C.clip(0.3 * n, norm)
    assert abs(norm.item() - n) <= n * (2.0 ** -24 + 1e-12)
    for t, b in zip(tensors, before):
        check(t, *expected(b, 0.3 * n / (n + 1e-6)), "clip")


def test_nothing_to_clip(ctx):
    norm = torch.full((1,), -1.0, device=DEV)
    for tensors in ([], [torch.empty(0, device=DEV)], [torch.zeros(100, device=DEV)]):
        C = S.GradClip(ctx, tensors)
        C.clip(1.0, norm)
        assert norm.item() == 0.0
        C.clip(0.0, norm, eps=0.0)
        assert norm.item() == 0.0 and all(not t.any() for t in tensors)


def test_squares_past_fp32(ctx):
    """1e30 and 1e-30: their squares leave fp32, not the sums."""
    for v in (1e30, 1e-30):
        for kind in (torch.float32, torch.bfloat16):
            t = torch.full((5000,), v, device=DEV, dtype=kind)
            n = norm_of([t])
            norm = torch.zeros(1, device=DEV)
            C = S.GradClip(ctx, [t])
            C.clip(n / 4, norm, eps=0.0)
            assert abs(norm.item() - n) <= n * (2.0 ** -24 + 1e-12)
            check(t, *expected(torch.full((5000,), v, device=DEV, dtype=kind), 0.25))


def test_norms_that_are_not_finite(ctx):
    norm = torch.zeros(1, device=DEV)
    a, b = torch.ones(10, device=DEV), torch.ones(20, device=DEV, dtype=torch.bfloat16)
    a[3] = math.nan
    S.GradClip(ctx, [a, b]).clip(1.0, norm)
    assert torch.isnan(norm).all() and torch.isnan(a).all() and torch.isnan(b).all()
    a, b = torch.ones(10, device=DEV), torch.ones(20, device=DEV, dtype=torch.bfloat16)
    a[3] = math.inf
    S.GradClip(ctx, [a, b]).clip(1.0, norm)
    assert norm.item() == math.inf and torch.isnan(a[3]) and not a[:3].any() and not b.any()
    big = torch.full((4,), 1e300, device=DEV, dtype=torch.float64)
    S.GradClip(ctx, [big]).clip(math.inf, norm)
    assert torch.equal(big, torch.full_like(big, 1e300)) or torch.isnan(big).all()


def test_same_bits_every_time_and_in_a_graph(ctx):
    g = torch.Generator(device=DEV).manual_seed(1)
    src = [torch.randn(n, generator=g, device=DEV).bfloat16() for n in (100003, 77, 5_000_000)]
    tensors = [t.clone() for t in src]
    C = S.GradClip(ctx, tensors)
    norm = torch.zeros(1, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        C.clip(1.0, norm)
    seen = []
    for run in range(4):
        for t, s in zip(tensors, src):
            t.copy_(s)
        graph.replay() if run % 2 else C.clip(1.0, norm)
        torch.cuda.synchronize()
        seen.append([norm.clone()] + [t.clone() for t in tensors])
    assert all(torch.equal(a, b) for other in seen[1:] for a, b in zip(seen[0], other))


def test_refusals(ctx):
    t = torch.zeros(100, device=DEV)
    for tensors in ([t.cpu()], [t.int()], [t.view(10, 10).t()[:, :5]]):
        with pytest.raises(ValueError):
            S.GradClip(ctx, tensors)
    for tensors in ([t, t], [t[:60], t[50:]]):
        with pytest.raises(S.SpmvbError) as e:
            S.GradClip(ctx, tensors)
        assert e.value.status == 1 and "overlap" in str(e.value)
    norm = torch.zeros(1, device=DEV)
    C = S.GradClip(ctx, [t[:50]])
    for call in (lambda: C.clip(-1.0, norm), lambda: C.clip(math.nan, norm), lambda: C.clip(1.0, norm, eps=-1.0),
                 lambda: C.clip(1.0, t[10:11])):
        with pytest.raises(S.SpmvbError) as e:
            call()
        assert e.value.status == 1
    for call in (lambda: C.clip(1.0, norm.double()), lambda: C.clip(1.0, torch.zeros(2, device=DEV)), lambda: C.norm(norm.cpu())):
        with pytest.raises(ValueError):
            call()
    moved = torch.zeros(8, device=DEV)
    C = S.GradClip(ctx, [moved])
    moved.data = torch.zeros(8, device=DEV)
    with pytest.raises(ValueError):
        C.norm(norm)
