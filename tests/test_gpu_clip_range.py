"""Norms and clipping of values near the ends of their types' ranges, against
exact arithmetic (fractions and integer square roots). Bounds: the norm is the
fp32 rounding (half a step) of an fp64 one (1e-12 for its sums); a clipped value
is a product with a factor, three roundings in fp32 (fp64 for doubles, and
1e-12), and one to its type."""
from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

import spmvbench_b200 as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEPS = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# Half the smallest subnormal.
HALF_LEAST = {torch.float64: Fraction(1, 2 ** 1075), torch.float32: Fraction(1, 2 ** 150), torch.float16: Fraction(1, 2 ** 25),
              torch.bfloat16: Fraction(1, 2 ** 134)}


def exact_norm(values):
    """sqrt of the sum of squares of Fractions, to 200 bits."""
    total = sum(v * v for v in values)
    if total == 0:
        return Fraction(0)
    shift = 2 * 1400  # squares of subnormals are above 2^-2148
    return Fraction(math.isqrt(int(total * 2 ** shift)), 2 ** (shift // 2))


def clip_and_compare(ctx, tensors, limit):
    """limit: a number, or a share of the norm given as a Fraction."""
    before = [[Fraction(x) for x in t.double().tolist()] for t in tensors]
    n = exact_norm([x for b in before for x in b])
    if isinstance(limit, Fraction):
        limit = float(n * limit) if n * limit < 2 ** 1024 else math.inf
    norm = torch.full((1,), -1.0, device=DEV)
    C = S.GradClip(ctx, tensors)
    C.norm(norm)
    if n > Fraction(torch.finfo(torch.float32).max) * (1 + Fraction(1, 2 ** 24)):
        assert norm.item() == math.inf
    else:
        assert abs(Fraction(norm.item()) - n) <= n * Fraction(2.0 ** -24 + 1e-12) + Fraction(1, 2 ** 150)
    C.clip(limit, norm, eps=0.0)
    factor = min(Fraction(1), Fraction(limit) / n) if limit < math.inf else Fraction(1)
    for t, b in zip(tensors, before):
        u = Fraction(2.0 ** -53 if t.dtype == torch.float64 else 2.0 ** -24) * 3 + Fraction(1e-12 if t.dtype == torch.float64 else 0)
        for got, x in zip(t.double().tolist(), b):
            want = x * factor
            err = abs(want) * u
            assert math.isfinite(got)
            assert abs(Fraction(got) - want) <= err + (abs(want) + err) * Fraction(HALF_STEPS[t.dtype]) + HALF_LEAST[t.dtype], \
                (got, float(want), t.dtype)


@pytest.mark.parametrize("values", [
    [1e200] * 5, [1e-200] * 5, [1e300, -1e300, 3e299], [1.7e308, 1.0], [5e-324, 1e-323], [1e-310] * 40, [1e300, 1.0, 1e-300],
    [1e150, 1e140, 1e-150], [2.0 ** 480, 2.0 ** 481, 2.0 ** -480, 2.0 ** -481], [3e-150, 1e-150, 4e-200], [0.0, 1e-250, 0.0], [2.0, 3.0]])
@pytest.mark.parametrize("limit", [Fraction(1, 4), Fraction(1, 1000003), Fraction(3, 2)])
def test_doubles_whose_squares_leave_fp64(ctx, values, limit):
    clip_and_compare(ctx, [torch.tensor(values, dtype=torch.float64, device=DEV)], limit)
    # Beside gradients of other types, which the mixed kernels sum with them.
    clip_and_compare(ctx, [torch.tensor(values, dtype=torch.float64, device=DEV), torch.tensor([1.0, -3.0], device=DEV),
                           torch.tensor([0.5] * 9, device=DEV, dtype=torch.bfloat16)], limit)


@pytest.mark.parametrize("limit", [1e-3, 1e-9, 1e300])
def test_doubles_and_factors_near_the_least(ctx, limit):
    """1e308 clipped to 1e-9: a factor of 1e-317 would have lost two thirds of
    its bits."""
    clip_and_compare(ctx, [torch.tensor([1e308, 3e307, -2e300, 1e290, 1.0], dtype=torch.float64, device=DEV)], limit)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("limit", [1.0, 1e-4, 1e-6, 1e-30, 1e30])
@pytest.mark.parametrize("count", [1, 7, 3001])
def test_factors_below_fp32s_normal_range(ctx, count, limit, kind):
    """Gradients of 1e38, finite, after a step that diverged: limit / norm is
    subnormal in fp32 or 0, the clipped values are ordinary."""
    t = torch.full((count,), 1e38, device=DEV).to(kind)
    t[count // 2] = 3e38
    clip_and_compare(ctx, [t], limit)
    mixed = [t.new_full((count,), 2e38), torch.tensor([1.0, 2e5], device=DEV, dtype=torch.float64),
             torch.tensor([6e4, 1.0], device=DEV, dtype=torch.float16)]
    clip_and_compare(ctx, mixed, limit)


def test_measuring_without_a_limit_leaves_finite_gradients(ctx):
    """max_norm = inf: the factor is 1 for every finite gradient, also where
    its squares leave fp64."""
    for v in (1e300, 1.0, 1e-300):
        t = torch.full((4,), v, device=DEV, dtype=torch.float64)
        norm = torch.zeros(1, device=DEV)
        S.GradClip(ctx, [t]).clip(math.inf, norm)
        assert torch.equal(t, torch.full_like(t, v))
        assert norm.item() == {1e300: math.inf, 1.0: 2.0, 1e-300: 0.0}[v]


def test_infinities_and_nan_beside_values_of_every_size(ctx):
    """What is not finite carries on: an infinite norm makes finite gradients 0
    and infinite ones NaN, a NaN makes all NaN."""
    for far in (1e300, 1e-300):
        for kind in (torch.float64, torch.float32):
            a = torch.tensor([far, 1.0, far], dtype=torch.float64, device=DEV)
            b = torch.tensor([math.inf, 1.0], dtype=kind, device=DEV)
            norm = torch.zeros(1, device=DEV)
            S.GradClip(ctx, [a, b]).clip(1.0, norm)
            assert norm.item() == math.inf and not a.any() and torch.isnan(b[0]) and b[1] == 0
            a = torch.tensor([far, 1.0, far], dtype=torch.float64, device=DEV)
            b = torch.tensor([math.nan, 1.0], dtype=kind, device=DEV)
            S.GradClip(ctx, [a, b]).clip(1.0, norm)
            assert torch.isnan(norm).all() and torch.isnan(a).all() and torch.isnan(b).all()
