"""Row-selection operators without a GPU: refusals of the C entry points and
of the Python layer, and the plain forms that the GPU tests compare with."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

import spmvbench_b200 as S
from selection_util import choose, plan_of, weights_of
from spmvbench_b200 import selection


@pytest.mark.parametrize("fields,what", [
    (dict(experts=0, k=1), "experts"), (dict(experts=1025, k=1), "experts"), (dict(experts=8, k=0), "k must"),
    (dict(experts=64, k=33), "k must"), (dict(experts=8, k=9), "k must"), (dict(experts=8, k=2, groups=3), "groups"),
    (dict(experts=66, k=2, groups=33), "groups"), (dict(experts=8, k=2, groups=0), "groups"),
    (dict(experts=8, k=2, groups=4, groups_kept=5), "groups_kept"), (dict(experts=8, k=2, groups=4, groups_kept=0), "groups_kept"),
    (dict(experts=8, k=3, groups=4, groups_kept=1), "k must"), (dict(experts=8, k=2, group_top=3), "group_top"),
    (dict(experts=8, k=2, scale=math.inf), "scale"), (dict(experts=8, k=2, scale=math.nan), "scale")])
def test_router_specs_that_are_refused(fields, what):
    with pytest.raises(S.SpmvbError) as e:
        selection.router_spec(**fields)
    assert e.value.status == 1 and what in str(e.value)


def test_router_specs_that_are_taken():
    for fields in (dict(experts=1, k=1), dict(experts=1024, k=32), dict(experts=256, k=8, score="sigmoid", groups=8, groups_kept=4,
                                                                       group_top=2, scale=2.5), dict(experts=96, k=32, groups=32)):
        selection.router_spec(**fields)
    with pytest.raises(ValueError):
        selection.router_spec(8, 2, score="tanh")
    with pytest.raises(TypeError):
        selection.router_spec(8, 2.5)


def test_null_handles_and_arguments_give_a_status():
    lib = S.load()
    out = C.c_void_p()
    spec = selection.router_spec(8, 2)
    calls = [
        lambda: lib.spmvb_embedding_create(None, 4, 4, 4, C.byref(out)),
        lambda: lib.spmvb_embedding_lookup(None, 0, 1, None, 1.0, None, 4, None, 4, None),
        lambda: lib.spmvb_embedding_lookup_grad(None, 0, 1, None, 1.0, None, 4, 0, None, 4, 0, None),
        lambda: lib.spmvb_router_check(None),
        lambda: lib.spmvb_router_create(None, C.byref(spec), 4, C.byref(out)),
        lambda: lib.spmvb_router_route(None, 0, 1, None, 8, None, None, None, None, None, None, None),
        lambda: lib.spmvb_router_route_grad(None, 0, 1, None, 8, None, None, None, 8, None),
        lambda: lib.spmvb_router_plan(None, 1, None, None, None, None, None),
        lambda: lib.spmvb_router_dispatch(None, 0, 1, 8, None, None, 8, 2, None, 8, None),
        lambda: lib.spmvb_router_dispatch_grad(None, 0, 1, 8, None, 2, None, 8, None, 8, None),
        lambda: lib.spmvb_router_combine(None, 0, 1, 8, None, None, 2, None, 8, None, 8, None),
        lambda: lib.spmvb_router_combine_grad(None, 0, 1, 8, None, None, 2, None, 8, None, 8, None, 8, None, None),
        lambda: lib.spmvb_clip_create(None, 0, None, None, None, C.byref(out)),
        lambda: lib.spmvb_clip_norm(None, None, None),
        lambda: lib.spmvb_clip_run(None, 1.0, 0.0, None, None),
    ]
    for call in calls:
        assert call() == 1
        assert lib.spmvb_last_error()
    for destroy in (lib.spmvb_embedding_destroy, lib.spmvb_router_destroy, lib.spmvb_clip_destroy):
        assert destroy(None) == 0


def test_matrices_refuse_16_bit_types():
    """The sparse matrix entry points take fp32 and fp64 only."""
    lib = S.load()
    for code in (S.F16, S.BF16):
        assert lib.spmvb_spmv_merge_noalloc(code, 1, 1, 0, None, None, None, None, None, S.F32, None) == 1


def test_tensors_that_are_refused_before_the_c_call():
    t = torch.zeros(4, 8)
    for call in (lambda: selection._rows(t, 4, 8, 0, "t"), lambda: selection._flat(t, S.F32, 32, 0, "t"),
                 lambda: selection._rows(None, 4, 8, 0, "t"), lambda: selection._flat([1.0], S.F32, 1, 0, "t")):
        with pytest.raises(ValueError, match="CUDA"):
            call()


class FakeCuda:
    """What the checks read of a CUDA tensor."""

    def __init__(self, t, device=0):
        self.t, self.device = t, device
        self.is_cuda, self.dtype, self.shape = True, t.dtype, t.shape

    def get_device(self):
        return self.device

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_strides_shapes_devices_and_types_that_are_refused():
    rows = lambda t, *a, device=0, **k: selection._rows(FakeCuda(t, device), *a, 0, "t", **k)  # noqa: E731
    t = torch.zeros(4, 8)
    assert rows(t, 4, 8) == (S.F32, 8, t.data_ptr()) and rows(t[:, 1:5], 4, 4) == (S.F32, 8, t.data_ptr() + 4)
    assert rows(t[::2], None, 8)[1] == 16 and rows(t[:1].expand(1, 8), 1, 8)[1] == 8 and rows(t[:, :1], 4, 1)[1] == 8
    for bad in (lambda: rows(t, 3, 8), lambda: rows(t, 4, 7), lambda: rows(t.t(), 8, 4), lambda: rows(t[:, ::2], 4, 4),
                lambda: rows(t[0], 4, 8), lambda: rows(t[:1].expand(4, 8), 4, 8), lambda: rows(t.int(), 4, 8),
                lambda: rows(t.double(), 4, 8), lambda: rows(t, 4, 8, device=1)):
        with pytest.raises(ValueError):
            bad()
    flat = lambda t, n, device=0: selection._flat(FakeCuda(t, device), selection.I32, n, 0, "t")  # noqa: E731
    i = torch.zeros(6, dtype=torch.int32)
    assert flat(i.view(2, 3), 6) == i.data_ptr()
    for bad in (lambda: flat(i, 5), lambda: flat(i.long(), 6), lambda: flat(i[::2], 3), lambda: flat(i, 6, device=1)):
        with pytest.raises(ValueError):
            bad()


def test_counts_past_int32_are_refused():
    class Long(FakeCuda):
        shape = (2 ** 31, 8)

        def __init__(self):
            super().__init__(torch.zeros(1, 8))
            self.shape = (2 ** 31, 8)

        def numel(self):
            return 2 ** 31

    with pytest.raises(ValueError):
        selection._flat(Long(), S.F32, 2 ** 31, 0, "t")
    with pytest.raises(ValueError):
        selection._rows(Long(), None, 8, 0, "t")


def test_plain_forms_by_hand():
    l = torch.tensor([[1.0, 3.0, 3.0, 0.0], [-math.inf, 2.0, -math.inf, -math.inf], [-math.inf] * 4])
    assert choose(l, None, 2, "softmax").tolist() == [[1, 2], [1, -1], [-1, -1]]
    assert choose(l, None, 2, "softmax", 2, 1, 2).tolist() == [[1, 0], [1, -1], [-1, -1]]  # e + e^3 against e^3 + 1
    assert choose(l, torch.tensor([1.0, 0, 0, 0]), 1, "sigmoid").tolist() == [[0], [1], [-1]]
    w = weights_of(l, choose(l, None, 2, "softmax"), "softmax", True, 3.0)
    assert torch.allclose(w, torch.tensor([[1.5, 1.5], [3.0, 0.0], [0.0, 0.0]]).double())
    assert plan_of(torch.tensor([[1, 0], [-1, 1], [1, 2]]), 3) == ([0, 1, 4, 5], [1, 0, 3, 4, 5], [1, 0, -1, 2, 3, 4])


def test_route_gradient_formula_against_differences():
    """The 64-bit weights' automatic derivative against central differences
    (h = 1e-5: truncation below 1e-9, rounding below 1e-10 of a weight)."""
    torch.manual_seed(0)
    l = torch.randn(5, 7, dtype=torch.float64)
    picks = choose(l, None, 3, "softmax")
    for score in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            x = l.clone().requires_grad_()
            d = torch.randn_like(l)
            dw = torch.randn(5, 3, dtype=torch.float64)
            weights_of(x, picks, score, renormalise, 1.0).backward(dw)
            h = 1e-5
            diff = (weights_of(l + h * d, picks, score, renormalise, 1.0) - weights_of(l - h * d, picks, score, renormalise, 1.0))
            assert abs(((diff / (2 * h)) * dw).sum() - (x.grad * d).sum()) < 1e-8
