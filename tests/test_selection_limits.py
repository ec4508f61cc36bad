"""Sizes past int32 in the Python layer of the row-selection operators (no GPU):
refused, not taken modulo 2^32."""
from __future__ import annotations

import pytest
import torch

import spmvbench_b200 as S
from spmvbench_b200 import selection


@pytest.mark.parametrize("sizes", [(2 ** 32 + 8, 16, 4), (8, 2 ** 32 + 16, 4), (8, 16, 2 ** 32 + 4), (2 ** 31, 16, 4),
                                   (8, 16, -2 ** 32 + 4)])
def test_embedding_sizes_past_int32_are_refused(sizes):
    with pytest.raises(ValueError, match="int32"):
        S.Embedding(None, *sizes)


@pytest.mark.parametrize("fields", [dict(experts=2 ** 32 + 8, k=2), dict(experts=8, k=2 ** 32 + 2), dict(experts=8, k=2, groups=2 ** 32 + 2),
                                    dict(experts=8, k=2, groups=2, groups_kept=2 ** 32 + 1), dict(experts=8, k=2, group_top=2 ** 32 + 1)])
def test_router_specs_past_int32_are_refused(fields):
    with pytest.raises(ValueError, match="int32"):
        selection.router_spec(**fields)


def test_router_tokens_past_int32_are_refused():
    with pytest.raises(ValueError, match="int32"):
        S.Router(None, 8, 2, max_tokens=2 ** 32 + 4)


class Wide:
    """A CUDA tensor of 1 x (2^32 + 16) values, as far as the checks look."""

    is_cuda, dtype, shape = True, torch.float32, (1, 2 ** 32 + 16)

    def get_device(self):
        return 0

    def stride(self):
        return 2 ** 32 + 16, 1

    def data_ptr(self):
        return 4096


def test_rows_longer_than_int32_are_refused():
    with pytest.raises(ValueError, match="shape"):
        selection._rows(Wide(), 1, 2 ** 32 + 16, 0, "X")


@pytest.mark.parametrize("code", [S.F16, S.BF16])
def test_the_merge_product_refuses_16_bit_types_for_their_type(code):
    """An empty product, which every other argument allows."""
    lib = S.load()
    empty = lambda dtype, acc: lib.spmvb_spmv_merge_noalloc(dtype, 0, 0, 0, None, None, None, None, None, acc, None)  # noqa: E731
    assert empty(S.F32, S.F32) == 0 and empty(S.F32, S.F64) == 0
    assert empty(code, S.F32) == 1 and lib.spmvb_last_error() == b"bad dtype"
    assert empty(S.F32, code) == 1 and lib.spmvb_last_error() == b"bad accumulator dtype"
