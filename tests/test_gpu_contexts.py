"""Handles that outlive their context."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import spmvbench_b200 as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("first", ["context", "handles"])
def test_handles_outlive_their_context(first):
    own = S.Context(0)
    E, R = S.Embedding(own, 6, 8, max_tokens=3000), S.Router(own, 6, 2, max_tokens=3)
    t = torch.randn(6, 8, device=DEV)
    C = S.GradClip(own, [t])
    A = S.generate(2, seed=3, scale_rows=500)
    M = S.DeviceMatrix(own, A, S.F64)
    if first == "context":
        own.close()
    # Indices past the end are still left out: the words that take their reports live on.
    tokens = torch.tensor([5, 9, -1, 0], dtype=torch.int32, device=DEV)
    out = torch.full((4, 8), 7.0, device=DEV)
    E.lookup(tokens, t, out)
    assert torch.equal(out[[0, 3]], t[[5, 0]]) and not out[1:3].any()
    grad = torch.empty(6, 8, device=DEV)
    E.lookup_grad(tokens.repeat(600), out.repeat(600, 1), grad)
    assert torch.allclose(grad[5], 600 * t[5], rtol=1e-4) and not grad[1:5].any()
    logits = torch.randn(3, 6, device=DEV)
    indices, weights = torch.empty(3, 2, dtype=torch.int32, device=DEV), torch.empty(3, 2, device=DEV)
    R.route(logits, indices, weights)
    assert torch.equal(indices.long(), logits.topk(2, 1).indices)
    R.dispatch(torch.tensor([[0, 8], [1, -1], [2, 3]], dtype=torch.int32, device=DEV), out[:3], grad)
    assert torch.equal(grad[:4], out[[0, 1, 2, 2]])
    norm = torch.zeros(1, device=DEV)
    C.norm(norm)
    assert abs(norm.item() - t.double().norm().item()) <= 2.0 ** -23 * norm.item()
    x = S.generate_vector(1, A.n)
    y = M.spmv_host(x, S.CSR_SCALAR)
    assert np.allclose(y, csr_product(A, x), rtol=1e-12, atol=1e-12)
    for h in (E, R, C, M):
        h.close()
    own.close()


def csr_product(A, x):
    y = np.zeros(A.m)
    np.add.at(y, np.repeat(np.arange(A.m), np.diff(A.rowptr)), A.values * x[A.colind])
    return y
