"""GradClip beside torch's optimizers: gradients that have been replaced since
the handle was made."""
from __future__ import annotations

import pytest
import torch

import spmvbench_b200 as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def model():
    torch.manual_seed(0)
    net = torch.nn.Linear(40, 30, device=DEV)
    return net, list(net.parameters()), torch.optim.SGD(net.parameters(), lr=0.1)


def backward(net, scale):
    (net(torch.ones(5, 40, device=DEV)).square().sum() * scale).backward()


def test_replaced_gradients_are_refused(ctx):
    net, parameters, optimizer = model()
    backward(net, 1.0)
    C = S.GradClip(ctx, [p.grad for p in parameters], parameters)
    norm = torch.zeros(1, device=DEV)
    C.clip(0.5, norm)
    optimizer.zero_grad()  # set_to_none
    for call in (lambda: C.clip(0.5, norm), lambda: C.norm(norm)):
        with pytest.raises(ValueError, match="parameter 0"):
            call()
    backward(net, 2.0)
    before = [p.grad.clone() for p in parameters]
    with pytest.raises(ValueError, match="another tensor"):
        C.clip(0.5, norm)
    assert all(torch.equal(p.grad, b) for p, b in zip(parameters, before))
    S.GradClip(ctx, [p.grad for p in parameters], parameters).clip(0.5, norm)
    assert abs(norm.item() - torch.cat([b.flatten() for b in before]).double().norm().item()) <= 2.0 ** -22 * norm.item()
    for p, b in zip(parameters, before):
        assert torch.allclose(p.grad, b * (0.5 / (norm + 1e-6)), rtol=1e-6, atol=0)


def test_gradients_zeroed_in_place_are_clipped(ctx):
    net, parameters, optimizer = model()
    backward(net, 1.0)
    C = S.GradClip(ctx, [p.grad for p in parameters], parameters)
    norm = torch.zeros(1, device=DEV)
    for turn in range(3):
        optimizer.zero_grad(set_to_none=False)
        backward(net, 1.0 + turn)
        whole = torch.cat([p.grad.flatten() for p in parameters]).double().norm().item()
        C.clip(0.5, norm)
        clipped = torch.cat([p.grad.flatten() for p in parameters]).double().norm().item()
        # fp32: a factor and a product of two roundings each, and 1e-6 of eps.
        assert abs(norm.item() - whole) <= 2.0 ** -23 * whole and abs(clipped - min(0.5, whole)) <= 0.5 * (4 * 2.0 ** -24) + 1e-6


def test_parameters_that_do_not_fit_the_tensors_are_refused(ctx):
    net, parameters, _ = model()
    backward(net, 1.0)
    with pytest.raises(ValueError, match="2 tensors of 1 parameters"):
        S.GradClip(ctx, [p.grad for p in parameters], parameters[:1])
    with pytest.raises(ValueError, match="parameter 0"):
        S.GradClip(ctx, [p.grad for p in parameters], parameters[::-1])
