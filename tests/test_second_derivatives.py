# SPDX-License-Identifier: MIT
"""rmsnorm()'s gradients cannot be differentiated again on CUDA, and say so; on the host they can."""

from __future__ import annotations

import pytest
import torch

import rmsnorm

GPU = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


def function(device, residual):
    torch.manual_seed(0)
    w, b = (torch.rand(32, device=device) + 0.5).requires_grad_(True), torch.randn(32, device=device)

    def f(x):
        if not residual:
            return rmsnorm.rmsnorm(x, w, b)
        out, h = rmsnorm.rmsnorm(x, w, b, residual=x * 2, prenorm=True)
        return out + h

    return f, w, torch.randn(5, 32).to(device), torch.randn(5, 32).to(device)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("device", [pytest.param("cuda", marks=GPU)])
def test_second_derivatives_on_cuda_are_refused(device, residual):
    f, w, x, c = function(device, residual)
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    want = torch.autograd.grad((f(a) * c).sum(), (a, w))
    got = torch.autograd.grad((f(b) * c).sum(), (b, w), create_graph=True)
    assert all(torch.equal(s, t) for s, t in zip(got, want))
    for g in got:
        with pytest.raises(RuntimeError, match="second derivatives"):
            ((b * b).sum() + (g * g).sum()).backward(retain_graph=True)


@pytest.mark.parametrize("residual", [False, True])
def test_second_derivatives_on_the_host(residual):
    """Against the formula's, differentiated by PyTorch in 64 bits; a second derivative of fp32
    terms of size about 1 to 10 is good to 1e-4 of its norm."""
    f, w, x, c = function("cpu", residual)

    def formula(x):
        h = x * 3 if residual else x
        out = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.detach().double() + b
        return out + h if residual else out

    torch.manual_seed(0)
    torch.rand(32)
    b = torch.randn(32).double()
    results = []
    for g, dt in ((f, torch.float32), (formula, torch.float64)):
        t = x.to(dt).requires_grad_(True)
        first, = torch.autograd.grad((g(t).tanh() * c.to(dt)).sum(), t, create_graph=True)
        results.append(torch.autograd.grad((first * first).sum(), t)[0].double())
    assert (results[0] - results[1]).norm() < 1e-4 * results[1].norm()
