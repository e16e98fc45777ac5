# SPDX-License-Identifier: MIT
"""The fused operators beyond plain calls: writing in place, as autograd sees it; second
derivatives."""

from __future__ import annotations

import pytest
import torch

from rmsnorm import fused

GPU = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=GPU)]


def rope_inputs(device, tokens=6, heads=2, d=16):
    torch.manual_seed(0)
    return (torch.randn(tokens, 3 * heads, d).to(device), torch.arange(tokens).to(device),
            fused.rope_table(tokens, d).to(device))


# ------------------------------------------------------------------ in place
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("with_k", [True, False])
def test_inplace_moves_the_version(device, with_k):
    packed, pos, table = rope_inputs(device)
    q, k = packed[:, :2], packed[:, 2:4] if with_k else None
    before = packed._version
    fused.qk_norm_rope_fwd(q, k, pos, table, inplace=True)
    assert packed._version > before and q._version == packed._version
    after = packed._version
    fused.qk_norm_rope_fwd(q, k, pos, table)
    assert packed._version == after


@pytest.mark.parametrize("device", DEVICES)
def test_inplace_over_a_saved_tensor_is_found(device):
    packed, pos, table = rope_inputs(device)
    w = torch.ones_like(packed[:, :2], requires_grad=True)
    loss = (w * packed[:, :2]).sum()  # saves the slice
    fused.qk_norm_rope_fwd(packed[:, :2], None, pos, table, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("leaf", [True, False])
@pytest.mark.parametrize("device", [pytest.param("cuda", marks=GPU)])
def test_inplace_on_cuda_refuses_inputs_with_gradients(device, which, leaf):
    packed, pos, table = rope_inputs(device)
    q, k = packed[:, :2].clone(), packed[:, 2:4].clone()
    t = q if which == "q" else k
    t.requires_grad_(True)
    if not leaf:
        q, k = q * 1, k * 1
    held = q.detach().clone(), k.detach().clone()
    with pytest.raises(ValueError, match="autograd"):
        fused.qk_norm_rope_fwd(q, k, pos, table, inplace=True)
    assert torch.equal(q, held[0]) and torch.equal(k, held[1])
    want = fused.qk_norm_rope_fwd(*held, pos, table)
    with torch.no_grad():
        fused.qk_norm_rope_fwd(q, k, pos, table, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("device", DEVICES)
def test_inplace_with_weights_that_train_and_in_inference_mode(device):
    packed, pos, table = rope_inputs(device)
    w = torch.ones(16, device=device, requires_grad=True)
    with torch.no_grad():
        want = fused.qk_norm_rope_fwd(packed[:, :2], packed[:, 2:4], pos, table, w, w)
        a = packed.clone()
        fused.qk_norm_rope_fwd(a[:, :2], a[:, 2:4], pos, table, w, w, inplace=True)
    assert torch.equal(a[:, :2], want[0]) and torch.equal(a[:, 2:4], want[1])
    with torch.inference_mode():
        a = packed.clone()
        fused.qk_norm_rope_fwd(a[:, :2], a[:, 2:4], pos, table, w, w, inplace=True)
        assert torch.equal(a[:, :2], want[0]) and torch.equal(a[:, 2:4], want[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_inplace_refuses_expanded_views(device, which, dim):
    """Elements that share a place would be turned more than once."""
    packed, pos, table = rope_inputs(device)
    q, k = packed[:, :2].clone(), packed[:, 2:4].clone()
    one = (q if which == "q" else k).narrow(dim, 0, 1).clone()
    wide = one.expand(6, 2, 16)
    a, b = (wide, k) if which == "q" else (q, wide)
    held = one.clone()
    with pytest.raises(ValueError, match="expanded"):
        fused.qk_norm_rope_fwd(a, b, pos, table, inplace=True)
    assert torch.equal(one, held)
    fused.qk_norm_rope_fwd(a, b, pos, table)  # as inputs they are fine
    fused.qk_norm_rope_fwd(q[:1].expand(1, 2, 16), k[:1].expand(1, 2, 16), pos[:1], table, inplace=True)


# ------------------------------------------------------------------ second derivatives
def operators(device):
    """(name, function of one tensor, that tensor): each operator with autograd."""
    torch.manual_seed(1)
    pos, table = torch.arange(6, device=device), fused.rope_table(6, 16, device=device)
    w = torch.rand(16).to(device) + 0.5

    def drop(x):
        return fused.dropout_add_rmsnorm(x, w, p=0.25, rng=(1, 2))

    def prenorm(x):
        out, h = fused.dropout_add_rmsnorm(x, w, residual=x * 2, p=0.25, rng=(1, 2), prenorm=True)
        return out + h

    def rope(x):
        q, k = fused.qk_norm_rope(x[:, :2], x[:, 2:], pos, table, w, w)
        return torch.cat([q, k], 1)

    return [("dropout", drop, torch.randn(6, 16).to(device)), ("prenorm", prenorm, torch.randn(6, 16).to(device)),
            ("rope", rope, torch.randn(6, 3, 16).to(device))]


@pytest.mark.parametrize("device,which", [
    pytest.param("cpu", 0), pytest.param("cpu", 1), *(pytest.param("cuda", i, marks=GPU) for i in range(3))])
def test_second_derivatives_are_refused(device, which):
    """Everywhere but for the host's rotary operator."""
    _, f, x = operators(device)[which]
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    c = torch.randn_like(f(a))
    want, = torch.autograd.grad((f(a) * c).sum(), a)
    out = f(b)
    got, = torch.autograd.grad((out * c).sum(), b, create_graph=True)
    assert torch.equal(got, want) and got.requires_grad
    # a penalty on the gradient beside an ordinary loss: an error, not the loss's part alone
    with pytest.raises(RuntimeError, match="second derivatives"):
        ((b * b).sum() + (got * got).sum()).backward()
    d = x.clone().requires_grad_(True)
    (f(d) * c).sum().backward(create_graph=True)  # without a second derivative all is well
    assert torch.equal(d.grad.detach(), want)


def test_second_derivatives_of_the_rotary_operator_on_the_host():
    """Central differences of the gradient, itself in 32 bits: with a step of 2^-7 rounding leaves
    about 2^-24 * 2^7 of the gradient's size and truncation a few 2^-14 of the third derivative's."""
    _, f, x = operators("cpu")[2]
    c, v = torch.randn_like(f(x)), torch.randn_like(x)

    def grad(x, **kw):
        x = x.clone().requires_grad_(True) if not x.requires_grad else x
        return torch.autograd.grad((f(x).tanh() * c).sum(), x, **kw)[0]

    x = x.requires_grad_(True)
    got, = torch.autograd.grad((grad(x, create_graph=True) * v).sum(), x)
    h, x = 2.0**-7, x.detach()
    want = (grad(x + h * v) - grad(x - h * v)) / (2 * h)
    assert (got - want).norm() < 2e-2 * want.norm()
