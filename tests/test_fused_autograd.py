# SPDX-License-Identifier: MIT
"""The fused operators beyond plain calls: writing in place, as autograd sees it."""

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
