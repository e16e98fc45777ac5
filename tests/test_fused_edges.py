# SPDX-License-Identifier: MIT
"""Calls of the fused operators at the edges of what they accept, on the host and on CUDA."""

from __future__ import annotations

import pytest
import torch

from rmsnorm import fused

GPU = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=GPU)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lead", [(), (5,), (2, 3), (2, 1, 3), (0, 3), (2, 0)])
@pytest.mark.parametrize("d", [16, 6])  # the vectorised kernels, the scalar ones
def test_k_without_heads(device, lead, d):
    """As k = None, with an empty k_out and dk; a weight of k's has a gradient of zeros."""
    torch.manual_seed(0)
    q, dq = torch.randn(*lead, 2, d, device=device), torch.randn(*lead, 2, d, device=device)
    k, w = q[..., :0, :], torch.ones(d, device=device)
    pos, table = torch.zeros(lead, dtype=torch.int64, device=device), fused.rope_table(4, d, device=device)
    want, _ = fused.qk_norm_rope_fwd(q, None, pos, table, w)
    got, none = fused.qk_norm_rope_fwd(q, k, pos, table, w, w)
    assert torch.equal(got, want) and none.shape == k.shape
    want = fused.qk_norm_rope_bwd(q, None, pos, table, dq, None, w)
    got = fused.qk_norm_rope_bwd(q, k, pos, table, dq, k, w, w)
    assert torch.equal(got[0], want[0]) and got[1].shape == k.shape and torch.equal(got[2], want[2])
    assert torch.equal(got[3], torch.zeros_like(w))
    if device == "cpu" or len(lead) < 2:  # on CUDA a view of several leading dimensions has to collapse
        a = q.clone()
        fused.qk_norm_rope_fwd(a, a[..., :0, :], pos, table, w, inplace=True)
        assert torch.equal(a, fused.qk_norm_rope_fwd(q, None, pos, table, w)[0])


@pytest.mark.parametrize("which", range(3))
def test_under_non_strict_export_on_the_host(which):
    """Non-strict export runs the Python code: the host's operators are exported as the PyTorch
    operations they consist of."""
    torch.manual_seed(0)
    w, pos, table = torch.rand(16) + 0.5, torch.arange(6), fused.rope_table(6, 16)

    class Quant(torch.nn.Module):
        def forward(self, x):
            q, s, h = fused.rmsnorm_quant_fwd(x, w, residual=x * 2)
            return q.float(), s, h

    class Drop(torch.nn.Module):
        def forward(self, x):
            return fused.dropout_add_rmsnorm_fwd(x, w, p=0.25, rng=(1, 2), store_rstd=True)

    class Rope(torch.nn.Module):
        def forward(self, x):
            return fused.qk_norm_rope_fwd(x[:, :2], x[:, 2:], pos, table, w, w)

    module = (Quant, Drop, Rope)[which]()
    x = torch.randn(6, 3, 16)
    program = torch.export.export(module, (x,), strict=False)
    for s, t in zip(program.module()(x + 1), module(x + 1)):
        assert torch.equal(s, t)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("quant_dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("n", [256, 257, 300])
def test_infinite_values_in_eight_bits(device, quant_dtype, n):
    """An infinite y makes its scale infinite and its finite neighbours 0; itself it is infinity /
    infinity, NaN in e4m3 and 0 in int8. An infinite h makes its own y NaN and the rest of its row 0."""
    torch.manual_seed(0)
    x, w = torch.randn(9, n, device=device), torch.ones(n, device=device)
    w[70] = float("inf")
    for group in (None, 64):
        q, s, _ = fused.rmsnorm_quant_fwd(x, w, quant_dtype=quant_dtype, group_size=group)
        plain, t, _ = fused.rmsnorm_quant_fwd(x, quant_dtype=quant_dtype, group_size=group)
        here = slice(None) if group is None else slice(64, 128)
        at = s if group is None else s[:, 1]
        assert (at == float("inf")).all()
        q = q.float()
        assert (q[:, 70].isnan() if quant_dtype != torch.int8 else q[:, 70] == 0).all()
        q[:, 70] = 0
        assert (q[:, here] == 0).all()
        if group:
            assert torch.equal(s[:, [0, 2, 3]], t[:, [0, 2, 3]]) and torch.equal(q[:, 128:], plain.float()[:, 128:])
        y = x.clone()
        y[4, 70] = float("-inf")
        q, s, _ = fused.rmsnorm_quant_fwd(y, quant_dtype=quant_dtype, group_size=group)
        assert torch.equal(s[[0, 8]], t[[0, 8]])
        at = s[4] if group is None else s[4, 1]
        assert at.isnan()
        if group:
            assert (s[4, [0, 2, 3]] == 2.0**-126).all() and (q[4, 128:].float() == 0).all()
