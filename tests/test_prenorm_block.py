# SPDX-License-Identifier: MIT
"""The example block: it trains, its masks move with the step, and it serves in 8 bits."""

from __future__ import annotations

import pytest
import torch

from rmsnorm import fused
from rmsnorm.examples.prenorm_block import PrenormBlock, train

DEVICES = [pytest.param("cpu"),
           pytest.param("cuda", marks=[pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")])]


@pytest.mark.parametrize("device", DEVICES)
def test_training_and_serving(device):
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    losses, blocks, (x, positions, table, axes) = train(12, 64, 128, torch.device(device), dtype)
    assert losses[-1] < 0.6 * losses[0]
    branch, residual, served, stream = x, None, x, None
    for b in blocks:
        b.eval()
        with torch.no_grad():
            branch, residual = b(branch, residual, positions, table, axes)
        served, stream = b.prepare_serving()(served, stream, positions, table, axes)
    want = branch.float() + residual.float()
    off = (served.float() + stream.float() - want).norm() / want.norm()
    # e4m3 keeps 4 significant bits: each of four products has an error of about 2^-5 in both
    # operands, of random sign
    assert off < 0.12


@pytest.mark.parametrize("device", DEVICES)
def test_the_step_moves_the_masks(device):
    torch.manual_seed(0)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    block = PrenormBlock(128, 2, 1, 64, 256, dropout=0.5, device=device, dtype=dtype)
    x = torch.randn(16, 128, device=device).to(dtype)
    table, positions = fused.rope_table(16, 64, device=device), torch.arange(16, device=device)
    steps = [torch.tensor([i], device=device) for i in (0, 1, 0)]
    a, b, c = (block(x, None, positions, table, seed=3, step=s)[1] for s in steps)
    assert torch.equal(a, c) and not torch.equal(a, b)
    # the residual of the first norm holds dropout(x): zero where its mask drops
    h = fused.dropout_add_rmsnorm_fwd(x, p=0.5, rng=(3, 0), rng_step=steps[1])[1]
    assert torch.equal(h == 0, ~fused.dropout_mask(x.shape, 0.5, (3, 1), x.device))


def test_the_block_on_cuda_matches_the_host():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    torch.manual_seed(0)
    block = PrenormBlock(128, 2, 1, 64, 256, dropout=0.25)
    x, g = torch.randn(32, 128), torch.randn(32, 128)
    table, positions = fused.rope_table(32, 64), torch.arange(32)
    results = []
    for device in ("cpu", "cuda"):
        block = block.to(device)
        block.zero_grad()
        branch, residual = block(x.to(device), None, positions.to(device), table.to(device), seed=5)
        ((branch + residual) * g.to(device)).sum().backward()
        results.append([branch.detach(), residual.detach(), *(p.grad for p in block.parameters())])
    for a, b in zip(*results):
        assert (a.cpu() - b.cpu()).norm() <= 1e-4 * a.cpu().norm()


test_the_block_on_cuda_matches_the_host = pytest.mark.gpu(test_the_block_on_cuda_matches_the_host)
