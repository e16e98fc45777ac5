# SPDX-License-Identifier: MIT
"""The example block as it generates (block-scaled products and a quantised cache, with the norm
and the rotary positions between them) and as it trains with block-scaled products."""

from __future__ import annotations

import pytest
import torch

from rmsnorm import fused
from rmsnorm.examples.prenorm_block import PagedSequences, PrenormBlock, generate, train

DEVICES = [pytest.param("cpu"),
           pytest.param("cuda", marks=[pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")])]


def blocks(device, n=1, hidden=256, **kw):
    torch.manual_seed(0)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    return [PrenormBlock(hidden, 4, 2, 64, 2 * hidden, i, device=device, dtype=dtype, **kw).eval() for i in range(n)], dtype


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("prompt,tokens", [(1, 6), (17, 21), (40, 41)])
def test_generation_matches_the_whole_sequence(device, prompt, tokens):
    """Token by token through the cache against all at once without quantisation. A product's two
    operands are each off by at most 2^-4 of a value, 0.037 together in the mean of random values;
    cached keys and values by 0.026 each. Four products and the cache, added up: 0.2 a block, and
    what is off goes through the next one once more."""
    layers, dtype = blocks(device, 2)
    x = torch.randn(3, tokens, 256, device=device).to(dtype)
    table = fused.rope_table(tokens, 64, device=device)
    got = generate(layers, x, prompt, table)
    for s in range(3):
        branch, residual = x[s], None
        with torch.no_grad():
            for b in layers:
                branch, residual = b(branch, residual, torch.arange(tokens, device=device), table)
        want = branch.float() + residual
        assert (got[s] - want).norm() <= 0.4 * want.norm()


@pytest.mark.parametrize("device", DEVICES)
def test_a_token_does_not_depend_on_what_it_is_batched_with(device):
    """Prompts together or a token at a time, alone or beside other sequences of other lengths: the
    cache holds the same, so the last token sees the same."""
    layers, dtype = blocks(device)
    table = fused.rope_table(40, 64, device=device)
    x = torch.randn(2, 24, 256, device=device).to(dtype)
    whole, steps, alone = generate(layers, x, 24, table), generate(layers, x, 3, table), generate(layers, x[1:], 24, table)
    for a, b in ((whole, steps), (whole[1:], alone)):
        # the products' and the attention's sums in another order flip some of the next roundings to
        # 8 bits, by a step of 2^-3 of the value each
        assert (a - b).norm() <= 0.05 * a.norm()


def test_pages():
    s = PagedSequences(2, 5, 4)
    positions, slots = s.extend([5, 1])
    assert positions.tolist() == [0, 1, 2, 3, 4, 0] and len(set(slots.tolist())) == 6
    positions, slots = s.extend([0, 4])
    assert positions.tolist() == [1, 2, 3, 4] and s.lengths == [5, 5]
    table, starts = s.table()
    assert table.shape == (2, 2) and starts.tolist() == [0, 5, 10] and s.total_pages == 5
    assert len(set(table.flatten().tolist())) == 4
    with pytest.raises(IndexError):
        s.extend([8, 0])


@pytest.mark.parametrize("device", DEVICES)
def test_training_with_block_scaled_products(device):
    """Runs, and its gradients are those of the unquantised block within the operands' rounding."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    losses, _, _ = train(3, 64, 128, torch.device(device), dtype, block_scaled=True)
    assert all(torch.isfinite(torch.tensor(losses)))
    grads = []
    x = torch.randn(48, 256, device=device, generator=torch.Generator(device=device).manual_seed(1)).to(dtype)
    g = torch.randn(48, 256, device=device, generator=torch.Generator(device=device).manual_seed(2))
    table = fused.rope_table(48, 64, device=device)
    for scaled in (False, True):
        (block,), _ = blocks(device, block_scaled=scaled)
        branch, residual = block(x, None, torch.arange(48, device=device), table)
        ((branch.float() + residual) * g).sum().backward()
        grads.append([p.grad.float() for p in block.parameters()])
    for plain, eight in zip(*grads):
        # the error of up to eight products in a row, 0.037 each
        assert (plain - eight).norm() <= 0.3 * plain.norm()
