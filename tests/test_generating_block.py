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


def peaked(device):
    """A block whose branch is that of its attention alone (its MLP gives zeros), with logits twice as
    wide as random heads' own, so that what a token reads depends on which keys it has."""
    (block,), dtype = blocks(device)
    with torch.no_grad():
        block.down.zero_()
        block.q_norm.fill_(2**0.5)
        block.k_norm.fill_(2**0.5)
    return block, dtype


def attention_off(block, x, prompt):
    """How far the generated attention branches are off the unquantised ones."""
    table = fused.rope_table(x.shape[1], 64, device=x.device)
    got = generate([block], x, prompt, table) - x.float()
    with torch.no_grad():
        want = torch.stack([sum(t.float() for t in block(s, None, torch.arange(x.shape[1], device=x.device), table)) for s in x])
    want = want - x.float()
    return float((got - want).norm() / want.norm())


# The branch is off by its two products' operands, 0.037 each, by the values' 0.026 and by its softmax:
# q and k are off by 0.037, k by 0.026 more, so a logit (0.06 of sqrt(2) sqrt(2) times a normal
# number each way) by 0.12 to 0.17, and what is read with such weights by as much. Added up: 0.27.
ATTENTION = 0.3


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("prompt,tokens", [(1, 24), (17, 40)])
def test_generated_attention_matches_the_whole_sequence(device, prompt, tokens):
    block, dtype = peaked(device)
    x = torch.randn(3, tokens, 256, device=device, generator=torch.Generator(device=device).manual_seed(3)).to(dtype)
    assert attention_off(block, x, prompt) <= ATTENTION


@pytest.mark.parametrize("mistake", ["no keys", "no values", "keys of the token before", "values of the token before",
                                     "keys of the other head", "keys turned to one position"])
def test_generated_attention_tells_mistakes(mistake, monkeypatch):
    """What the bound above is good for: each of these exceeds it."""
    from rmsnorm.examples import prenorm_block

    read, turn = fused.cache_read, fused.qk_norm_rope_fwd

    def wrong_read(*args, **kw):
        k, v = read(*args, **kw)
        if mistake == "no keys":
            k = torch.zeros_like(k)
        elif mistake == "no values":
            v = torch.zeros_like(v)
        elif mistake == "keys of the token before":
            k = k.roll(1, 0)
        elif mistake == "values of the token before":
            v = v.roll(1, 0)
        elif mistake == "keys of the other head":
            k = k.flip(1)
        return k, v

    def wrong_turn(q, k, positions, *args, **kw):
        if mistake == "keys turned to one position":
            turn(q, k.clone(), positions, *args, **kw)
            positions = positions * 0
            return turn(q.clone(), k, positions, *args, **kw)
        return turn(q, k, positions, *args, **kw)

    block, dtype = peaked("cpu")
    x = torch.randn(3, 24, 256, generator=torch.Generator().manual_seed(3)).to(dtype)
    wrong = type("wrong", (), {n: staticmethod(getattr(fused, n)) for n in fused.__all__})
    wrong.cache_read, wrong.qk_norm_rope_fwd = staticmethod(wrong_read), staticmethod(wrong_turn)
    monkeypatch.setattr(prenorm_block, "fused", wrong)
    table = fused.rope_table(24, 64)
    got = generate([block], x, 7, table) - x
    monkeypatch.undo()
    with torch.no_grad():
        want = torch.stack([sum(t.float() for t in block(s, None, torch.arange(24), table)) for s in x]) - x
    assert (got - want).norm() > ATTENTION * want.norm()


@pytest.mark.parametrize("device", DEVICES)
def test_sequences_without_new_tokens(device):
    """Some, or all, have none in a step: the others' results are what they are alone."""
    (block,), dtype = blocks(device)
    table = fused.rope_table(16, 64, device=device)
    x = torch.randn(5, 256, device=device, generator=torch.Generator(device=device).manual_seed(4)).to(dtype)

    def step(layer, sequences, new, x):
        positions, slots = sequences.extend(new)
        assert positions.dtype == slots.dtype == torch.int64
        branch, residual = layer(x, None, new, slots, positions, table)
        return branch.float() + residual

    alone, among = (PagedSequences(n, 8, 4, device) for n in (1, 3))
    one, three = block.prepare_generating(alone), block.prepare_generating(among)
    want = step(one, alone, [3], x[:3]), step(one, alone, [2], x[3:])
    got = step(three, among, [0, 3, 0], x[:3]), step(three, among, [0, 2, 0], x[3:])
    # the same sums in the same order, but for the library's attention
    assert all((a - b).norm() <= 0.05 * a.norm() for a, b in zip(want, got))
    assert step(three, among, [0, 0, 0], x[:0]).shape == (0, 256)
