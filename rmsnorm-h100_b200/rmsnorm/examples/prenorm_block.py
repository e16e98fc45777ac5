# SPDX-License-Identifier: MIT
"""A pre-norm transformer block on the fused operators, as it trains and as it serves.

Training: the branch that a sublayer leaves goes through dropout, joins the residual stream
and is normalised in one operator (`dropout_add_rmsnorm`); q and k are normalised per head and
turned by their positions, as views of the packed projection, in one more (`qk_norm_rope`).
Serving: the norm leaves 8-bit values with a scale per token (`rmsnorm_quant_fwd`) for 8-bit
products. The products and the attention between them are PyTorch's.
Generating: the same with a scale for every block of 128 and the framework's own products
(`block_mm`), the turned keys and the values in the pages of an 8-bit cache (`cache_write`,
`cache_read`); the attention between them is PyTorch's. `block_scaled=True` trains with such
products (`block_linear`) too.

    python -m rmsnorm.examples.prenorm_block --steps 20
"""

from __future__ import annotations

import argparse
from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from .. import fused


class PrenormBlock(torch.nn.Module):
    """Attention (grouped heads) and MLP. `layer` numbers the block: it chooses its masks."""

    def __init__(self, hidden: int, q_heads: int, k_heads: int, head_dim: int, mlp: int, layer: int = 0, dropout: float = 0.1,
                 device=None, dtype=None, block_scaled: bool = False):
        super().__init__()
        self.q_heads, self.k_heads, self.head_dim = q_heads, k_heads, head_dim
        self.layer, self.dropout = layer, dropout
        self._linear = fused.block_linear if block_scaled else _linear
        kw = dict(device=device, dtype=dtype)

        def matrix(n_out: int, n_in: int) -> torch.nn.Parameter:
            return torch.nn.Parameter(torch.randn(n_out, n_in, **kw) * n_in**-0.5)

        self.norm1 = torch.nn.Parameter(torch.ones(hidden, device=device))
        self.norm2 = torch.nn.Parameter(torch.ones(hidden, device=device))
        self.q_norm = torch.nn.Parameter(torch.ones(head_dim, device=device))
        self.k_norm = torch.nn.Parameter(torch.ones(head_dim, device=device))
        self.qkv = matrix((q_heads + 2 * k_heads) * head_dim, hidden)
        self.out = matrix(hidden, q_heads * head_dim)
        self.up = matrix(mlp, hidden)
        self.down = matrix(hidden, mlp)

    def _attention(self, packed: Tensor, positions: Tensor, table: Tensor, axes, inplace: bool) -> Tensor:
        """packed: [tokens, (q_heads + 2 k_heads) head_dim] of one sequence."""
        d, hq, hk = self.head_dim, self.q_heads, self.k_heads
        n = packed.shape[0]
        q = packed[:, : hq * d].view(n, hq, d)
        k = packed[:, hq * d: (hq + hk) * d].view(n, hk, d)
        v = packed[:, (hq + hk) * d:].view(n, hk, d)
        if inplace:
            fused.qk_norm_rope_fwd(q, k, positions, table, self.q_norm, self.k_norm, axes, inplace=True)
        else:
            q, k = fused.qk_norm_rope(q, k, positions, table, self.q_norm, self.k_norm, axes)
        y = torch.nn.functional.scaled_dot_product_attention(
            q.transpose(0, 1)[None], k.transpose(0, 1)[None], v.transpose(0, 1)[None], is_causal=True, enable_gqa=True)
        return y[0].transpose(0, 1).reshape(n, hq * d)

    def forward(self, branch: Tensor, residual: Optional[Tensor], positions: Tensor, table: Tensor, axes=None, seed: int = 0,
                step: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        """(branch, residual) of the next block; the residual stream is kept in fp32. `step`, an
        int64 tensor of one element, moves the masks on from one training step to the next."""
        p = self.dropout if self.training else 0.0
        # a mask of its own for every place in the model; `step` counts in the low 32 bits
        at = (2 * self.layer) << 32
        h, residual = fused.dropout_add_rmsnorm(
            branch, self.norm1, residual=residual, p=p, rng=(seed, at), residual_dtype=torch.float32, prenorm=True, rng_step=step)
        branch = self._linear(self._attention(self._linear(h, self.qkv), positions, table, axes, False), self.out)
        h, residual = fused.dropout_add_rmsnorm(
            branch, self.norm2, residual=residual, p=p, rng=(seed, at + (1 << 32)), residual_dtype=torch.float32, prenorm=True,
            rng_step=step)
        return self._linear(torch.nn.functional.silu(self._linear(h, self.up)), self.down), residual

    @torch.no_grad()
    def prepare_serving(self) -> "ServingBlock":
        return ServingBlock(self)

    @torch.no_grad()
    def prepare_generating(self, sequences: "PagedSequences", kept: torch.dtype = torch.float8_e4m3fn) -> "GeneratingBlock":
        return GeneratingBlock(self, sequences, kept)


def _linear(x: Tensor, w: Tensor) -> Tensor:
    return x @ w.t()


def _quantise_rows(w: Tensor) -> Tuple[Tensor, Tensor]:
    """A weight matrix in e4m3 with a scale per row (per output)."""
    s = w.float().abs().amax(1, keepdim=True).clamp_min(1e-30) / 448.0
    return (w.float() / s).to(torch.float8_e4m3fn), s


def _product(q: Tensor, s: Tensor, w: Tuple[Tensor, Tensor], dtype: torch.dtype) -> Tensor:
    """(q s) (w_q w_s)^T: an 8-bit product on CUDA, a 32-bit one of the same values on the host."""
    if q.is_cuda:
        return torch._scaled_mm(q, w[0].t(), scale_a=s[:, None], scale_b=w[1].t(), out_dtype=dtype)
    return ((q.float() * s[:, None]) @ (w[0].float() * w[1]).t()).to(dtype)


class ServingBlock:
    """The block with its two normalised products in 8 bits."""

    def __init__(self, block: PrenormBlock):
        self.block = block
        self.qkv, self.up = _quantise_rows(block.qkv), _quantise_rows(block.up)

    @torch.no_grad()
    def __call__(self, branch: Tensor, residual: Optional[Tensor], positions: Tensor, table: Tensor, axes=None):
        b, dtype = self.block, branch.dtype
        q, s, residual = fused.rmsnorm_quant_fwd(branch, b.norm1, residual=residual, residual_dtype=torch.float32)
        branch = b._attention(_product(q, s, self.qkv, dtype), positions, table, axes, True) @ b.out.t()
        q, s, residual = fused.rmsnorm_quant_fwd(branch, b.norm2, residual=residual, residual_dtype=torch.float32)
        return torch.nn.functional.silu(_product(q, s, self.up, dtype)) @ b.down.t(), residual


class PagedSequences:
    """Which pages of the caches hold which sequence's tokens: the same for every layer."""

    def __init__(self, sequences: int, pages: int, page_size: int, device=None):
        self.page_size, self.device = page_size, device
        self.free = list(range(pages))
        self.pages: List[List[int]] = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences

    @property
    def total_pages(self) -> int:
        return len(self.free) + sum(len(p) for p in self.pages)

    def extend(self, new: Sequence[int]) -> Tuple[Tensor, Tensor]:
        """Room for new[s] more tokens of sequence s: (their positions, their slots), sequence by
        sequence."""
        at, slots = [], []
        for s, n in enumerate(new):
            first, last = self.lengths[s], self.lengths[s] + n
            while len(self.pages[s]) * self.page_size < last:
                self.pages[s].append(self.free.pop())
            at += range(first, last)
            slots += [self.pages[s][t // self.page_size] * self.page_size + t % self.page_size for t in range(first, last)]
            self.lengths[s] = last
        return tuple(torch.tensor(t, dtype=torch.int64, device=self.device) for t in (at, slots))

    def table(self) -> Tuple[Tensor, Tensor]:
        """(page table, starts) as `cache_read` takes them."""
        wide = max(1, max(len(p) for p in self.pages))
        starts = torch.tensor([0] + self.lengths).cumsum(0)
        rows = [p + [-1] * (wide - len(p)) for p in self.pages]
        return torch.tensor(rows, dtype=torch.int32, device=self.device), starts.to(dtype=torch.int32, device=self.device)


class GeneratingBlock:
    """The block with all its products in 8 bits, a scale for every block of 128, and its keys and
    values in an 8-bit cache."""

    def __init__(self, block: PrenormBlock, sequences: PagedSequences, kept: torch.dtype):
        self.block, self.sequences = block, sequences
        self.qkv, self.out, self.up, self.down = (
            fused.block_quantize(w, 128) for w in (block.qkv, block.out, block.up, block.down))
        lead = (sequences.total_pages, sequences.page_size, block.k_heads)
        device = block.qkv.device
        self.cache = (*(torch.zeros(*lead, block.head_dim, device=device).to(kept) for _ in range(2)),
                      *(torch.zeros(lead, device=device) for _ in range(2)))

    @torch.no_grad()
    def __call__(self, branch: Tensor, residual: Optional[Tensor], new: Sequence[int], slots: Tensor, positions: Tensor,
                 table: Tensor, axes=None):
        """new[s] tokens of sequence s, sequence by sequence, which `PagedSequences.extend` made room
        for."""
        b, dtype = self.block, branch.dtype
        d, hq, hk, n = b.head_dim, b.q_heads, b.k_heads, branch.shape[0]
        q8, s, residual = fused.rmsnorm_quant_fwd(branch, b.norm1, residual=residual, group_size=128,
                                                  residual_dtype=torch.float32, scales_column_major=True)
        packed = fused.block_mm(q8, s, *self.qkv, out_dtype=dtype)
        q, k, v = (packed[:, i * d: j * d].view(n, j - i, d) for i, j in ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk)))
        fused.qk_norm_rope_fwd(q, k, positions, table, b.q_norm, b.k_norm, axes, inplace=True)
        fused.cache_write(k, v, *self.cache, slots)
        pages, starts = self.sequences.table()
        lengths = self.sequences.lengths
        k, v = fused.cache_read(*self.cache, pages, starts, sum(lengths), dtype)
        ys, at_q, at_k = [], 0, 0
        for m, length in zip(new, lengths):
            # a new token sees all before it
            seen = torch.ones(m, length, dtype=torch.bool, device=q.device).tril(length - m)
            y = torch.nn.functional.scaled_dot_product_attention(
                q[at_q: at_q + m].transpose(0, 1)[None], k[at_k: at_k + length].transpose(0, 1)[None],
                v[at_k: at_k + length].transpose(0, 1)[None], attn_mask=seen, enable_gqa=True)
            ys.append(y[0].transpose(0, 1).reshape(m, hq * d))
            at_q, at_k = at_q + m, at_k + length
        y8, s = fused.block_quantize(torch.cat(ys), scales_column_major=True)
        branch = fused.block_mm(y8, s, *self.out, out_dtype=dtype, power_of_two=True)
        q8, s, residual = fused.rmsnorm_quant_fwd(branch, b.norm2, residual=residual, group_size=128,
                                                  residual_dtype=torch.float32, scales_column_major=True)
        h8, s = fused.block_quantize(torch.nn.functional.silu(fused.block_mm(q8, s, *self.up, out_dtype=dtype)),
                                     scales_column_major=True)
        return fused.block_mm(h8, s, *self.down, out_dtype=dtype, power_of_two=True), residual


@torch.no_grad()
def generate(blocks, x: Tensor, prompt: int, table: Tensor, page_size: int = 16):
    """Runs x [sequences, tokens, hidden] through the blocks as generation does: the first `prompt`
    tokens of every sequence at once, then one token of each at a time; the sums of branch and
    residual, [sequences, tokens, hidden] in fp32."""
    count, tokens = x.shape[:2]
    sequences = PagedSequences(count, count * -(-tokens // page_size), page_size, x.device)
    layers = [b.prepare_generating(sequences) for b in blocks]
    out = []
    for first, last in [(0, prompt)] + [(t, t + 1) for t in range(prompt, tokens)]:
        new = [last - first] * count
        positions, slots = sequences.extend(new)
        branch, residual = x[:, first:last].flatten(0, 1), None
        for layer in layers:
            branch, residual = layer(branch, residual, new, slots, positions, table)
        out.append((branch.float() + residual).view(count, last - first, -1))
    return torch.cat(out, 1)


def train(steps: int, tokens: int, hidden: int, device, dtype, layers: int = 2, lr: float = 0.002, block_scaled: bool = False):
    """Fits a fixed target with `layers` blocks; (the losses, the blocks, an input to try them on)."""
    torch.manual_seed(0)
    d = 64
    blocks = [PrenormBlock(hidden, hidden // d, max(1, hidden // d // 4), d, 4 * hidden, i, device=device, dtype=dtype,
                           block_scaled=block_scaled)
              for i in range(layers)]
    table = fused.rope_table(tokens, d, device=device)
    axes = fused.rope_axes((d // 2 - 2 * (d // 8), d // 8, d // 8))
    t = torch.arange(tokens, device=device)
    positions = torch.stack([t // 16 * 16, t % 16 // 4, t % 4])  # patches of 4 x 4 at one time each
    x = torch.randn(tokens, hidden, device=device).to(dtype)
    target = torch.randn(tokens, hidden, device=device).to(dtype)
    opt = torch.optim.Adam([p for b in blocks for p in b.parameters()], lr=lr)
    step = torch.zeros(1, dtype=torch.int64, device=device)
    losses = []
    for _ in range(steps):
        branch, residual = x, None
        for b in blocks:
            branch, residual = b(branch, residual, positions, table, axes, seed=7, step=step)
        loss = (branch.float() + residual - target.float()).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        step += 1
        losses.append(loss.detach())
    return torch.stack(losses).tolist(), blocks, (x, positions, table, axes)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--tokens", type=int, default=256)
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--block-scaled", action="store_true", help="train with 8-bit products, a scale per block of 128")
    a = ap.parse_args()
    device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    dtype = torch.bfloat16 if device.type == "cuda" else torch.float32
    losses, blocks, (x, positions, table, axes) = train(a.steps, a.tokens, a.hidden, device, dtype, block_scaled=a.block_scaled)
    print(f"training on {device}: loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    branch, residual = x, None
    served, stream = x, None
    for b in blocks:
        b.eval()
        with torch.no_grad():
            branch, residual = b(branch, residual, positions, table, axes)
        served, stream = b.prepare_serving()(served, stream, positions, table, axes)
    off = (served.float() + stream - branch.float() - residual).norm() / (branch.float() + residual).norm()
    print(f"serving with 8-bit products: {off.item():.4f} off the unquantised blocks")
    branch, residual = x, None
    with torch.no_grad():
        for b in blocks:
            branch, residual = b(branch, residual, torch.arange(a.tokens, device=device), table)
    got = generate(blocks, x[None], a.tokens - 4, table)[0]
    off = (got - branch.float() - residual).norm() / (branch.float() + residual).norm()
    print(f"generating with an 8-bit cache: {off.item():.4f} off the unquantised blocks")


if __name__ == "__main__":
    main()
