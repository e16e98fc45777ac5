# SPDX-License-Identifier: MIT
"""A pre-norm transformer block on the fused operators, as it trains and as it serves.

Training: the branch that a sublayer leaves goes through dropout, joins the residual stream
and is normalised in one operator (`dropout_add_rmsnorm`); q and k are normalised per head and
turned by their positions, as views of the packed projection, in one more (`qk_norm_rope`).
Serving: the norm leaves 8-bit values with a scale per token (`rmsnorm_quant_fwd`) for 8-bit
products. The products and the attention between them are PyTorch's.

    python -m rmsnorm.examples.prenorm_block --steps 20
"""

from __future__ import annotations

import argparse
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import fused


class PrenormBlock(torch.nn.Module):
    """Attention (grouped heads) and MLP. `layer` numbers the block: it chooses its masks."""

    def __init__(self, hidden: int, q_heads: int, k_heads: int, head_dim: int, mlp: int, layer: int = 0, dropout: float = 0.1,
                 device=None, dtype=None):
        super().__init__()
        self.q_heads, self.k_heads, self.head_dim = q_heads, k_heads, head_dim
        self.layer, self.dropout = layer, dropout
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
        branch = self._attention(h @ self.qkv.t(), positions, table, axes, False) @ self.out.t()
        h, residual = fused.dropout_add_rmsnorm(
            branch, self.norm2, residual=residual, p=p, rng=(seed, at + (1 << 32)), residual_dtype=torch.float32, prenorm=True,
            rng_step=step)
        return torch.nn.functional.silu(h @ self.up.t()) @ self.down.t(), residual

    @torch.no_grad()
    def prepare_serving(self) -> "ServingBlock":
        return ServingBlock(self)


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


def train(steps: int, tokens: int, hidden: int, device, dtype, layers: int = 2, lr: float = 0.002):
    """Fits a fixed target with `layers` blocks; (the losses, the blocks, an input to try them on)."""
    torch.manual_seed(0)
    d = 64
    blocks = [PrenormBlock(hidden, hidden // d, max(1, hidden // d // 4), d, 4 * hidden, i, device=device, dtype=dtype)
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
    a = ap.parse_args()
    device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    dtype = torch.bfloat16 if device.type == "cuda" else torch.float32
    losses, blocks, (x, positions, table, axes) = train(a.steps, a.tokens, a.hidden, device, dtype)
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


if __name__ == "__main__":
    main()
