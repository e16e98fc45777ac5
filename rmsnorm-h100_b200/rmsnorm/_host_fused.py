# SPDX-License-Identifier: MIT
"""Host-tensor semantics of the fused operators, in plain PyTorch (fp32 math).

`rmsnorm.fused` calls these for tensors that are not on a CUDA device; CUDA tensors always
go to the native library. `philox_words` works on any device.
"""

from __future__ import annotations

import torch

from ._host import _affine, sum_to_affine_shape

_LOW = 0xFFFFFFFF


def philox_words(rows: int, hidden: int, seed: int, offset: int, row_offset: int, device) -> torch.Tensor:
    """The 32-bit words of the dropout mask as int64 [rows, hidden]: word j % 4 of
    Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) with key `seed` and counter
    (j / 4, row_offset + i, offset). Products wrap modulo 2^64, so the arithmetic shift and
    the mask give their high words."""
    quads = (hidden + 3) // 4
    c0 = torch.arange(quads, dtype=torch.int64, device=device)[None, :]
    c1 = torch.arange(row_offset, row_offset + rows, dtype=torch.int64, device=device)[:, None]
    c2 = torch.tensor(offset & _LOW, dtype=torch.int64, device=device)
    c3 = torch.tensor(offset >> 32, dtype=torch.int64, device=device)
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & _LOW) ^ c1 ^ k0, b & _LOW, (a >> 32 & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = k0 + 0x9E3779B9 & _LOW, k1 + 0xBB67AE85 & _LOW
    return torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), -1).reshape(rows, quads * 4)[:, :hidden]


def dropout_mask(shape, p, seed, offset, row_offset, device) -> torch.Tensor:
    hidden = shape[-1]
    rows = 1
    for d in shape[:-1]:
        rows *= d
    return (philox_words(rows, hidden, seed, offset, row_offset, device) >= int(p * 2**32)).reshape(shape)


def rmsnorm_quant_fwd(x, weight, bias, residual, quant_dtype, group_size, residual_dtype, eps, scales):
    h = x.float()
    if residual is not None:
        h = h + residual.float()
        residual_out = h.to(residual_dtype or residual.dtype)
    else:
        residual_out = x if residual_dtype in (None, x.dtype) else x.to(residual_dtype)
    y = _affine(h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps), weight, bias)
    n = y.shape[-1]
    size = group_size or n
    groups = (n + size - 1) // size
    g = torch.nn.functional.pad(y, (0, groups * size - n)).reshape(*y.shape[:-1], groups, size)
    top = 127.0 if quant_dtype == torch.int8 else 448.0
    s = (g.abs().amax(-1, keepdim=True) / top).clamp_min(torch.finfo(torch.float32).tiny)
    q = (g / s).clamp(-top, top)
    if quant_dtype == torch.int8:
        q = torch.where(q.isnan(), 0.0, q).round()
    scales.copy_(s.reshape(scales.shape))
    return q.reshape(*y.shape[:-1], groups * size)[..., :n].to(quant_dtype).contiguous(), residual_out


def dropout_add_rmsnorm_fwd(x, weight, bias, residual, mask, p, out_dtype, residual_dtype, eps, store_rstd):
    h = torch.where(mask, x.float() * (1.0 / (1.0 - p)), 0.0)
    if residual is not None:
        h = h + residual.float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
    out = _affine(h * rstd, weight, bias).to(out_dtype)
    return out, h.to(residual_dtype), rstd.squeeze(-1) if store_rstd else None


def dropout_add_rmsnorm_bwd(h, weight, dout, rstd, dresidual_out, mask, p, has_bias, bias, dx_dtype):
    """(dx, dweight, dbias, dh in fp32)."""
    r = rstd.reshape(h.shape[:-1]).unsqueeze(-1)
    xhat = h.float() * r
    dy = dout.float()
    dw = sum_to_affine_shape(dy * xhat, weight.shape).to(weight.dtype) if weight is not None else None
    db = None
    if has_bias:
        like = bias if bias is not None else weight
        db = sum_to_affine_shape(dy, h.shape[-1:]).to(like.dtype if like is not None else dout.dtype)
    wdy = dy * weight.float() if weight is not None else dy
    dh = (wdy - xhat * (xhat * wdy).mean(-1, keepdim=True)) * r
    if dresidual_out is not None:
        dh = dh + dresidual_out.float()
    return torch.where(mask, dh * (1.0 / (1.0 - p)), 0.0).to(dx_dtype), dw, db, dh


def rope_cos_sin(positions, table, axes):
    """cos, sin [tokens..., pairs] with a NaN pair where the position lies outside the table."""
    pairs = table.shape[-1] // 2
    at = positions.long()[torch.tensor(axes, dtype=torch.int64, device=positions.device)].movedim(0, -1)
    bad = (at < 0) | (at >= table.shape[0])
    at = torch.where(bad, 0, at)
    i = torch.arange(pairs, device=table.device)
    nan = table.new_full((), float("nan"))
    return torch.where(bad, nan, table[at, i]), torch.where(bad, nan, table[at, i + pairs])


def rope_turn(y, cos, sin, interleaved):
    n = cos.shape[-1]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    turned, rest = y[..., : 2 * n], y[..., 2 * n:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :n], turned[..., n:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def qk_norm_rope_fwd(x, weight, cos, sin, interleaved, norm, eps):
    y = x.float()
    if norm:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    return rope_turn(y, cos, sin, interleaved).to(x.dtype)


def qk_norm_rope_bwd(x, weight, dout, cos, sin, interleaved, norm, eps):
    g = rope_turn(dout.float(), cos, -sin, interleaved)
    xhat = x.float()
    rstd = 1.0
    if norm:
        rstd = torch.rsqrt(xhat.square().mean(-1, keepdim=True) + eps)
        xhat = xhat * rstd
    dw = None
    if weight is not None:
        dw = sum_to_affine_shape(g * xhat, weight.shape).to(weight.dtype)
        g = g * weight.float()
    if norm:
        g = (g - xhat * (g * xhat).mean(-1, keepdim=True)) * rstd
    return g.to(x.dtype), dw
