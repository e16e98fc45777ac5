# SPDX-License-Identifier: MIT
"""The fused operators in 64 bits, and the error their results may have. Test infrastructure.

A result that is rounded once to a type with unit roundoff u from fp32 arithmetic may be off
by u |r| plus the fp32 error. The latter is at most a few units of 2^-24 for each of the
handful of operations on an element, and for a sum over n terms (added in a tree, or in
short runs whose sums are added) a few units of the sum of magnitudes: FP32 below, 32 units,
bounds both with room for the order of additions."""

from __future__ import annotations

import torch

FP32 = 32 * 2.0**-24
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # 2^-(bits of the significand)
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}


def check(got, want, size, what):
    """|got - want| within one rounding to got's type and the fp32 error of terms of magnitude
    `size` (a 64-bit tensor that broadcasts to want)."""
    want = want.to(got.device)
    size = size.to(got.device) if isinstance(size, torch.Tensor) else size
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    allowed = UNIT[got.dtype] * want.abs() + FP32 * (want.abs() + size) + TINY[got.dtype]
    bad = ~(off <= allowed)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off - allowed)[bad].max())} beyond"


def normalise(x, weight, bias, residual, eps=1e-6, keep=None, p=0.0):
    """(h, rstd, y, the magnitude of y's terms: those of the residual addition may cancel)."""
    h = x.double()
    if keep is not None:
        h = torch.where(keep, h / (1 - p), 0.0)
    size = h.abs()
    if residual is not None:
        h = h + residual.double()
        size = size + residual.double().abs()
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    y, size = h * rstd, size * rstd
    if weight is not None:
        y, size = y * weight.double(), size * weight.double().abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return h, rstd, y, size


def check_quant(q, scales, y, size, quant_dtype, group):
    """q * scales holds y: scales exact to fp32, q rounded to nearest (one part in 16 of a
    normal e4m3 value, half of its smallest step 2^-9 below; half a step of int8)."""
    n = y.shape[-1]
    g = group or n
    top = 127.0 if quant_dtype == torch.int8 else 448.0
    groups = -(-n // g)
    wide = torch.nn.functional.pad(y.abs(), (0, groups * g - n)).reshape(*y.shape[:-1], groups, g)
    s64 = (wide.amax(-1) / top).clamp_min(2.0**-126)
    most = torch.nn.functional.pad(size, (0, groups * g - n)).reshape(wide.shape).amax(-1)
    s = scales if group else scales.unsqueeze(-1)
    check(s, s64, most / top, "scales")
    each = s.double().repeat_interleave(g, -1)[..., :n]
    v = y / each
    slack = FP32 * (v.abs() + size / each)
    step = 0.5 if quant_dtype == torch.int8 else torch.clamp(v.abs() / 16, min=2.0**-10)
    off = (q.double() - v).abs()
    bad = ~(off <= step + slack)
    assert not bad.any(), f"q: {int(bad.sum())} of {bad.numel()} not the nearest value, worst off {float(off[bad].max())}"
    assert q.double().abs().max() <= top


def backward(h, weight, dout, rstd, dro, keep, p):
    r = rstd.double().reshape(h.shape[:-1]).unsqueeze(-1)
    xhat = h.double() * r
    g = dout.double()
    wdy = g * weight.double() if weight is not None else g
    c = (xhat * wdy).mean(-1, keepdim=True)
    size = (wdy.abs() + xhat.abs() * (xhat * wdy).abs().mean(-1, keepdim=True)) * r
    dh = (wdy - xhat * c) * r
    if dro is not None:
        dh = dh + dro.double()
        size = size + dro.double().abs()
    dx = torch.where(keep, dh / (1 - p), 0.0)
    lead = tuple(range(h.dim() - 1))
    return {"dh": dh, "size": size, "dx": dx, "dw": (g * xhat).sum(lead), "dw_size": (g * xhat).abs().sum(lead),
            "db": g.sum(lead), "db_size": g.abs().sum(lead)}


def turn(y, cos, sin, interleaved):
    n = cos.shape[-1]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out = y.clone()
    out[..., a] = y[..., a] * cos - y[..., b] * sin
    out[..., b] = y[..., b] * cos + y[..., a] * sin
    return out


def cos_sin(positions, table, axes):
    """positions [axes, tokens...]."""
    pairs = table.shape[1] // 2
    t = table.double()
    cos = torch.stack([t[positions[a].long(), i] for i, a in enumerate(axes)], -1) if pairs else t.new_zeros(*positions.shape[1:], 0)
    sin = torch.stack([t[positions[a].long(), pairs + i] for i, a in enumerate(axes)], -1) if pairs else cos
    return cos.unsqueeze(-2), sin.unsqueeze(-2)


def rope(x, weight, cos, sin, interleaved, norm, eps=1e-6):
    y = x.double()
    if norm:
        y = y * (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    if weight is not None:
        y = y * weight.double()
    return turn(y, cos, sin, interleaved), turn(y.abs(), cos.abs(), -sin.abs(), interleaved).abs() + turn(
        y.abs(), cos.abs(), sin.abs(), interleaved)


def rope_backward(x, weight, dout, cos, sin, interleaved, norm, eps=1e-6):
    g = turn(dout.double(), cos, -sin, interleaved)
    gs = dout.double().abs()
    gs = gs + turn(gs, cos.abs(), sin.abs(), interleaved).abs() + turn(gs, cos.abs(), -sin.abs(), interleaved).abs()
    xhat = x.double()
    r = 1.0
    if norm:
        r = (xhat.square().mean(-1, keepdim=True) + eps).rsqrt()
        xhat = xhat * r
    dw, dw_size = g * xhat, gs * xhat.abs()
    if weight is not None:
        g, gs = g * weight.double(), gs * weight.double().abs()
    dx, size = g, gs
    if norm:
        dx = (g - xhat * (g * xhat).mean(-1, keepdim=True)) * r
        size = (gs + xhat.abs() * (gs * xhat.abs()).mean(-1, keepdim=True)) * r
    return dx, size, dw, dw_size
