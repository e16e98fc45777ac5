# SPDX-License-Identifier: MIT
"""The 8-bit products, their quantisation and the quantised cache in 64 bits, and the error that
their results may have. Test infrastructure.

A quantised value has one right answer: the scales are powers of two, so x / scale is exact and
its nearest e4m3 number (ties to even) is the same in any precision. A product sums 128 terms of
exact products in a tensor core and adds the groups' sums, times two scales, in fp32: whatever the
order, and rounding down or to nearest, each of the 128 + groups additions and the 3
multiplications loses at most 2^-23 of the sum of magnitudes. The result is rounded once (half a
step of its type)."""

from __future__ import annotations

import torch

from fused_ref import TINY, UNIT

E4M3 = torch.float8_e4m3fn


def power_scale(most):
    """The smallest power of two (from 2^-126) s with most <= 448 s, by trying."""
    e = torch.floor(torch.log2(torch.where(most == 0, 1.0, most))) - 10
    for _ in range(4):
        e = torch.where(most > 448.0 * torch.exp2(e), e + 1, e)
    return torch.exp2(torch.where(most == 0, -126.0, e).clamp_min(-126.0))


def nearest_e4m3(v):
    e = torch.floor(torch.log2(torch.where(v == 0, 1.0, v).abs()))
    step = torch.exp2(e.clamp_min(-6) - 3)
    return (v / step).round() * step


def quantize(x, rows):
    """(values of q, scales) in 64 bits."""
    x = x.double()
    n, k = x.shape
    gn, gk = -(-n // rows), -(-k // 128)
    wide = torch.nn.functional.pad(x, (0, gk * 128 - k, 0, gn * rows - n)).view(gn, rows, gk, 128)
    s = power_scale(wide.abs().amax((1, 3)))
    q = nearest_e4m3(wide / s[:, None, :, None]).view(gn * rows, gk * 128)[:n, :k]
    return q, s


def check_quantized(q, scales, x, rows):
    want, s = quantize(x, rows)
    assert q.dtype == E4M3 and scales.dtype == torch.float32
    assert q.shape == want.shape and scales.shape == s.shape, (q.shape, want.shape, scales.shape, s.shape)
    assert torch.equal(scales.double(), s)
    assert torch.equal(q.double(), want)


def values(q, scales):
    """q * scales in 64 bits; rows of scales: q's, or its blocks of 128."""
    n, k = q.shape
    rows = 1 if scales.shape[0] == n else 128
    return q.double() * scales.double().repeat_interleave(128, 1)[:, :k].repeat_interleave(rows, 0)[:n]


def check_product(got, a, b, bias, what, in_cores=False):
    """got against a b^T + bias for 64-bit a and b."""
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    groups = -(-a.shape[1] // 128)
    off = (got.double() - want).abs()
    # where the tensor cores add all of k, 32 products at a time, there are 4 additions a group
    allowed = UNIT[got.dtype] * want.abs() + (128 + (4 if in_cores else 1) * groups + 4) * 2.0**-23 * size + TINY[got.dtype]
    bad = ~(off <= allowed)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off - allowed)[bad].max())} beyond"


def check_cached(q, scales, x, top):
    """q and scales of x's heads: the scale is max |x| / top rounded to fp32; q is x / scale within
    half a step of its type, and one part in 2^22 for the two roundings before it."""
    x = x.double()
    s = (x.abs().amax(-1) / top).clamp_min(2.0**-126)
    assert ((scales.double() - s).abs() <= 2.0**-24 * s).all()
    v = x / scales.double()[..., None]
    step = 0.5 if q.dtype == torch.int8 else torch.clamp(v.abs() / 16, min=2.0**-10)
    assert ((q.double() - v).abs() <= step + 2.0**-22 * v.abs()).all()
    assert (q.double().abs() <= top).all()
