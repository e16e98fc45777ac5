# SPDX-License-Identifier: MIT
"""The fused operators around the norm (`rmsnorm.fused`), as workloads.

  quant      residual addition + RMSNorm with an 8-bit output and scales (e4m3 or int8; one
             scale per row, or one per group of columns): the input of an 8-bit product.
  drop_fwd   dropout from a counter-based generator + residual addition + RMSNorm; the mask
             is never stored.
  drop_bwd   its gradient, which draws the same mask again.
  rope_fwd   per-head RMSNorm of q and k followed by rotary positions with one to three axes
             (time, height, width), on q and k as they lie in a packed projection.
  rope_bwd   its gradient.

`run` computes an operator either with elementary torch operations in 32 bits (`own` false)
or with one call of `rmsnorm.fused` (`own` true); `exact` computes it in 64 bits.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6
_QMAX = {"e4m3": 448.0, "int8": 127.0}


def _quant(name, rows, hidden, dtype, residual, rdtype, q, group, bias=False):
    return {"name": name, "op": "quant", "rows": rows, "hidden": hidden, "dtype": dtype, "residual": residual,
            "rdtype": rdtype, "q": q, "group": group, "bias": bias}


def _drop(name, op, rows, hidden, dtype, residual, rdtype, bias, p):
    return {"name": name, "op": op, "rows": rows, "hidden": hidden, "dtype": dtype, "residual": residual,
            "rdtype": rdtype, "bias": bias, "p": p}


def _rope(name, op, tokens, q_heads, k_heads, head_dim, rotary_dim, sections, interleaved, dtype):
    return {"name": name, "op": op, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim,
            "rotary_dim": rotary_dim, "sections": sections, "interleaved": interleaved, "dtype": dtype}


def listed():
    return [
        # one token of one sequence before an 8-bit product: nothing but latency
        _quant("quant one token", 1, 4096, "bf16", True, "bf16", "e4m3", 0),
        # a decoding batch, block-scaled
        _quant("quant decode batch", 64, 8192, "bf16", True, "bf16", "e4m3", 128),
        # a prompt, block-scaled
        _quant("quant prompt", 8192, 4096, "bf16", True, "bf16", "e4m3", 128),
        # a ragged batch at a width that no 16-byte vector divides, int8, with a bias
        _quant("quant ragged int8", 1000, 4100, "f16", False, "f16", "int8", 0, True),
        # a long prompt at a wide model, the residual stream kept in 32 bits
        _quant("quant wide rows", 32768, 16384, "bf16", True, "f32", "e4m3", 0),
        # a small step of a training run
        _drop("dropout small", "drop_fwd", 64, 4096, "bf16", True, "bf16", False, 0.1),
        # a training step's forward
        _drop("dropout forward", "drop_fwd", 32768, 4096, "bf16", True, "f32", True, 0.1),
        # a training step's backward at a wide model: the largest
        _drop("dropout backward wide", "drop_bwd", 32768, 16384, "bf16", True, "bf16", True, 0.1),
        # an odd width in 32 bits
        _drop("dropout backward odd", "drop_bwd", 2000, 1001, "f32", True, "f32", False, 0.25),
        # sixteen sequences, one new token each
        _rope("rope decode batch", "rope_fwd", 16, 32, 8, 128, 128, "16,24,24", False, "bf16"),
        # a prompt of text and images
        _rope("rope prompt", "rope_fwd", 16384, 32, 8, 128, 128, "16,24,24", False, "bf16"),
        # a training step's backward
        _rope("rope backward", "rope_bwd", 16384, 32, 8, 128, 128, "64", False, "f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    n = _log(rng, 256, 32768)
    return n | 1 if rng.random() < 0.25 else max(256, n // 64 * 64)


def draw(rng):
    op = rng.choice(["quant", "drop_fwd", "drop_bwd", "rope_fwd", "rope_bwd"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("rope_fwd", "rope_bwd"):
        head_dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2])
        pairs = rotary_dim // 2
        n = rng.choice([1, 2, 3])
        first = [pairs // n] * (n - 1)
        sections = ",".join(str(s) for s in first + [pairs - sum(first)])
        k_heads = rng.choice([1, 2, 4, 8])
        q_heads = k_heads * rng.choice([1, 3, 4, 7, 8])
        most = (1 << 26) // ((q_heads + k_heads) * head_dim)
        return _rope("", op, _log(rng, 1, most), q_heads, k_heads, head_dim, rotary_dim, sections, rng.random() < 0.3,
                     dtype)
    hidden = _width(rng)
    rows = _log(rng, 1, (1 << 27) // hidden)
    residual = rng.random() < 0.75
    rdtype = rng.choice([dtype, "f32"]) if residual else dtype
    if op == "quant":
        return _quant("", rows, hidden, dtype, residual, rdtype, rng.choice(["e4m3", "e4m3", "int8"]),
                      rng.choice([0, 32, 64, 128, 256]), rng.random() < 0.25)
    return _drop("", op, rows, hidden, dtype, residual, rdtype, rng.random() < 0.5, rng.choice([0.05, 0.1, 0.25, 0.5]))


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _axes(case):
    """The position axis of each rotary pair: consecutive sections."""
    return tuple(a for a, n in enumerate(_sections(case)) for _ in range(n))


def _positions(axes, tokens, gen, dev):
    """Positions as text with images gives them: one axis counts the tokens; three have runs
    of text (all axes equal) and blocks of patches (one time, rows and columns of a grid)."""
    t = torch.arange(tokens, device=dev)
    start = int(torch.randint(0, 1000, (1,), device=dev, generator=gen))
    if axes == 1:
        return (t + start)[None].contiguous()
    in_image = (t // 512) % 2 == 1
    base = t // 512 * 512 + start
    patch = t % 512
    rows = [torch.where(in_image, base, t + start), torch.where(in_image, base + patch // 32, t + start),
            torch.where(in_image, base + patch % 32, t + start)]
    return torch.stack(rows[:axes]).contiguous()


def _table(longest, rotary_dim, dev):
    """Row p: the cosines, then the sines, of p * base^(-2i / rotary_dim)."""
    inv = 10000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=dev) / rotary_dim)
    angle = torch.arange(longest, dtype=torch.float64, device=dev)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, device=dev, dtype=dtype, generator=gen)

    s = {"case": case}
    if case["op"].startswith("rope"):
        n, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["head_dim"]
        packed = normal(n, (hq + 2 * hk) * d)
        s["q"] = packed[:, : hq * d].view(n, hq, d)
        s["k"] = packed[:, hq * d: (hq + hk) * d].view(n, hk, d)
        s["q_weight"] = 1 + 0.1 * normal(d, dtype=torch.float32)
        s["k_weight"] = 1 + 0.1 * normal(d, dtype=torch.float32)
        s["axes"] = _axes(case)
        s["positions"] = _positions(len(_sections(case)), n, gen, dev)
        s["table"] = _table(n + 2048, case["rotary_dim"], dev)
        if case["op"] == "rope_bwd":
            s["dq_out"], s["dk_out"] = normal(n, hq, d), normal(n, hk, d)
        return s
    rows, hidden = case["rows"], case["hidden"]
    s["weight"] = 1 + 0.1 * normal(hidden, dtype=torch.float32)
    s["bias"] = 0.02 * normal(hidden, dtype=torch.float32) if case["bias"] else None
    if case["op"] != "quant":
        s["rng"] = (int(torch.randint(0, 1 << 62, (1,), device=dev, generator=gen)),
                    int(torch.randint(0, 1 << 40, (1,), device=dev, generator=gen)))
    rdt = _DTYPES[case["rdtype"]]
    if case["op"] == "drop_bwd":
        s["h"] = normal(rows, hidden, dtype=rdt)
        s["dout"] = normal(rows, hidden)
        s["dresidual_out"] = normal(rows, hidden, dtype=rdt) if case["residual"] else None
        s["rstd"] = torch.empty(rows, device=dev, dtype=torch.float32)
        for a in range(0, rows, 4096):
            s["rstd"][a: a + 4096] = torch.rsqrt(s["h"][a: a + 4096].float().square().mean(-1) + _EPS)
        return s
    s["x"] = normal(rows, hidden)
    s["residual"] = normal(rows, hidden) if case["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        at = os.path.join(os.getcwd(), "rmsnorm-h100_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        from rmsnorm import fused

        s["fused"] = fused
    return s


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if op == "quant":
        q, scales, residual_out = (_own_quant if own else _plain_quant)(s)
        out = {"q": q.to(torch.bfloat16) if q.dtype == torch.int8 else q, "scales": scales}
        if s["residual"] is not None:
            out["residual_out"] = residual_out
        return out
    if op == "drop_fwd":
        out, residual_out, rstd = (_own_drop_fwd if own else _plain_drop_fwd)(s)
        return {"out": out, "residual_out": residual_out, "rstd": rstd}
    if op == "drop_bwd":
        dx, dweight, dbias, dresidual = (_own_drop_bwd if own else _plain_drop_bwd)(s)
        return {"dx": dx, "dweight": dweight, "dbias": dbias, "dresidual": dresidual}
    if op == "rope_fwd":
        q, k = (_own_rope_fwd if own else _plain_rope_fwd)(s)
        return {"q": q, "k": k}
    dq, dk, dq_weight, dk_weight = (_own_rope_bwd if own else _plain_rope_bwd)(s)
    return {"dq": dq, "dk": dk, "dq_weight": dq_weight, "dk_weight": dk_weight}


def _own_quant(s):
    c = s["case"]
    return s["fused"].rmsnorm_quant_fwd(
        s["x"], s["weight"], s["bias"], residual=s["residual"],
        quant_dtype=torch.int8 if c["q"] == "int8" else torch.float8_e4m3fn, group_size=c["group"] or None,
        residual_dtype=_DTYPES[c["rdtype"]], eps=_EPS)


def _own_drop_fwd(s):
    c = s["case"]
    return s["fused"].dropout_add_rmsnorm_fwd(
        s["x"], s["weight"], s["bias"], residual=s["residual"], p=c["p"], rng=s["rng"],
        residual_dtype=_DTYPES[c["rdtype"]], eps=_EPS, store_rstd=True)


def _own_drop_bwd(s):
    c = s["case"]
    return s["fused"].dropout_add_rmsnorm_bwd(
        s["h"], s["weight"], s["dout"], s["rstd"], s["dresidual_out"], p=c["p"], rng=s["rng"], has_bias=c["bias"],
        has_residual=c["residual"], bias=s["bias"])


def _own_rope_fwd(s):
    return s["fused"].qk_norm_rope_fwd(
        s["q"], s["k"], s["positions"], s["table"], s["q_weight"], s["k_weight"], axes=s["axes"],
        interleaved=s["case"]["interleaved"], eps=_EPS)


def _own_rope_bwd(s):
    return s["fused"].qk_norm_rope_bwd(
        s["q"], s["k"], s["positions"], s["table"], s["dq_out"], s["dk_out"], s["q_weight"], s["k_weight"],
        axes=s["axes"], interleaved=s["case"]["interleaved"], eps=_EPS)


# ---------------------------------------------------------------------------------------
# Plain forms, in 32 bits
# ---------------------------------------------------------------------------------------
def _affine(y, s):
    y = y * s["weight"]
    return y if s["bias"] is None else y + s["bias"]


def _plain_quant(s):
    c = s["case"]
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    residual_out = h.to(_DTYPES[c["rdtype"]])
    y = _affine(h * torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS), s)
    rows, hidden = y.shape
    group = c["group"] or hidden
    groups = -(-hidden // group)
    pad = groups * group - hidden
    if pad:
        y = torch.cat([y, y.new_zeros(rows, pad)], 1)
    y = y.view(rows, groups, group)
    top = _QMAX[c["q"]]
    scales = (y.abs().amax(-1, keepdim=True) / top).clamp_min(torch.finfo(torch.float32).tiny)
    y = (y / scales).clamp(-top, top).view(rows, groups * group)[:, :hidden]
    q = y.round().to(torch.int8) if c["q"] == "int8" else y.to(torch.float8_e4m3fn).contiguous()
    return q, scales.view(rows, groups) if c["group"] else scales.view(rows), residual_out


def _keep(s, rows, hidden):
    """The mask: word (column mod 4) of Philox4x32-10 with the counter (column / 4, row,
    offset) and the key seed, at least p * 2^32 (Salmon, Moraes, Dror, Shaw, 2011)."""
    dev = s["weight"].device
    low = 0xFFFFFFFF
    seed, offset = s["rng"]
    quads = -(-hidden // 4)
    c0 = torch.arange(quads, device=dev)[None, :]
    c1 = torch.arange(rows, device=dev)[:, None]
    c2, c3 = torch.tensor(offset & low, device=dev), torch.tensor(offset >> 32, device=dev)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    least = int(s["case"]["p"] * 2 ** 32)
    return torch.stack([c0 >= least, c1 >= least, c2 >= least, c3 >= least], -1).view(rows, quads * 4)[:, :hidden]


def _plain_drop_fwd(s):
    c = s["case"]
    h = s["x"].float() * (1 / (1 - c["p"]))
    h = torch.where(_keep(s, *h.shape), h, 0.0)
    if s["residual"] is not None:
        h = h + s["residual"].float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS)
    out = _affine(h * rstd, s).to(s["x"].dtype)
    return out, h.to(_DTYPES[c["rdtype"]]), rstd.view(-1)


def _plain_drop_bwd(s):
    c = s["case"]
    rstd = s["rstd"][:, None]
    xhat = s["h"].float() * rstd
    dy = s["dout"].float()
    dweight = (dy * xhat).sum(0)
    dbias = dy.sum(0) if c["bias"] else None
    dy = dy * s["weight"]
    dh = (dy - xhat * (xhat * dy).mean(-1, keepdim=True)) * rstd
    del xhat, dy
    dresidual = None
    if s["dresidual_out"] is not None:
        dh = dh + s["dresidual_out"].float()
        dresidual = dh.to(s["h"].dtype)
    dx = torch.where(_keep(s, *dh.shape), dh * (1 / (1 - c["p"])), 0.0).to(s["dout"].dtype)
    return dx, dweight, dbias, dresidual


def _cos_sin(s):
    pairs = s["case"]["rotary_dim"] // 2
    axes = torch.tensor(s["axes"], device=s["table"].device)
    at = s["positions"][axes].t()
    i = torch.arange(pairs, device=at.device)
    return s["table"][at, i][:, None, :], s["table"][at, i + pairs][:, None, :]


def _turn(y, cos, sin, interleaved):
    n = cos.shape[-1]
    turned, rest = y[..., : 2 * n], y[..., 2 * n:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :n], turned[..., n:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_rope_fwd(s):
    cos, sin = _cos_sin(s)

    def one(x, w):
        h = x.float()
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS) * w
        return _turn(y, cos, sin, s["case"]["interleaved"]).to(x.dtype)

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def _plain_rope_bwd(s):
    cos, sin = _cos_sin(s)

    def one(x, w, dout):
        g = _turn(dout.float(), cos, -sin, s["case"]["interleaved"])
        h = x.float()
        rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS)
        xhat = h * rstd
        dw = (g * xhat).sum((0, 1))
        g = g * w
        return ((g - xhat * (g * xhat).mean(-1, keepdim=True)) * rstd).to(x.dtype), dw

    dq, dqw = one(s["q"], s["q_weight"], s["dq_out"])
    dk, dkw = one(s["k"], s["k_weight"], s["dk_out"])
    return dq, dk, dqw, dkw


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    b = _BYTES[case["dtype"]]
    if case["op"].startswith("rope"):
        n, d = case["tokens"], case["head_dim"]
        values = n * (case["q_heads"] + case["k_heads"]) * d
        positions = n * len(_sections(case)) * 8 + n * case["rotary_dim"] * 4
        if case["op"] == "rope_fwd":
            return {"bytes": values * 2 * b + positions + 8 * d, "flops": 7 * values}
        return {"bytes": values * 3 * b + positions + 16 * d, "flops": 16 * values}
    rows, hidden = case["rows"], case["hidden"]
    values, rb = rows * hidden, _BYTES[case["rdtype"]]
    affine = hidden * 4 * (2 if case["bias"] else 1)
    if case["op"] == "quant":
        scales = rows * (-(-hidden // case["group"]) if case["group"] else 1) * 4
        return {"bytes": values * (b + 1 + (b + rb if case["residual"] else 0)) + affine + scales, "flops": 8 * values}
    if case["op"] == "drop_fwd":
        return {"bytes": values * (2 * b + rb + (b if case["residual"] else 0)) + affine + rows * 4,
                "flops": 30 * values}
    return {"bytes": values * (rb + 2 * b + (2 * rb if case["residual"] else 0)) + 2 * affine + rows * 4,
            "flops": 40 * values}


# ---------------------------------------------------------------------------------------
# The definitions, in 64 bits, some rows at a time
# ---------------------------------------------------------------------------------------
def _words(rng, first, rows, hidden, dev):
    """The generator's words for rows first .. first + rows - 1, column by column: every
    product of two 32-bit words from 16-bit halves, so nothing passes 64 bits."""
    seed, offset = rng

    def product(v, m):
        lo, hi = (v & 0xFFFF) * m, (v >> 16) * m
        total = (hi >> 16) + (((hi & 0xFFFF) << 16) + lo >> 32)
        return total, ((hi & 0xFFFF) << 16) + lo & 0xFFFFFFFF

    quads = (hidden + 3) // 4
    column = torch.arange(quads, device=dev, dtype=torch.int64).expand(rows, quads)
    row = torch.arange(first, first + rows, device=dev, dtype=torch.int64)[:, None].expand(rows, quads)
    state = [column, row, torch.full_like(column, offset % 2 ** 32), torch.full_like(column, offset // 2 ** 32)]
    for turn in range(10):
        key = [(seed % 2 ** 32 + turn * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + turn * 0xBB67AE85) % 2 ** 32]
        high0, low0 = product(state[0], 0xD2511F53)
        high1, low1 = product(state[2], 0xCD9E8D57)
        state = [high1 ^ state[1] ^ key[0], low1, high0 ^ state[3] ^ key[1], low0]
    return torch.stack(state, 2).reshape(rows, 4 * quads)[:, :hidden]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"].startswith("rope"):
        return _exact_rope(s)
    hidden, rows = case["hidden"], case["rows"]
    step = max(1, (1 << 25) // hidden)
    parts = [_exact_rows(s, a, min(rows, a + step)) for a in range(0, rows, step)]
    found = {}
    for key in list(parts[0]):
        if parts[0][key] is None:
            found[key] = None
        elif key in ("dweight", "dbias"):
            found[key] = torch.stack([p.pop(key) for p in parts]).sum(0)
        else:
            found[key] = torch.cat([p.pop(key) for p in parts])
    return found


def _exact_rows(s, a, z):
    c = s["case"]
    w = s["weight"].double()
    b = s["bias"].double() if s["bias"] is not None else 0.0
    scale = 1.0
    if c["op"] != "quant":
        kept = _words(s["rng"], a, z - a, c["hidden"], w.device) >= math.floor(c["p"] * 4294967296.0)
        scale = kept.double() / (1.0 - c["p"])
    if c["op"] == "drop_bwd":
        g, h, r = s["dout"][a:z].double(), s["h"][a:z].double(), s["rstd"][a:z].double()
        n = torch.einsum("ij,i->ij", h, r)
        along = torch.einsum("ij,ij,j->i", g, n, w) / c["hidden"]
        dh = (g * w - n * along[:, None]) * r[:, None]
        if s["dresidual_out"] is not None:
            dh += s["dresidual_out"][a:z].double()
        return {"dx": dh * scale, "dweight": (g * n).sum(0), "dbias": g.sum(0) if c["bias"] else None,
                "dresidual": dh if s["dresidual_out"] is not None else None}
    h = s["x"][a:z].double() * scale
    if s["residual"] is not None:
        h = h + s["residual"][a:z].double()
    rstd = (h.pow(2).sum(1) / c["hidden"] + _EPS).pow(-0.5)
    y = h * rstd[:, None] * w + b
    if c["op"] == "drop_fwd":
        return {"out": y, "residual_out": h, "rstd": rstd}
    size = c["group"] or c["hidden"]
    places = torch.arange(c["hidden"], device=y.device) // size
    most = torch.zeros(z - a, int(places[-1]) + 1, device=y.device, dtype=torch.float64)
    most = most.scatter_reduce(1, places.expand(z - a, -1), y.abs(), "amax")
    scales = most / _QMAX[c["q"]]
    found = {"q": y / scales[:, places], "scales": scales if c["group"] else scales[:, 0]}
    if s["residual"] is not None:
        found["residual_out"] = h
    return found


def _exact_rope(s):
    c = s["case"]
    pairs = c["rotary_dim"] // 2
    first = torch.arange(pairs, device=s["table"].device) * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else pairs)
    rows = torch.stack([s["positions"][axis] for axis in s["axes"]], 1)
    z = torch.complex(s["table"].double().gather(0, rows), s["table"][:, pairs:].double().gather(0, rows))

    def rotate(y, by):
        turned = torch.complex(y[..., first], y[..., second]) * by[:, None, :]
        y = y.clone()
        y[..., first], y[..., second] = turned.real, turned.imag
        return y

    found = {}
    for n in ("q", "k"):
        x, w = s[n].double(), s[n + "_weight"].double()
        r = (x.pow(2).sum(-1, keepdim=True) / c["head_dim"] + _EPS).pow(-0.5)
        if c["op"] == "rope_fwd":
            found[n] = rotate(x * r * w, z)
            continue
        g = rotate(s["d%s_out" % n].double(), z.conj())
        along = (g * w * x).sum(-1, keepdim=True) * r.pow(3) / c["head_dim"]
        found["d" + n] = g * w * r - x * along
        found["d%s_weight" % n] = torch.einsum("thd,thd,thx->d", g, x, r)
    return found
