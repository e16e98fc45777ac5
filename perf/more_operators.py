# SPDX-License-Identifier: MIT
"""The operators that take the norm's 8-bit outputs and the turned keys further
(`rmsnorm.fused`), as workloads.

  quantize     e4m3 values with a power of two as scale, per 1 x 128 group or per 128 x 128
               block; where asked, those of the transposed matrix too.
  product      the product of two such matrices, a bias added.
  linear       a linear layer on those two, forward and backward: three products of operands
               quantised on the way.
  cache_write  keys and values of new tokens, 8 bits with a scale per token and head, into the
               pages of a cache.
  cache_read   the tokens of some sequences read back through their page tables, one sequence
               after the other.

`run` computes an operator either with elementary torch operations in 32 bits (`own` false)
or with calls of `rmsnorm.fused` (`own` true); `exact` computes it in 64 bits.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn,
           "int8": torch.int8}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_TOP = {"e4m3": 448.0, "int8": 127.0}
_TINY = 2.0 ** -126


def _quantize(name, rows, hidden, dtype, block_rows, transposed):
    return {"name": name, "op": "quantize", "rows": rows, "hidden": hidden, "dtype": dtype, "block_rows": block_rows,
            "transposed": transposed}


def _product(name, m, n, k, out, bias, b_block_rows, column_major):
    return {"name": name, "op": "product", "m": m, "n": n, "k": k, "out": out, "bias": bias,
            "b_block_rows": b_block_rows, "column_major": column_major}


def _linear(name, tokens, n, k, dtype, bias):
    return {"name": name, "op": "linear", "tokens": tokens, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _cache(name, op, tokens, sequences, heads, head_dim, page, dtype, kept):
    return {"name": name, "op": op, "tokens": tokens, "sequences": sequences, "heads": heads, "head_dim": head_dim,
            "page": page, "dtype": dtype, "kept": kept}


def listed():
    return [
        # one token's activations between two products: nothing but latency
        _quantize("quantize one token", 1, 4096, "bf16", 1, False),
        # a layer's weight in a training step, for the forward product and, transposed, the backward
        _quantize("quantize weight", 16384, 4096, "bf16", 128, True),
        # one new token of one sequence: the weight has to be read, once
        _product("product one token", 1, 4096, 4096, "bf16", False, 128, False),
        # a decoding batch at a wide model
        _product("product decode batch", 64, 8192, 8192, "bf16", False, 128, True),
        # a prompt through the first product of an MLP
        _product("product prompt", 8192, 16384, 4096, "bf16", False, 128, True),
        # a ragged batch at widths that no 16 bytes divide, with a bias
        _product("product ragged", 1000, 4100, 1001, "f16", True, 128, False),
        # a training step of a layer, forward and backward: the largest
        _linear("linear training step", 8192, 8192, 4096, "bf16", False),
        # a small layer of odd sizes, in 32 bits, with a bias
        _linear("linear ragged", 333, 520, 1001, "f32", True),
        # sixteen sequences, one new token each
        _cache("cache write decode batch", "cache_write", 16, 16, 8, 128, 64, "bf16", "e4m3"),
        # prompts, packed, with padding behind the last
        _cache("cache write prompts", "cache_write", 16384, 7, 8, 128, 64, "bf16", "e4m3"),
        # a ragged batch of short sequences, small pages
        _cache("cache read ragged", "cache_read", 3001, 16, 8, 128, 16, "f16", "e4m3"),
        # some long sequences
        _cache("cache read long", "cache_read", 131072, 5, 8, 128, 64, "bf16", "e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    n = _log(rng, lo, hi)
    if rng.random() < 0.25:
        return n | 1
    return max(lo, n // 128 * 128 if rng.random() < 0.6 else n // 8 * 8)


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "product", "linear", "cache_write", "cache_read"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quantize":
        hidden = _width(rng, 128, 16384)
        return _quantize("", _log(rng, 1, (1 << 26) // hidden), hidden, dtype, rng.choice([1, 1, 128]),
                         rng.random() < 0.5)
    if op == "product":
        n, k = _width(rng, 128, 16384), _width(rng, 128, 16384)
        m = _log(rng, 1, min(16384, (1 << 39) // (n * k)))
        return _product("", m, n, k, dtype, rng.random() < 0.3, rng.choice([128, 128, 1]), rng.random() < 0.5)
    if op == "linear":
        n, k = _width(rng, 128, 8192), _width(rng, 128, 8192)
        tokens = _log(rng, 16, min(16384, (1 << 37) // (n * k)))
        return _linear("", tokens, n, k, dtype, rng.random() < 0.5)
    heads, head_dim = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([64, 80, 96, 128, 128, 192, 256])
    most = (1 << 26) // (heads * head_dim)
    tokens = _log(rng, 1, most)
    return _cache("", op, tokens, min(tokens, _log(rng, 1, 256)), heads, head_dim, rng.choice([1, 8, 16, 17, 64, 256]),
                  dtype, rng.choice(["e4m3", "e4m3", "int8"]))


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _cuts(tokens, sequences, gen, dev):
    """sequences + 1 starts that share out `tokens`: uneven, some of no tokens."""
    cuts = torch.randint(0, tokens + 1, (sequences - 1,), device=dev, generator=gen).sort().values
    ends = torch.tensor([0], device=dev), cuts, torch.tensor([tokens], device=dev)
    return torch.cat(ends).to(torch.int32)


def _groups_of(x, rows):
    """(q, scales) of x with a scale per `rows` x 128 values, as a program has them before it
    calls the product."""
    n, k = x.shape
    gn, gk = -(-n // rows), -(-k // 128)
    wide = torch.nn.functional.pad(x.float(), (0, gk * 128 - k, 0, gn * rows - n)).view(gn, rows, gk, 128)
    s = (wide.abs().amax((1, 3)) / 448.0).clamp_min(_TINY)
    q = (wide / s[:, None, :, None]).clamp(-448.0, 448.0).view(gn * rows, gk * 128)[:n, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), s


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=dev, dtype=dtype, generator=gen)

    def activations(rows, hidden, dtype=torch.float32):
        """Normal values; one column in 64 is ten times as large, as outlier channels are."""
        column = torch.where(torch.rand(hidden, device=dev, generator=gen) < 1 / 64, 10.0, 1.0).to(dtype)
        return normal(rows, hidden, dtype=dtype) * column

    s = {"case": case}
    op = case["op"]
    if op == "quantize":
        s["x"] = activations(case["rows"], case["hidden"], _DTYPES[case["dtype"]])
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], a_scales = _groups_of(activations(m, k), 1)
        s["a_scales"] = a_scales.t().contiguous().t() if case["column_major"] else a_scales
        s["b"], s["b_scales"] = _groups_of(normal(n, k) * k ** -0.5, case["b_block_rows"])
        s["bias"] = 0.1 * normal(n) if case["bias"] else None
    elif op == "linear":
        dt = _DTYPES[case["dtype"]]
        t, n, k = case["tokens"], case["n"], case["k"]
        s["x"] = activations(t, k, dt).requires_grad_(True)
        s["weight"] = (normal(n, k) * k ** -0.5).to(dt).requires_grad_(True)
        s["bias"] = (0.1 * normal(n)).to(dt).requires_grad_(True) if case["bias"] else None
        s["dy"] = normal(t, n, dtype=dt)
    else:
        t, h, d, page, sequences = (case[i] for i in ("tokens", "heads", "head_dim", "page", "sequences"))
        starts = _cuts(t, sequences, gen, dev)
        lengths = starts[1:] - starts[:-1]
        each = (lengths + page - 1) // page
        per = int(each.max())
        pages = t // page + sequences + 2
        # the pages of a sequence lie anywhere; page 0 belongs to none
        free = 1 + torch.randperm(pages - 1, device=dev, generator=gen)
        first = torch.cumsum(each, 0) - each
        column = torch.arange(per, device=dev)[None, :]
        table = torch.where(column < each[:, None], free[(first[:, None] + column).clamp_max(pages - 2)], -1)
        s["table"], s["starts"] = table.to(torch.int32).contiguous(), starts
        kept = _DTYPES[case["kept"]]
        for name in ("k", "v"):
            held = torch.randint(-119, 120, (pages, page, h, d), device=dev, dtype=torch.int8, generator=gen)
            # as e4m3 the bytes 0 to 126 and 128 to 254 are numbers: the sign moves to the top bit
            s[name + "_cache"] = held if kept == torch.int8 else (
                held.abs().view(torch.uint8) + (held < 0).to(torch.uint8) * 128).view(kept)
            s[name + "_scales"] = torch.rand(pages, page, h, device=dev, generator=gen) * 0.02 + 0.001
        if op == "cache_write":
            packed = normal(t, 3 * h * d, dtype=_DTYPES[case["dtype"]])
            s["k"] = packed[:, h * d: 2 * h * d].view(t, h, d)
            s["v"] = packed[:, 2 * h * d:].view(t, h, d)
            at = torch.arange(t, device=dev)
            seq = torch.searchsorted(starts, at.to(torch.int32), right=True) - 1
            pos = at - starts[seq]
            slots = s["table"][seq, pos // page].long() * page + pos % page
            # the last of many tokens are padding
            s["slots"] = torch.where(at < t - t // 16, slots, -1)
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
    if op == "quantize":
        names = ("q", "scales", "q_t", "scales_t")
        return dict(zip(names, (_own_quantize if own else _plain_quantize)(s)))
    if op == "product":
        return (_own_product if own else _plain_product)(s)
    if op == "linear":
        y, dx, dw, db = (_own_linear if own else _plain_linear)(s)
        out = {"y": y, "dx": dx, "dweight": dw}
        return out if db is None else {**out, "dbias": db}
    if op == "cache_write":
        (_own_cache_write if own else _plain_cache_write)(s)
        out = {}
        for name in ("k", "v"):
            held = s[name + "_cache"]
            out[name + "_cache"] = held.to(torch.bfloat16) if held.dtype == torch.int8 else held
            out[name + "_scales"] = s[name + "_scales"]
        return out
    k, v = (_own_cache_read if own else _plain_cache_read)(s)
    return {"k": k, "v": v}


def _own_quantize(s):
    return s["fused"].block_quantize(s["x"], block_rows=s["case"]["block_rows"], transposed=s["case"]["transposed"])


def _own_product(s):
    return s["fused"].block_mm(s["a"], s["a_scales"], s["b"], s["b_scales"], bias=s["bias"],
                               out_dtype=_DTYPES[s["case"]["out"]])


def _own_linear(s):
    y = s["fused"].block_linear(s["x"], s["weight"], s["bias"])
    leaves = [s["x"], s["weight"]] + ([] if s["bias"] is None else [s["bias"]])
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return y.detach(), grads[0], grads[1], grads[2] if len(grads) == 3 else None


def _own_cache_write(s):
    s["fused"].cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["slots"])


def _own_cache_read(s):
    return s["fused"].cache_read(s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["table"], s["starts"],
                                 s["case"]["tokens"], dtype=_DTYPES[s["case"]["dtype"]])


# ---------------------------------------------------------------------------------------
# Plain forms, in 32 bits
# ---------------------------------------------------------------------------------------
def _plain_power(most):
    """The smallest power of two, 2^-126 at least, that brings `most` to 448 = 0.875 * 2^9 or below."""
    part, exponent = torch.frexp(most)
    exponent = exponent - 9 + (part > 0.875).to(torch.int32)
    return (exponent.clamp_min(-126) + 127 << 23).view(torch.float32)


def _plain_blocks(x, rows):
    """(e4m3 values, scales) of x, a scale per `rows` x 128 values."""
    n, k = x.shape
    gn, gk = -(-n // rows), -(-k // 128)
    y = x.float()
    if gn * rows != n or gk * 128 != k:
        wide = y.new_zeros(gn * rows, gk * 128)
        wide[:n, :k] = y
        y = wide
    y = y.view(gn, rows, gk, 128)
    scales = _plain_power(y.abs().amax(3).amax(1))
    y = (y / scales[:, None, :, None]).view(gn * rows, gk * 128)
    return y[:n, :k].to(torch.float8_e4m3fn).contiguous(), scales


def _plain_values(q, scales):
    """The values that q and its scales hold."""
    n, k = q.shape
    rows = 1 if scales.shape[0] == n else 128
    wide = scales.repeat_interleave(128, 1)[:, :k]
    if rows > 1:
        wide = wide.repeat_interleave(rows, 0)[:n]
    return q.float() * wide


def _plain_quantize(s):
    c = s["case"]
    out = _plain_blocks(s["x"], c["block_rows"])
    return out + _plain_blocks(s["x"].t(), c["block_rows"]) if c["transposed"] else out


def _plain_product(s):
    out = _plain_values(s["a"], s["a_scales"]) @ _plain_values(s["b"], s["b_scales"]).t()
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(_DTYPES[s["case"]["out"]])


@torch.no_grad()
def _plain_linear(s):
    x, w, dy = s["x"], s["weight"], s["dy"]
    wv = _plain_values(*_plain_blocks(w, 128))
    y = _plain_values(*_plain_blocks(x, 1)) @ wv.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    dx = _plain_values(*_plain_blocks(dy, 1)) @ wv
    dw = _plain_values(*_plain_blocks(dy.t(), 1)) @ _plain_values(*_plain_blocks(x.t(), 1)).t()
    db = None if s["bias"] is None else dy.float().sum(0).to(s["bias"].dtype)
    return y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype), db


def _plain_cache_write(s):
    c = s["case"]
    top = _TOP[c["kept"]]
    valid = s["slots"] >= 0
    at = torch.where(valid, s["slots"], 0)  # padding writes what slot 0 has back to it
    for name in ("k", "v"):
        x = s[name].float()
        scales = (x.abs().amax(-1) / top).clamp_min(_TINY)
        q = (x / scales[..., None]).clamp(-top, top)
        q = (q.round() if c["kept"] == "int8" else q).to(_DTYPES[c["kept"]]).view(torch.uint8)
        cache = s[name + "_cache"].view(torch.uint8).view(-1, c["heads"], c["head_dim"])
        held = s[name + "_scales"].view(-1, c["heads"])
        cache[at] = torch.where(valid[:, None, None], q, cache[0])
        held[at] = torch.where(valid[:, None], scales, held[0])


def _plain_cache_read(s):
    c = s["case"]
    at = torch.arange(c["tokens"], device=s["starts"].device, dtype=torch.int32)
    seq = torch.searchsorted(s["starts"], at, right=True) - 1
    pos = at - s["starts"][seq]
    page = s["table"][seq, pos // c["page"]]
    slot = pos % c["page"]
    out = []
    for name in ("k", "v"):
        q = s[name + "_cache"].view(torch.uint8)[page, slot].view(_DTYPES[c["kept"]])
        out.append((q.float() * s[name + "_scales"][page, slot][..., None]).to(_DTYPES[c["dtype"]]))
    return out


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "quantize":
        rows, hidden = case["rows"], case["hidden"]
        copies = 2 if case["transposed"] else 1
        return {"bytes": rows * hidden * (_BYTES[case["dtype"]] + copies), "flops": 3 * copies * rows * hidden}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * _BYTES[case["out"]], "flops": 2 * m * n * k}
    if op == "linear":
        t, n, k, b = case["tokens"], case["n"], case["k"], _BYTES[case["dtype"]]
        return {"bytes": 2 * (t * k + n * k + t * n) * b, "flops": 6 * t * n * k}
    values = 2 * case["tokens"] * case["heads"] * case["head_dim"]
    scales = 8 * case["tokens"] * case["heads"]
    return {"bytes": values * (_BYTES[case["dtype"]] + 1) + scales + 8 * case["tokens"],
            "flops": (3 if op == "cache_write" else 1) * values}


# ---------------------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------------------
def _two_to(exponent):
    return (exponent.long() + 1023 << 52).view(torch.float64)


def _nearest_e4m3(v):
    """The e4m3 number next to each value, ties to the even one: three bits behind the first,
    steps of 2^-9 at the least."""
    exponent = torch.frexp(v).exponent - 1
    step = _two_to(exponent.clamp_min(-6) - 3)
    return ((v / step).round() * step).clamp(-448.0, 448.0)


def _exact_blocks(x, rows, values=True):
    """(the e4m3 numbers, scales) of x, or with `values` their products; strip by strip."""
    x = x.detach().double()
    n, k = x.shape
    q = torch.empty_like(x)
    scales = x.new_empty(-(-n // rows), -(-k // 128))
    for j in range(scales.shape[1]):
        part = x[:, 128 * j: 128 * j + 128]
        most = part.abs().amax(1)
        if rows > 1:
            most = torch.stack([p.amax() for p in most.split(rows)])
        low = _two_to(torch.frexp(most).exponent - 9)  # 448 low <= 1.75 most
        scales[:, j] = torch.where(most == 0, _TINY, torch.where(most > 448.0 * low, 2 * low, low).clamp_min(_TINY))
        each = scales[:, j].repeat_interleave(rows)[:n, None]
        q[:, 128 * j: 128 * j + 128] = _nearest_e4m3(part / each) * (each if values else 1.0)
    return q if values else (q, scales)


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        out = dict(zip(("q", "scales"), _exact_blocks(s["x"], case["block_rows"], False)))
        if case["transposed"]:
            out["q_t"], out["scales_t"] = _exact_blocks(s["x"].t(), case["block_rows"], False)
        return out
    if op == "product":
        rows = case["b_block_rows"]
        total = 0.0
        for j in range(s["a_scales"].shape[1]):  # group by group of 128 columns
            cols = slice(128 * j, 128 * j + 128)
            a = s["a"][:, cols].double() * s["a_scales"][:, j: j + 1].double()
            each = s["b_scales"][:, j].double().repeat_interleave(rows)[: case["n"], None]
            total = total + a @ (s["b"][:, cols].double() * each).t()
        return total if s["bias"] is None else total + s["bias"].double()
    if op == "linear":
        x, w, dy = s["x"], s["weight"], s["dy"]
        wv = _exact_blocks(w, 128)
        y = _exact_blocks(x, 1) @ wv.t()
        out = {"dx": _exact_blocks(dy, 1) @ wv}
        del wv
        out["dweight"] = _exact_blocks(dy.t(), 1) @ _exact_blocks(x.t(), 1).t()
        if s["bias"] is not None:
            y = y + s["bias"].detach().double()
            out["dbias"] = dy.double().sum(0)
        return {"y": y, **out}
    t, page = case["tokens"], case["page"]
    if op == "cache_write":
        out = {}
        top = _TOP[case["kept"]]
        keep = s["slots"] >= 0
        at = s["slots"][keep]
        for name in ("k", "v"):
            x = s[name][keep].double()
            scales = torch.clamp(x.abs().amax(-1) / top, min=_TINY)
            v = x / scales[..., None]
            cache = s[name + "_cache"].double()
            cache.view(-1, *x.shape[1:])[at] = v.round() if case["kept"] == "int8" else _nearest_e4m3(v)
            held = s[name + "_scales"].double()
            held.view(-1, x.shape[1])[at] = scales
            out[name + "_cache"], out[name + "_scales"] = cache, held
        return out
    starts, table = s["starts"].tolist(), s["table"].long()
    out = {}
    for name in ("k", "v"):
        parts = []
        for i in range(case["sequences"]):
            length = starts[i + 1] - starts[i]
            pages = table[i, : -(-length // page)]
            values = s[name + "_cache"][pages].double() * s[name + "_scales"][pages][..., None].double()
            parts.append(values.flatten(0, 1)[:length])
        out[name] = torch.cat(parts)
    return out
