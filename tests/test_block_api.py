# SPDX-License-Identifier: MIT
"""The 8-bit products and the quantised cache on the host: values, and what they refuse. Refusals
do not depend on the device: they come before anything runs."""

from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

import block_ref as ref
from rmsnorm import _lib, fused
from test_abi import _c_layout

E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------ values
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 129), (130, 257), (256, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize(rows, cols, dtype):
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows)).to(dtype)
    for block_rows in (1, 128):
        q, s, q_t, s_t = fused.block_quantize(x, block_rows, transposed=True)
        ref.check_quantized(q, s, x, block_rows)
        ref.check_quantized(q_t, s_t, x.t(), block_rows)


def test_quantize_ends_of_the_range():
    x = torch.zeros(5, 128)
    x[1], x[2], x[3, 0] = 448.0, 449.0, torch.finfo(torch.float32).max
    x[4, :2] = torch.tensor([1e-45, -1e-38])
    q, s = fused.block_quantize(x)
    ref.check_quantized(q, s, x, 1)
    assert s[:3, 0].tolist() == [2.0**-126, 1.0, 2.0]
    x[0, 3], x[1, 3] = float("nan"), float("inf")
    q, s = fused.block_quantize(x)
    assert s[0, 0].isnan() and s[1, 0].isinf() and q[1, 3].isnan() and (q[1, 4:].float() == 0).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_product(block_rows):
    a, sa = fused.block_quantize(torch.randn(2, 9, 200))
    b, sb = fused.block_quantize(torch.randn(150, 200), block_rows)
    bias = torch.randn(150)
    out = fused.block_mm(a, sa, b, sb, bias, torch.float32)
    assert out.shape == (2, 9, 150)
    ref.check_product(out.view(18, 150), ref.values(a.view(18, 200), sa.view(18, 2)), ref.values(b, sb), bias, "host")
    assert fused.block_mm(a, sa, b, sb).dtype == torch.bfloat16


def test_linear_gradients():
    x = torch.randn(20, 200, requires_grad=True)
    w = torch.randn(150, 200, requires_grad=True)
    b = torch.randn(150, requires_grad=True)
    dy = torch.randn(20, 150)
    y = fused.block_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    val = lambda t, rows: ref.values(*ref.quantize(t.detach(), rows))  # noqa: E731
    ref.check_product(y.detach(), val(x, 1), val(w, 128), b.detach(), "y")
    ref.check_product(dx, val(dy, 1), val(w, 128).t(), None, "dx")
    ref.check_product(dw, val(dy.t(), 1), val(x.t(), 1), None, "dw")
    assert torch.allclose(db, dy.sum(0))
    with pytest.raises(RuntimeError, match="second derivatives"):
        dx, = torch.autograd.grad(fused.block_linear(x, w, b).sum(), [x], create_graph=True)
        dx.sum().backward()


@pytest.mark.parametrize("kept", [E4M3, torch.int8])
@pytest.mark.parametrize("d", [5, 64])
def test_cache_round_trip(kept, d):
    k_cache, v_cache = (torch.zeros(6, 4, 2, d).to(kept) for _ in range(2))
    k_scales, v_scales = torch.zeros(6, 4, 2), torch.zeros(6, 4, 2)
    table = torch.tensor([[3, 1, -1], [0, -1, -1], [5, 2, 4]], dtype=torch.int32)
    starts = torch.tensor([0, 7, 7, 17], dtype=torch.int32)
    seq = torch.tensor([0] * 7 + [2] * 10)
    pos = torch.cat([torch.arange(7), torch.arange(10)])
    slots = table[seq, pos // 4] * 4 + pos % 4
    k, v = torch.randn(18, 2, d), torch.randn(18, 2, d)
    fused.cache_write(k, v, k_cache, v_cache, k_scales, v_scales, torch.cat([slots, torch.tensor([-1], dtype=torch.int32)]))
    at = slots.long()
    ref.check_cached(k_cache.view(24, 2, d)[at], k_scales.view(24, 2)[at], k[:17], 127.0 if kept == torch.int8 else 448.0)
    rk, rv = fused.cache_read(k_cache, v_cache, k_scales, v_scales, table, starts, 20, torch.float32)
    assert torch.equal(rk[:17], k_cache.view(24, 2, d)[at].float() * k_scales.view(24, 2, 1)[at])
    assert torch.equal(rv[:17], v_cache.view(24, 2, d)[at].float() * v_scales.view(24, 2, 1)[at])
    assert (rk[17:] == 0).all()
    out = (torch.full((20, 2, d), 3.0), torch.full((20, 2, d), 3.0))
    fused.cache_read(k_cache, v_cache, k_scales, v_scales, table, starts, 20, torch.float32, out)
    assert torch.equal(out[0][:17], rk[:17]) and (out[0][17:] == 3).all()


# ------------------------------------------------------------------ refusals
def test_quantize_refusals():
    x = torch.randn(4, 8)
    with pytest.raises(AssertionError, match="Unsupported dtype"):
        fused.block_quantize(x.double())
    with pytest.raises(ValueError, match="block_rows"):
        fused.block_quantize(x, 64)
    with pytest.raises(ValueError, match="matrix"):
        fused.block_quantize(x[None], 128)
    with pytest.raises(ValueError):
        fused.block_quantize(torch.randn(4, 0))
    with pytest.raises(ValueError):
        fused.block_quantize(torch.randn(()))


def test_product_refusals():
    a, sa = fused.block_quantize(torch.randn(4, 200))
    b, sb = fused.block_quantize(torch.randn(6, 200))
    bad = [
        (AssertionError, "float8", (a.float(), sa, b, sb)),
        (AssertionError, "float8", (a, sa, b.view(torch.int8), sb)),
        (AssertionError, "float32", (a, sa.double(), b, sb)),
        (AssertionError, "float32", (a, sa, b, sb.half())),
        (ValueError, "b must be", (a, sa, b[:, :100], sb)),
        (ValueError, "b must be", (a, sa, b[None], sb)),
        (ValueError, "b must be", (a, sa, b[:0], sb[:0])),
        (ValueError, "a_scales", (a, sa[:, :1], b, sb)),
        (ValueError, "a_scales", (a, sa[:3], b, sb)),
        (ValueError, "b_scales", (a, sa, b, sb[:2])),
        (ValueError, "b_scales", (a, sa, b, sb[:, :1])),
        (ValueError, "bias shape", (a, sa, b, sb, torch.randn(5))),
        (AssertionError, "Bias", (a, sa, b, sb, torch.randn(6).double())),
        (AssertionError, "out_dtype", (a, sa, b, sb, None, torch.float64)),
        (ValueError, "same device", (a, sa, b, sb, torch.randn(6, device="meta"))),
    ]
    for error, match, args in bad:
        with pytest.raises(error, match=match):
            fused.block_mm(*args)


def test_linear_refusals():
    x, w = torch.randn(4, 200), torch.randn(6, 200)
    with pytest.raises(AssertionError, match="X"):
        fused.block_linear(x.double(), w)
    with pytest.raises(AssertionError, match="Weight"):
        fused.block_linear(x, w.double())
    with pytest.raises(ValueError, match="weight must be"):
        fused.block_linear(x, w[:, :5])
    with pytest.raises(ValueError, match="weight must be"):
        fused.block_linear(x, w[:0])
    with pytest.raises(ValueError, match="bias shape"):
        fused.block_linear(x, w, torch.randn(4))


def _cache(d=16):
    return [torch.zeros(3, 4, 2, d).to(E4M3), torch.zeros(3, 4, 2, d).to(E4M3), torch.zeros(3, 4, 2), torch.zeros(3, 4, 2)]


def test_cache_refusals():
    c = _cache()
    k, slots = torch.randn(5, 2, 16), torch.arange(5)
    table, starts = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)

    def both(error, match, cache):
        with pytest.raises(error, match=match):
            fused.cache_write(k, k, *cache, slots)
        with pytest.raises(error, match=match):
            fused.cache_read(*cache, table, starts, 5)

    both(AssertionError, "float8_e4m3fn or int8", [c[0].float(), c[1], c[2], c[3]])
    both(AssertionError, "float8_e4m3fn or int8", [c[0], c[1].view(torch.int8), c[2], c[3]])
    both(ValueError, "pages, page_size", [c[0][0], c[1], c[2], c[3]])
    both(ValueError, "v_cache must have", [c[0], c[1][:2], c[2], c[3]])
    both(ValueError, "k_scales", [c[0], c[1], c[2].double(), c[3]])
    both(ValueError, "v_scales", [c[0], c[1], c[2], c[3][:, :3]])
    both(ValueError, "contiguous", [c[0].transpose(2, 3).contiguous().transpose(2, 3), c[1], c[2], c[3]])
    both(ValueError, "1 to", [t.to(E4M3) for t in (torch.zeros(1, 4, 2, 300),) * 2] + [torch.zeros(1, 4, 2)] * 2)
    both(ValueError, "same device", [c[0], c[1], c[2], c[3].to("meta")])
    bad = [
        (AssertionError, "same dtype", (k, k.half(), *c, slots)),
        (AssertionError, "same dtype", (k.double(), k.double(), *c, slots)),
        (ValueError, "two dimensions", (k[0, 0], k[0, 0], *c, slots)),
        (ValueError, "k must be", (k[:, :1], k, *c, slots)),
        (ValueError, "v must be", (k, k[:, :, :8], *c, slots)),
        (ValueError, "int32 or int64", (k, k, *c, slots.float())),
        (ValueError, "leading shape", (k, k, *c, slots[:4])),
        (ValueError, "places of their own", (k, k, c[0][:, :1].expand(3, 4, 2, 16), *c[1:], slots)),
        (IndexError, "beyond", (k, k, *c, slots + 8)),
    ]
    for error, match, args in bad:
        with pytest.raises(error, match=match):
            fused.cache_write(*args)
    with pytest.raises(ValueError, match="different"):
        fused.cache_write(k, k, c[0], c[0], c[2], c[3], slots)
    grad = [*c[:3], c[3].clone().requires_grad_(True)]
    with pytest.raises(ValueError, match="autograd"):
        fused.cache_write(k, k, *grad, slots)
    with torch.no_grad():
        fused.cache_write(k, k, *grad, slots)
    bad = [
        ("page_table", (*c, table.long(), starts, 5)),
        ("page_table", (*c, table[0], starts, 5)),
        ("starts", (*c, table, starts.long(), 5)),
        ("starts", (*c, table, starts[:2], 5)),
        ("negative", (*c, table, starts, -1)),
        ("out must be", (*c, table, starts, 5, torch.bfloat16, (k, k.clone()))),
        ("out must be", (*c, table, starts, 5, torch.float32, (k[:4], k.clone()))),
        ("different", (*c, table, starts, 5, torch.float32, (k, k))),
        ("same device", (*c, table.to("meta"), starts, 5)),
    ]
    for match, args in bad:
        with pytest.raises(ValueError, match=match):
            fused.cache_read(*args)
    with pytest.raises(AssertionError, match="dtype"):
        fused.cache_read(*c, table, starts, 5, torch.float64)
    with pytest.raises(IndexError):
        fused.cache_read(*c, table + 3, torch.tensor([0, 2, 4], dtype=torch.int32), 5)


# ------------------------------------------------------------------ C ABI
@pytest.mark.parametrize("cls,cname", [
    (_lib.BlockQuantArgs, "rmsnorm_b200_block_quant_args"), (_lib.BlockMmArgs, "rmsnorm_b200_block_mm_args"),
    (_lib.CacheTensor, "rmsnorm_b200_cache_tensor"), (_lib.CacheArgs, "rmsnorm_b200_cache_args"),
    (_lib.CacheWriteArgs, "rmsnorm_b200_cache_write_args"), (_lib.CacheReadArgs, "rmsnorm_b200_cache_read_args")])
def test_struct_layouts_match_c(cls, cname, tmp_path):
    fields = [f[0] for f in cls._fields_]
    c = tmp_path / "probe.c"
    c.write_text(_c_layout(cname, fields))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-o", str(exe), str(c)], check=True)
    vals = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(cls)
    for name, off in zip(fields, vals[1:]):
        assert getattr(cls, name).offset == off, name


def test_c_entries_check_their_arguments():
    lib = _lib.load_library()
    n = ctypes.c_size_t(1)
    ok = dict(rows=4, cols=200, x=0x1000, x_row_stride=200, q=0x2000, q_row_stride=208, scales=0x3000, scale_row_stride=2,
              scale_group_stride=1, x_dtype=1, block_rows=1)
    for change in (dict(rows=-1), dict(cols=0), dict(x=0), dict(q=0), dict(scales=0), dict(x_dtype=3), dict(block_rows=2),
                   dict(q_row_stride=199), dict(x_row_stride=-1), dict(q_t=0x4000), dict(q_t=0x4000, scales_t=0x5000, q_t_row_stride=3),
                   dict(column_sums=0x4000, column_sums_dtype=9), dict(scale_row_stride=-2)):
        a = _lib.BlockQuantArgs(**{**ok, **change})
        assert lib.rmsnorm_b200_block_quant(ctypes.byref(a), None, 0, None) == 1, change
        assert lib.rmsnorm_b200_block_quant_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 1, change
    assert lib.rmsnorm_b200_block_quant(None, None, 0, None) == 1
    a = _lib.BlockQuantArgs(**{**ok, "rows": 0})
    assert lib.rmsnorm_b200_block_quant(ctypes.byref(a), None, 0, None) == 0
    a = _lib.BlockQuantArgs(**ok, column_sums=0x4000, column_sums_dtype=2)
    assert lib.rmsnorm_b200_block_quant_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value == 800
    assert lib.rmsnorm_b200_block_quant(ctypes.byref(a), None, 0, None) not in (0, 1)  # no workspace

    ok = dict(m=4, n=8, k=200, a=0x1000, a_row_stride=208, b=0x2000, b_row_stride=208, a_scales=0x3000, a_scale_row_stride=2,
              a_scale_group_stride=1, b_scales=0x4000, b_scale_row_stride=2, b_scale_group_stride=1, out=0x5000, b_block_rows=1,
              out_dtype=1)
    for change in (dict(m=-1), dict(n=0), dict(k=0), dict(k=1 << 31), dict(m=1 << 31), dict(a=0), dict(b=0), dict(a_scales=0),
                   dict(b_scales=0), dict(out=0), dict(b_block_rows=64), dict(out_dtype=3), dict(bias=0x6000, bias_dtype=7),
                   dict(a_row_stride=199), dict(b_row_stride=-1), dict(b_scale_row_stride=-1)):
        a = _lib.BlockMmArgs(**{**ok, **change})
        assert lib.rmsnorm_b200_block_mm(ctypes.byref(a), None, 0, None) == 1, change
    assert lib.rmsnorm_b200_block_mm(None, None, 0, None) == 1
    a = _lib.BlockMmArgs(**{**ok, "m": 0})
    assert lib.rmsnorm_b200_block_mm(ctypes.byref(a), None, 0, None) == 0
    a = _lib.BlockMmArgs(**{**ok, "a_row_stride": 200})
    assert lib.rmsnorm_b200_block_mm_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value == 4 * 208

    side = dict(data=0x1000, page_stride=64, slot_stride=32, head_stride=16, scales=0x2000, scale_page_stride=4,
                scale_slot_stride=2, scale_head_stride=1)
    cache = dict(pages=3, page_size=2, heads=2, head_dim=16, cache_dtype=3)
    token = dict(data=0x3000, token_stride=32, head_stride=16)

    def make(change=(), k=(), write=(), read=()):
        t = _lib.CacheTensor(**{**side, **dict(k)})
        c = _lib.CacheArgs(k=t, v=_lib.CacheTensor(**side), **{**cache, **dict(change)})
        h = _lib.RopeTensor(**token)
        w = _lib.CacheWriteArgs(**{**dict(tokens=5, k=h, v=h, slots=0x4000, dtype=1), **dict(write)})
        r = _lib.CacheReadArgs(**{**dict(tokens=5, sequences=1, table_width=3, table_stride=3, page_table=0x5000,
                                         starts=0x6000, k=0x7000, v=0x8000, dtype=1), **dict(read)})
        return (lib.rmsnorm_b200_cache_write(ctypes.byref(c), ctypes.byref(w), None),
                lib.rmsnorm_b200_cache_read(ctypes.byref(c), ctypes.byref(r), None))

    for change in (dict(pages=-1), dict(pages=1 << 31), dict(page_size=0), dict(heads=0), dict(heads=65537), dict(head_dim=0),
                   dict(head_dim=257), dict(cache_dtype=1)):
        assert make(change) == (1, 1), change
    for change in (dict(data=0), dict(scales=0), dict(page_stride=-1), dict(scale_head_stride=-1)):
        assert make(k=change) == (1, 1), change
    for change in (dict(tokens=-1), dict(slots=0), dict(dtype=3), dict(k=_lib.RopeTensor(data=0)),
                   dict(v=_lib.RopeTensor(data=0x3000, token_stride=-1))):
        assert make(write=change)[0] == 1, change
    for change in (dict(tokens=-1), dict(sequences=-1), dict(table_width=-1), dict(table_stride=-1), dict(starts=0), dict(k=0),
                   dict(v=0), dict(page_table=0), dict(dtype=4)):
        assert make(read=change)[1] == 1, change
    assert make(write=dict(tokens=0), read=dict(tokens=0)) == (0, 0)


def test_untraced_under_compile():
    """A graph break each, as the other fused operators."""
    x, w = torch.randn(6, 200), torch.randn(5, 200)
    k, slots = torch.randn(5, 2, 16), torch.arange(5)

    def f(x):
        q, s = fused.block_quantize(x + 0)
        b, sb = fused.block_quantize(w, 128)
        c = _cache()
        fused.cache_write(k, k, *c, slots)
        r = fused.cache_read(*c, torch.arange(3, dtype=torch.int32)[None], torch.tensor([0, 5], dtype=torch.int32), 5)
        return fused.block_mm(q, s, b, sb) + 1, fused.block_linear(x, w) * 2, r[0]

    for got, want in zip(torch.compile(f, backend="eager")(x), f(x)):
        assert torch.equal(got, want)


def test_product_of_expanded_and_overlapping_rows():
    a, sa = fused.block_quantize(torch.randn(1, 128))
    b, sb = fused.block_quantize(torch.randn(6, 128))
    out = fused.block_mm(a.expand(4, 128), sa.expand(4, 1), b, sb, out_dtype=torch.float32)
    # The values are exact in fp32, and so are their products (4 bits by 4, powers of two as scales).
    # One row and four may be summed in different orders on the host: each sum of 128 is off by at
    # most 127 u / (1 - 127 u) times the sum of magnitudes, u = 2^-24, two differ by less than 256 u of it.
    values = (q.double() * s.double() for q, s in ((a, sa), (b, sb)))
    bound = 256 * 2.0**-24 * torch.mm(*(v.abs() if i == 0 else v.abs().t() for i, v in enumerate(values)))
    assert ((out - fused.block_mm(a, sa, b, sb, out_dtype=torch.float32).expand(4, 6)).abs() <= bound).all()


def test_cache_write_refuses_one_tensor_for_both_scales():
    k_cache, v_cache, scales, _ = _cache()
    x = torch.randn(3, *k_cache.shape[2:])
    with pytest.raises(ValueError, match="k_scales and v_scales must be different"):
        fused.cache_write(x, x, k_cache, v_cache, scales, scales, torch.arange(3))


def test_quantised_values_are_outside_autograd():
    assert not any(t.requires_grad for t in fused.block_quantize(torch.randn(5, 130, requires_grad=True), transposed=True))


def test_linear_without_gradients_quantises_nothing_for_them(monkeypatch):
    from rmsnorm import _block

    wanted, quantize = [], _block._quantize
    monkeypatch.setattr(_block, "_quantize", lambda x, rows, want, want_t, *a: wanted.append(want_t) or quantize(x, rows, want, want_t, *a))
    x, w = torch.randn(3, 130, requires_grad=True), torch.randn(7, 130, requires_grad=True)
    y = fused.block_linear(x, w)
    with torch.no_grad():
        assert torch.equal(fused.block_linear(x, w), y)
    assert wanted == [True, True, False, False]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_products_do_not_depend_on_autocast(dtype):
    """Their sums are fp32 whatever mode another part of the program has set, as they are on CUDA."""
    g = torch.Generator().manual_seed(0)
    x, w, dy = (torch.randn(*s, generator=g) for s in ((8, 256), (4, 256), (8, 4)))
    a, sa = fused.block_quantize(x)
    b, sb = fused.block_quantize(w)

    def results():
        out = [fused.block_mm(a, sa * f, b, sb * f, out_dtype=torch.float32) for f in (1.0, 1.1)]  # powers of two and none
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        y = fused.block_linear(*leaves)
        return [*out, y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = results()
    with torch.autocast("cpu", dtype=dtype):
        got = results()
    assert all(i.dtype == j.dtype and torch.equal(i, j) for i, j in zip(got, want))


@pytest.mark.parametrize("starts,sequences", [([1, 10], 1), ([3, 3, 9], 2), ([2], 0)])
def test_cache_read_refuses_rows_before_the_first_sequence(starts, sequences):
    """On CUDA they are NaN and the device status tells; on the host, like a page outside the table, an error."""
    c = _cache()
    table = torch.zeros(sequences, 3, dtype=torch.int32)
    with pytest.raises(IndexError, match="first"):
        fused.cache_read(*c, table, torch.tensor(starts, dtype=torch.int32), 12)
    assert fused.cache_read(*c, table, torch.tensor(starts, dtype=torch.int32), 0)[0].shape == (0, 2, 16)
    nothing = torch.zeros(sequences + 1, dtype=torch.int32)
    assert (fused.cache_read(*c, table, nothing, 12)[0] == 0).all()


def _halves(shape, *axes, dtype=torch.float32):
    """k's and v's part of one buffer, in every place that the axis of both can have."""
    for axis in axes:
        both = torch.zeros(*shape[:axis], 2, *shape[axis:]).to(dtype)
        yield both.select(axis, 0), both.select(axis, 1)


def test_cache_write_takes_caches_that_share_a_buffer():
    shape, slots = (3, 4, 2, 16), torch.tensor([0, 5, 11, 7, 2])
    k, v = torch.randn(5, 2, 16), torch.randn(5, 2, 16)
    want = _cache()
    fused.cache_write(k, v, *want, slots)
    wide = torch.zeros(3, 4, 2, 32).to(E4M3)
    across = torch.zeros(2, 4, 3, 2, 16).to(E4M3).transpose(1, 2)  # slots before pages
    for kc, vc in [*_halves(shape, 0, 1, 2, 3, dtype=E4M3), wide.split(16, -1), across]:
        for ks, vs in [(torch.zeros(3, 4, 2), torch.zeros(3, 4, 2)), *_halves(shape[:3], 0, 1, 2, 3)]:
            fused.cache_write(k, v, kc, vc, ks, vs, slots)
            got = (kc, vc, ks, vs)
            assert all(torch.equal(i.float(), j.float()) for i, j in zip(got, want))


def test_cache_write_refuses_caches_that_overlap():
    k, slots = torch.randn(5, 2, 16), torch.arange(5)
    c = _cache()
    pages = torch.zeros(5, 4, 2, 16).to(E4M3)
    slots_apart = torch.zeros(4, 8, 2, 16).to(E4M3)
    columns = torch.zeros(3, 4, 2, 31).to(E4M3)
    across = torch.zeros(4, 4, 2, 16).to(E4M3).transpose(0, 1)[:, 1:]
    for kc, vc in [(pages[:3], pages[1:4]), (pages[:3], pages[2:]), (slots_apart[:3, :4], slots_apart[:3, 3:7]),
                   (slots_apart[:3, 4:], slots_apart[1:, 4:]), (columns[..., :16], columns[..., 15:]),
                   (across, torch.as_strided(across, across.shape, across.stride(), 0))]:
        c2, c3 = (torch.zeros(kc.shape[:3]) for _ in range(2))
        for one, other in ((kc, vc), (vc, kc)):
            with pytest.raises(ValueError, match="k_cache and v_cache must"):
                fused.cache_write(k, k, one, other, c2, c3, slots)
    scales = torch.zeros(5, 4, 2)
    for ks, vs in [(scales[:3], scales[1:4]), (scales[:3], scales[2:])]:
        with pytest.raises(ValueError, match="k_scales and v_scales must"):
            fused.cache_write(k, k, *c[:2], ks, vs, slots)


def test_cache_read_refuses_outputs_that_overlap():
    c = _cache()
    table, starts = torch.zeros(1, 3, dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    both = torch.zeros(10, 2, 16)
    for k, v in ((both[:5], both[1:6]), (both[4:9], both[:5])):
        with pytest.raises(ValueError, match="overlap"):
            fused.cache_read(*c, table, starts, 5, torch.float32, (k, v))
    fused.cache_read(*c, table, starts, 5, torch.float32, (both[5:], both[:5]))
