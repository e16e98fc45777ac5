# SPDX-License-Identifier: MIT
"""The 8-bit products and their quantisation against 64 bits (tests/block_ref.py has the error
bounds)."""

from __future__ import annotations

import pytest
import torch

import block_ref as ref
from rmsnorm import _lib, fused

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _status_stays_clear():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status(DEV) == (0, 0)


def rand(*shape, dtype=F32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 7), (127, 129), (128, 128), (129, 127), (300, 1001), (1, 5000),
                                       (2000, 16), (16, 2000), (1000, 4096)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize(rows, cols, dtype, block_rows):
    x = rand(rows, cols, dtype=dtype, seed=rows + cols)
    x[0] *= 100
    q, s = fused.block_quantize(x, block_rows)
    ref.check_quantized(q, s, x, block_rows)
    q, s, q_t, s_t = fused.block_quantize(x, block_rows, transposed=True)
    ref.check_quantized(q, s, x, block_rows)
    ref.check_quantized(q_t, s_t, x.t(), block_rows)
    assert all(t.stride(0) % 16 == 0 or t.shape[0] == 1 for t in (q, q_t))


@pytest.mark.parametrize("rows,cols,pitch,at", [(3000, 4096, 4096, 0), (3001, 4200, 4208, 8), (3001, 4201, 4201, 0), (3001, 4096, 4104, 4)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_quantize_many_groups(rows, cols, pitch, at, dtype):
    """Enough of them for whole tiles: aligned, ragged, without vectors, from rows that start off a vector."""
    x = rand(rows * pitch + at, dtype=dtype, seed=cols)[at:].view(rows, pitch)[:, :cols]
    ref.check_quantized(*fused.block_quantize(x), x, 1)


def test_quantize_ends_of_the_range():
    """Zeros, the largest and smallest numbers, a maximum that is a power of two times 448."""
    x = torch.zeros(6, 256, device=DEV)
    x[1, :128], x[1, 128:] = 448.0, 449.0
    x[2] = torch.finfo(F32).max
    x[3] = torch.finfo(F32).tiny
    x[4, 3], x[4, 200] = 1e-45, -1e-38
    x[5, 0], x[5, 1], x[5, 2] = 448 * 2.0**-20, 8.5 * 2.0**-20, 9.5 * 2.0**-20  # ties of 16 and 8 steps
    for transposed in (False, True):
        q, s = fused.block_quantize(x, transposed=transposed)[:2]
        ref.check_quantized(q, s, x, 1)
    assert s[0, 0] == 2.0**-126 and s[1, 0] == 1 and s[1, 1] == 2
    q, s = fused.block_quantize(x, 128)
    ref.check_quantized(q, s, x, 128)


@pytest.mark.parametrize("transposed", [False, True])
def test_quantize_nan_and_infinity(transposed):
    x = rand(130, 300, seed=4)
    x[0, 5], x[2, 130], x[3, 299] = float("nan"), float("inf"), float("-inf")
    q, s = fused.block_quantize(x, transposed=transposed)[:2]
    assert s[0, 0].isnan() and s[2, 1].isinf() and s[3, 2].isinf()
    assert q[2, 130].double().isnan() and (q[2, 131:256].double() == 0).all()
    fine = torch.ones(130, dtype=torch.bool, device=DEV)
    fine[[0, 2, 3]] = False
    ref.check_quantized(q[fine], s[fine], x[fine], 1)
    if transposed:
        q_t, s_t = fused.block_quantize(x, transposed=True)[2:]
        assert s_t[5, 0].isnan() and s_t[130, 0].isinf() and s_t[299, 0].isinf() and int(s_t.isfinite().sum()) == s_t.numel() - 3


def test_quantize_shapes_strides_and_layouts():
    x = rand(4, 70, 256, dtype=BF16)
    q, s, q_t, s_t = fused.block_quantize(x, transposed=True)
    assert q.shape == x.shape and s.shape == (4, 70, 2) and q_t.shape == (256, 280) and s_t.shape == (256, 3)
    ref.check_quantized(q.view(280, 256), s.view(280, 2), x.view(280, 256), 1)
    ref.check_quantized(q_t, s_t, x.view(280, 256).t(), 1)
    q2, s2 = fused.block_quantize(x, scales_column_major=True)
    assert torch.equal(s2, s) and torch.equal(q2.double(), q.double()) and s2.stride()[-1] == 280
    one = rand(100)
    q, s = fused.block_quantize(one)
    assert q.shape == (100,) and s.shape == (1,)
    ref.check_quantized(q[None], s[None], one[None], 1)
    odd = rand(3, 5, 33)
    q, s = fused.block_quantize(odd)
    assert q.shape == (3, 5, 33) and s.shape == (3, 5, 1)
    ref.check_quantized(q.reshape(15, 33), s.view(15, 1), odd.view(15, 33), 1)
    wide = rand(200, 600, dtype=F16)
    for view in (wide[:, 100:400], wide[::2, :300], wide[:, 1:258], wide.t(), wide[:1].expand(50, 600)):
        q, s, q_t, s_t = fused.block_quantize(view, transposed=True)
        ref.check_quantized(q, s, view, 1)
        ref.check_quantized(q_t, s_t, view.t(), 1)
    for empty in (rand(0, 128), rand(2, 0, 5)):
        q, s, q_t, s_t = fused.block_quantize(empty, transposed=True)
        assert q.shape == empty.shape and q_t.shape == (empty.shape[-1], 0) and s_t.shape == (empty.shape[-1], 0)


# ------------------------------------------------------------------ product
def operand(rows, k, block_rows, seed, spread=4.0):
    """e4m3 numbers of all sizes and scales that are no powers of two, over some octaves."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randint(-126, 127, (rows, k), device=DEV, generator=g)
    q = (q.abs() + (q < 0) * 128).to(torch.uint8).view(E4M3)
    s = torch.exp2(spread * (torch.rand(-(-rows // block_rows), -(-k // 128), device=DEV, generator=g) - 0.5)) / 448
    return q, s


def product_case(m, n, k, block_rows, out_dtype, bias=True, change_a=lambda t: t, change_b=lambda t: t, change_s=lambda t: t):
    a, sa = operand(m, k, 1, 1)
    b, sb = operand(n, k, block_rows, 2)
    bias = rand(n, seed=3) if bias else None
    out = fused.block_mm(change_a(a), change_s(sa), change_b(b), change_s(sb), bias, out_dtype)
    assert out.dtype == out_dtype and out.shape == (m, n)
    ref.check_product(out, ref.values(a, sa), ref.values(b, sb), bias, f"{m}x{n}x{k}")


# every tile of rows, ragged ones, splits over k and none, one group to many
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 257, 500])
@pytest.mark.parametrize("n,k", [(1, 1), (8, 16), (127, 129), (128, 128), (130, 1000), (520, 2049), (4100, 512)])
def test_product_sizes(m, n, k):
    for block_rows in (1, 128):
        product_case(m, n, k, block_rows, F32)


@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (40, 1000, 4096), (1000, 1040, 640), (777, 4100, 384), (300, 5000, 1001)])
@pytest.mark.parametrize("bias", [False, True])
def test_product_types(out_dtype, m, n, k, bias):
    for block_rows in (1, 128):
        product_case(m, n, k, block_rows, out_dtype, bias)


@pytest.mark.parametrize("m,n,k", [(1, 128, 200000), (300, 260, 70000), (64, 16384, 300), (20000, 128, 256), (3000, 20000, 128)])
def test_product_long_and_wide(m, n, k):
    product_case(m, n, k, 128, BF16, False)


def test_product_many_tiles_use_every_stage_again():
    product_case(2500, 9000, 1152, 128, BF16, False)
    product_case(2500, 9000, 1152, 1, F32, True)


def padded(t):
    """The same values in rows that begin at multiples of 16 bytes."""
    pitch = -(-t.shape[1] // 16) * 16 + 16
    buf = torch.zeros(t.shape[0], pitch, dtype=torch.uint8, device=DEV).view(E4M3)
    buf[:, : t.shape[1]] = t
    return buf[:, : t.shape[1]]


def shifted(t):
    """The same values one byte past a 16-byte boundary."""
    buf = torch.zeros(t.numel() + 16, dtype=torch.uint8, device=DEV)[1: 1 + t.numel()].view(t.shape).view(E4M3)
    buf.copy_(t)
    return buf


@pytest.mark.parametrize("m,n", [(1, 100), (48, 300), (130, 129), (600, 5000)])
@pytest.mark.parametrize("k", [16, 100, 640, 1001])
def test_product_strides_and_alignment(m, n, k):
    flip = lambda t: t.t().contiguous().t()  # noqa: E731 -- column by column
    product_case(m, n, k, 128, F32, True, padded, shifted, flip)
    product_case(m, n, k, 1, BF16, False, shifted, padded, flip)
    product_case(m, n, k, 1, F16, True, flip, flip)


def test_product_of_norm_outputs_and_leading_dimensions():
    x, w = rand(3, 50, 640, dtype=BF16, seed=1), rand(640, seed=2)
    weight = rand(200, 640, seed=3)
    q, s, _ = fused.rmsnorm_quant_fwd(x, w, group_size=128, scales_column_major=True)
    wq, ws = fused.block_quantize(weight, 128)
    out = fused.block_mm(q, s, wq, ws, out_dtype=F32)
    assert out.shape == (3, 50, 200)
    ref.check_product(out.view(150, 200), ref.values(q.view(150, 640), s.reshape(150, 5)), ref.values(wq, ws), None, "norm")
    one = fused.block_mm(q[0, 0], s[0, 0], wq, ws, out_dtype=F32)
    assert one.shape == (200,) and torch.equal(one, fused.block_mm(q[0, :1], s[0, :1], wq, ws, out_dtype=F32)[0])
    assert fused.block_mm(q[:0], s[:0], wq, ws).shape == (0, 50, 200)


def test_product_of_expanded_and_overlapping_rows():
    a, sa = operand(1, 256, 1, 1)
    b, sb = operand(300, 256, 1, 2)
    out = fused.block_mm(a.expand(40, 256), sa.expand(40, 2), b, sb[:1].expand(300, 2), out_dtype=F32)
    ref.check_product(out, ref.values(a, sa).expand(40, 256), ref.values(b, sb[:1].expand(300, 2)), None, "expanded")
    long, _ = operand(1, 400, 1, 3)
    windows = long.as_strided((20, 256), (7, 1))
    out = fused.block_mm(windows, sa.expand(20, 2), b, sb, out_dtype=F32)
    ref.check_product(out, ref.values(windows.contiguous(), sa.expand(20, 2)), ref.values(b, sb), None, "windows")


def test_product_bias_types():
    a, sa = operand(200, 256, 1, 1)
    b, sb = operand(333, 256, 128, 2)
    for dtype in (BF16, F16, F32):
        for m in (5, 200):
            bias = rand(333, dtype=dtype)
            out = fused.block_mm(a[:m], sa[:m], b, sb, bias, F32)
            ref.check_product(out, ref.values(a[:m], sa[:m]), ref.values(b, sb), bias, "bias")


@pytest.mark.parametrize("m", [3, 100, 400])
def test_product_nan_stays_in_its_row_and_column(m):
    a, sa = operand(m, 300, 1, 1)
    b, sb = operand(700, 300, 1, 2)
    a.view(torch.uint8)[1, 7] = 0x7F  # NaN
    sb[5, 2] = float("nan")
    out = fused.block_mm(a, sa, b, sb, out_dtype=F32)
    nan = out.isnan()
    assert nan[1].all() and nan[:, 5].all() and int(nan.sum()) == m + 700 - 1
    # zeros times what lies behind the matrices stay zeros
    a.zero_()
    out = fused.block_mm(a, sa, b[:5], sb[:5], out_dtype=F32)
    assert (out == 0).all()


def test_product_results_do_not_depend_on_the_run():
    for m in (1, 64, 128, 3000):
        a, sa = operand(m, 4096, 1, 1)
        b, sb = operand(1024, 4096, 128, 2)
        first = fused.block_mm(a, sa, b, sb, out_dtype=F32)
        for _ in range(3):
            assert torch.equal(fused.block_mm(a, sa, b, sb, out_dtype=F32), first)


def test_product_on_streams_and_in_graphs():
    """Two streams at once, and two captured graphs replayed at once: nothing is shared."""
    sets = [(*operand(m, k, 1, 10 + i), *operand(1000, k, 128, 20 + i)) for i, (m, k) in enumerate([(64, 1001), (300, 1001)])]
    want = [fused.block_mm(*s, out_dtype=F32) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[] for _ in sets]
    for _ in range(5):
        for s, st, o in zip(sets, streams, outs):
            with torch.cuda.stream(st):
                o.append(fused.block_mm(*s, out_dtype=F32))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for o, w in zip(outs, want) for x in o)
    graphs, results = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(fused.block_mm(*s, out_dtype=F32))
        graphs.append(g)
    for _ in range(3):
        for r in results:
            r.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(r, w) for r, w in zip(results, want))


# ------------------------------------------------------------------ scales left to the tensor cores
def power_case(m, n, k, block_rows, out_dtype, bias=True, column_major=False):
    """Scales over many octaves, that differ from row to row and from group to group."""
    a, _ = operand(m, k, 1, 1)
    b, _ = operand(n, k, block_rows, 2)
    g = torch.Generator(device=DEV).manual_seed(5)
    groups = -(-k // 128)
    sa = torch.exp2(torch.randint(-14, -5, (m, groups), device=DEV, generator=g).float())
    sb = torch.exp2(torch.randint(-14, -5, (-(-n // block_rows), groups), device=DEV, generator=g).float())
    if column_major:
        sa, sb = sa.t().contiguous().t(), sb.t().contiguous().t()
    bias = rand(n, seed=3) if bias else None
    out = fused.block_mm(a, sa, b, sb, bias, out_dtype, power_of_two=True)
    assert out.dtype == out_dtype and out.shape == (m, n)
    ref.check_product(out, ref.values(a, sa), ref.values(b, sb), bias, f"{m}x{n}x{k}", True)


# tiles of 256, 224 and 192 columns: one round of them, two, several; ragged ones; one group to many
@pytest.mark.parametrize("m,n,k", [(129, 9600, 100), (200, 20000, 128), (300, 12345, 700), (1000, 4096, 2048), (1024, 4100, 512),
                                   (600, 4096, 1001), (2300, 5000, 1280), (4096, 1024, 640), (5000, 3000, 300), (257, 19000, 130)])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_powers_of_two(m, n, k, out_dtype):
    power_case(m, n, k, 128, out_dtype, False)
    power_case(m, n, k, 1, out_dtype, True, True)


@pytest.mark.parametrize("m", [1, 16, 40, 100, 200])
def test_powers_of_two_of_few_rows(m):
    power_case(m, 1000, 1024, 128, BF16)
    power_case(m, 130, 2000, 1, F16)


def test_powers_of_two_tiles_are_what_the_test_means_them_to_be():
    tiles = set()
    for m, n, k in [(1000, 4096, 2048), (2300, 5000, 1280), (600, 4096, 1001)]:
        power_case(m, n, k, 128, BF16)
        plan = _lib.last_plan()
        assert plan.startswith("block_mm_scaled"), plan
        tiles.add(plan.split("tile=")[1].split()[0])
    assert tiles == {"192", "224", "256"}, tiles


def test_powers_of_two_at_the_ends_of_the_range():
    a, b = (torch.full((300, 128), v, device=DEV).to(E4M3) for v in (448.0, 1.0))
    b = b.repeat(40, 1)
    low, high = (torch.full((300, 1), 2.0**e, device=DEV) for e in (-126, 120))
    sb = torch.ones(94, 1, device=DEV)
    out = fused.block_mm(a, high * 2.0**-110, b, sb * 2.0**-10, None, BF16, power_of_two=True)
    assert (out == 448 * 128).all()
    out = fused.block_mm(a, low, b, sb * 2.0**100, None, BF16, power_of_two=True)
    assert (out.double() == 448 * 128 * 2.0**-26).all()
    out = fused.block_mm(a, high, b, sb * 2.0**-126, None, BF16, power_of_two=True)
    assert (out.double() == 448 * 128 * 2.0**-6).all()
    sa = torch.ones(300, 1, device=DEV)
    sa[7], sb[3] = float("nan"), float("inf")
    nan = fused.block_mm(a, sa, b, sb, None, BF16, power_of_two=True).isnan()
    assert nan[7].all() and nan[:, 384:512].all() and int(nan.sum()) == 12000 + 299 * 128


def test_powers_of_two_do_not_depend_on_the_run_and_replay():
    x, w = rand(1500, 1024, dtype=BF16), rand(5000, 1024, dtype=BF16, seed=1)
    a, sa = fused.block_quantize(x)
    b, sb = fused.block_quantize(w, 128)
    first = fused.block_mm(a, sa, b, sb, power_of_two=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fused.block_mm(a, sa, b, sb, power_of_two=True)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        outs = []
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                outs.append(fused.block_mm(a, sa, b, sb, power_of_two=True))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, first) for o in (*outs, out))


# ------------------------------------------------------------------ linear layer
def linear_reference(x, w, b, dy):
    """y, dx, dw as pairs of 64-bit factors, db."""
    val = lambda t, rows: (lambda q, s: ref.values(q, s))(*ref.quantize(t, rows))  # noqa: E731
    wv = val(w, 128)
    return (val(x, 1), wv), (val(dy, 1), wv.t()), (val(dy.t(), 1), val(x.t(), 1))


@pytest.mark.parametrize("t,n,k", [(1, 8, 16), (7, 100, 300), (128, 256, 384), (333, 520, 1001), (1500, 1300, 640),
                                   (3000, 2500, 2304)])
@pytest.mark.parametrize("dtype,w_dtype", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32)])
def test_linear(t, n, k, dtype, w_dtype):
    x = rand(t, k, dtype=dtype, seed=1).requires_grad_(True)
    w = (rand(n, k, seed=2) * k**-0.5).to(w_dtype).requires_grad_(True)
    b = rand(n, seed=3).requires_grad_(True)
    dy = rand(t, n, dtype=dtype, seed=4)
    y = fused.block_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    fy, fdx, fdw = linear_reference(x.detach(), w.detach(), b.detach(), dy)
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == w_dtype and db.dtype == F32
    ref.check_product(y.detach(), *fy, b.detach(), "y", True)
    ref.check_product(dx, *fdx, None, "dx", True)
    ref.check_product(dw, *fdw, None, "dw", True)
    off = (db.double() - dy.double().sum(0)).abs()
    assert (off <= (t + 8) * 2.0**-24 * dy.double().abs().sum(0) + 2.0**-140).all()


def test_linear_wanted_gradients_and_shapes():
    x, w = rand(4, 30, 256, dtype=BF16), rand(192, 256, dtype=BF16, seed=1)
    b = rand(192, dtype=BF16, seed=2)
    dy = rand(4, 30, 192, dtype=BF16, seed=3)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(fused.block_linear(*full), full, dy)
    assert want[0].shape == x.shape and want[1].shape == w.shape and want[2].shape == b.shape
    for which in range(3):
        some = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(fused.block_linear(*some), [some[which]], dy)
        assert torch.equal(got, want[which])
    # a gradient that is one expanded value, as sum() sends
    a = [t.clone().requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(fused.block_linear(*a).sum(), a)
    c = [t.clone().requires_grad_(True) for t in (x, w)]
    again = torch.autograd.grad(fused.block_linear(*c), c, torch.ones_like(dy))
    assert all(torch.equal(i, j) for i, j in zip(got, again))
    with torch.no_grad():
        assert torch.equal(fused.block_linear(x, w, b), fused.block_linear(*full).detach())


def test_linear_of_no_rows():
    x, w, b = rand(0, 256).requires_grad_(True), rand(100, 256).requires_grad_(True), rand(100).requires_grad_(True)
    y = fused.block_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], rand(0, 100))
    assert y.shape == (0, 100) and dx.shape == (0, 256) and (dw == 0).all() and (db == 0).all()


def test_linear_second_derivatives_are_refused():
    x, w = rand(8, 128).requires_grad_(True), rand(16, 128).requires_grad_(True)
    dx, = torch.autograd.grad(fused.block_linear(x, w).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        dx.sum().backward()


def test_products_one_behind_the_other_share_tensor_memory():
    """Each may start before the one before it has ended; small ones of a single group fit beside a
    large one on an SM, whose tensor memory they cannot share."""
    a, sa = operand(2000, 128, 1, 1)
    b, sb = operand(3000, 128, 128, 2)
    (a2, sa2), (b2, sb2) = fused.block_quantize(rand(2000, 256, seed=3)), fused.block_quantize(rand(3000, 256, seed=4), 128)
    want = fused.block_mm(a[:8], sa[:8], b, sb), fused.block_mm(a2, sa2, b2, sb2, power_of_two=True), fused.block_mm(a2, sa2, b2, sb2)
    for _ in range(40):
        got = (fused.block_mm(a[:8], sa[:8], b, sb), fused.block_mm(a2, sa2, b2, sb2, power_of_two=True),
               fused.block_mm(a[:8], sa[:8], b, sb), fused.block_mm(a2, sa2, b2, sb2))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[0]) and torch.equal(got[3], want[2])


def test_linear_captured_and_replayed():
    x, w = rand(200, 512, dtype=BF16).requires_grad_(True), rand(384, 512, dtype=BF16, seed=1).requires_grad_(True)
    dy = rand(200, 384, dtype=BF16, seed=2)
    want = torch.autograd.grad(fused.block_linear(x, w), [x, w], dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(fused.block_linear(x, w), [x, w], dy)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(fused.block_linear(x, w), [x, w], dy)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(i, j) for i, j in zip(got, want))


def test_linear_gradient_against_differences():
    """Along weights whose quantised values move by whole steps the loss changes as the gradient
    says: x and weight hold e4m3 numbers times powers of two, so the layer is exact."""
    x = torch.randint(-8, 9, (40, 256), device=DEV).float()
    w = torch.randint(-8, 9, (24, 256), device=DEV).float()
    x[:, ::128], w[:, ::128] = 8.0, 8.0  # every group's and block's scale stays where it is
    g = torch.randint(-8, 9, (40, 24), device=DEV).float()
    g[:, 0], g[0, :] = 8.0, 8.0
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = fused.block_linear(xr, wr)
    assert torch.equal(y.double(), x.double() @ w.double().t())
    dx, dw = torch.autograd.grad(y, [xr, wr], g)
    move = torch.randint(-1, 2, w.shape, device=DEV).float()
    move[:, ::128] = 0
    there = (w + move).clamp(-8, 8)
    change = ((fused.block_linear(x, there) - y.detach()) * g).double().sum()
    assert torch.equal(change, ((there - w).double() * dw.double()).sum())
    move = torch.randint(-1, 2, x.shape, device=DEV).float()
    move[:, ::128] = 0
    there = (x + move).clamp(-8, 8)
    change = ((fused.block_linear(there, w) - y.detach()) * g).double().sum()
    assert torch.equal(change, ((there - x).double() * dx.double()).sum())


def test_host_and_device_agree():
    x, w, b = rand(50, 300), rand(70, 300, seed=1), rand(70, seed=2)
    for rows in (1, 128):
        for d, h in zip(fused.block_quantize(x, rows, True), fused.block_quantize(x.cpu(), rows, True)):
            assert torch.equal(d.cpu().float(), h.float())
    assert torch.allclose(fused.block_linear(x, w, b).cpu(), fused.block_linear(x.cpu(), w.cpu(), b.cpu()), rtol=1e-5, atol=1e-4)


# ------------------------------------------------------------------ what the tests above leave out
@pytest.mark.parametrize("m", [5, 40, 100, 300])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("far", [100, 119])
def test_product_of_far_scales_whose_product_is_near(m, block_rows, far):
    """Scales far up and far down: their product is a number, and so are the sums times it, wherever
    the sums times one of them are not."""
    a, _ = operand(m, 384, 1, 1)
    b, _ = operand(2000, 384, block_rows, 2)
    g = torch.Generator(device=DEV).manual_seed(9)
    near_a = 1 + torch.rand(m, 3, device=DEV, generator=g)
    near_b = 1 + torch.rand(-(-2000 // block_rows), 3, device=DEV, generator=g)
    for up in (2.0**far, 2.0**-far):
        sa, sb = near_a * up, near_b / up
        out = fused.block_mm(a, sa, b, sb, out_dtype=F32)
        ref.check_product(out, ref.values(a, sa), ref.values(b, sb), None, f"{m} rows, {up}")


@pytest.mark.parametrize("rows,width", [(4, 1001), (300, 1001), (8, 4096), (2000, 4096)])
def test_products_behind_and_beside_dropout_backwards_share_tensor_memory(rows, width):
    """The dropout's backward holds its columns' sums in tensor memory, on shifted vectors or whole ones,
    and with no weight no reduction stands between it and what follows it on its stream: a product,
    directly or behind a quantisation. Products of few rows run on another stream meanwhile."""
    x, dy = rand(rows, width, dtype=BF16, seed=1), rand(rows, width, dtype=BF16, seed=2)
    _, h, rstd = fused.dropout_add_rmsnorm_fwd(x, None, p=0.1, rng=(1, 2), store_rstd=True)
    a, sa = operand(2000, 256, 1, 1)
    b, sb = operand(3000, 256, 128, 2)
    (a2, sa2), (b2, sb2) = fused.block_quantize(rand(2000, 256, seed=3)), fused.block_quantize(rand(3000, 256, seed=4), 128)

    def chain():
        return (fused.dropout_add_rmsnorm_bwd(h, None, dy, rstd, p=0.1, rng=(1, 2))[0], fused.block_mm(a, sa, b, sb),
                fused.dropout_add_rmsnorm_bwd(h, None, dy, rstd, p=0.1, rng=(1, 2))[0], *fused.block_quantize(x),
                fused.block_mm(a2, sa2, b2, sb2, power_of_two=True), fused.block_mm(a[:8], sa[:8], b, sb))

    bits = lambda ts: [t.view(torch.uint8).clone() for t in ts]  # noqa: E731
    want = bits(chain())
    few = fused.block_mm(a[:40], sa[:40], b, sb)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            got = chain()
        with torch.cuda.stream(streams[1]):
            beside = [fused.block_mm(a[:40], sa[:40], b, sb) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(i, j) for i, j in zip(bits(got), want)) and all(torch.equal(t, few) for t in beside)


@pytest.mark.parametrize("k", [16384, 131072])
@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("out_dtype", [BF16, F16])
def test_powers_of_two_of_long_sums(k, positive, out_dtype):
    """All of k is added in the tensor cores, 32 products at a time: what every addition may lose
    adds up where no value is negative."""
    m, n = 256, 4864
    a, b = operand(m, k, 1, 1)[0], operand(n, k, 128, 2)[0]
    if positive:
        a, b = (t.view(torch.uint8).bitwise_and(127).view(E4M3) for t in (a, b))
    g = torch.Generator(device=DEV).manual_seed(5)
    sa = torch.exp2(torch.randint(-12, -9, (m, k // 128), device=DEV, generator=g).float())
    sb = torch.exp2(torch.randint(-12, -9, (n // 128, k // 128), device=DEV, generator=g).float())
    out = fused.block_mm(a, sa, b, sb, out_dtype=out_dtype, power_of_two=True)
    assert _lib.last_plan().startswith("block_mm_scaled")
    ref.check_product(out, ref.values(a, sa), ref.values(b, sb), None, f"k = {k}", True)


def test_linear_without_gradients_quantises_nothing_for_them(monkeypatch):
    """What the host's test of that name says, of the kernels' calls."""
    from rmsnorm import _block

    wanted, enqueue = [], _block._enqueue_quantize
    monkeypatch.setattr(_block, "_enqueue_quantize", lambda *a: wanted.append(a[6] != 0) or enqueue(*a))
    x, w = rand(30, 130).requires_grad_(True), rand(7, 130, seed=1).requires_grad_(True)
    y = fused.block_linear(x, w)
    with torch.no_grad():
        assert torch.equal(fused.block_linear(x, w), y)
    assert torch.equal(fused.block_linear(x.detach(), w), y) and torch.equal(fused.block_linear(x, w.detach()), y)
    assert wanted == [True, True, False, False, True, False, False, True]


@pytest.mark.parametrize("case", ["quantize", "many rows", "powers of two", "few rows"])
def test_offsets_beyond_32_bits(case):
    """More than 2^31 elements; the ends are what they are by themselves."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB")
    same = lambda x, y: torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))  # noqa: E731
    if case == "quantize":
        rows, cols, last = 128 * 8192 + 77, 2056, 128 * 8190
        x = torch.empty(rows, cols, dtype=BF16, device=DEV).normal_()
        q, s, q_t, s_t = fused.block_quantize(x, transposed=True)
        e, es, e_t, es_t = fused.block_quantize(x[last:], transposed=True)
        assert same(q[last:], e) and torch.equal(s[last:], es) and same(q_t[:, last:], e_t) and torch.equal(s_t[:, last // 128:], es_t)
        ref.check_quantized(q[last:], s[last:], x[last:], 1)
        q, s = fused.block_quantize(x, 128)
        e, es = fused.block_quantize(x[last:], 128)
        assert same(q[last:], e) and torch.equal(s[last // 128:], es)
        return
    few = case == "few rows"
    m, n, k = (100, (1 << 25) + 40, 16) if few else (70000, 33000, 64)
    a, b = operand(m, k, 1, 1)[0], operand(n, k, 1, 2)[0]
    sa, sb = torch.ones(m, 1, device=DEV) / 512, torch.ones(-(-n // 128), 1, device=DEV) / 512
    out = fused.block_mm(a, sa, b, sb, power_of_two=case == "powers of two")
    if few:
        last = 128 * ((n - 5000) // 128)
        end, got = fused.block_mm(a, sa, b[last:], sb[last // 128:]), out[:, last:]
        factors = (a, sa), (b[last:], sb[last // 128:])
    else:
        last = 256 * 272
        end, got = fused.block_mm(a[last:], sa[last:], b, sb, power_of_two=case == "powers of two"), out[last:]
        factors = (a[last:], sa[last:]), (b, sb)
    assert same(got, end)
    ref.check_product(end, ref.values(*factors[0]), ref.values(*factors[1]), None, case, True)
