# SPDX-License-Identifier: MIT
"""The fused operators' kernels against 64 bits (tests/fused_ref.py has the error bounds)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import fused_ref as ref
from rmsnorm import _lib, fused

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3, I8 = torch.float8_e4m3fn, torch.int8


@pytest.fixture(autouse=True)
def _status_stays_clear():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status(DEV) == (0, 0)


def rand(*shape, dtype=F32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def affine(n, seed=5):
    return 1 + 0.1 * rand(n, seed=seed), rand(n, seed=seed + 1)


def unaligned(t):
    """The same values at an address 2 or 4 bytes past a 16-byte boundary."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    return buf[1:].view(t.shape).copy_(t)


# one row, few, odd counts; widths of one vector, odd ones, whole and ragged slices, several CTAs
WIDTHS = [1, 7, 8, 100, 256, 264, 1001, 2048, 4096, 4100, 5120, 8192, 16384, 16392, 24576, 32768, 65536, 131072, 262144,
          270000]


def rows_for(n):
    return 5 if n > 32768 else 37 if n > 4096 else 301


# ------------------------------------------------------------------ 8-bit output
def quant_case(rows, n, dtype, residual, residual_dtype, weight, bias, quant_dtype, group, change=lambda t: t):
    x = change(rand(rows, n, dtype=dtype, seed=1))
    r = change(rand(rows, n, dtype=residual, seed=2)) if residual else None
    w, b = affine(n)
    w, b = (w if weight else None), (b if bias else None)
    q, s, ro = fused.rmsnorm_quant_fwd(x, w, b, r, quant_dtype, group, residual_dtype)
    h, _, y, size = ref.normalise(x, w, b, r)
    ref.check_quant(q, s, y, size, quant_dtype, group)
    assert q.dtype == quant_dtype and s.dtype == F32
    if r is None and residual_dtype in (None, dtype):
        assert ro is x
    else:
        assert ro.dtype == (residual_dtype or residual)
        ref.check(ro, h, h.abs() + (0 if r is None else r.double().abs()), "residual_out")


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("group", [None, 128])
def test_quant_widths(n, group):
    quant_case(rows_for(n), n, BF16, BF16, None, True, False, E4M3, group)


@pytest.mark.parametrize("rows", [1, 2, 3, 64, 147, 149, 1000])
@pytest.mark.parametrize("n,group", [(4096, None), (1024, 32), (520, 256)])
def test_quant_row_counts(rows, n, group):
    quant_case(rows, n, BF16, BF16, None, True, True, E4M3, group)


@pytest.mark.parametrize("dtype,residual,residual_dtype", [
    (BF16, None, None), (F16, None, None), (F32, None, None), (F16, F16, None), (F32, F32, None), (BF16, F32, None),
    (F16, F32, None), (BF16, BF16, F32), (F16, F16, F32), (F32, BF16, None), (BF16, F16, None), (BF16, None, F32),
    (F32, None, BF16), (F32, F32, F16)])
@pytest.mark.parametrize("quant_dtype", [E4M3, I8])
@pytest.mark.parametrize("n", [1000, 1001])
def test_quant_types(dtype, residual, residual_dtype, quant_dtype, n):
    quant_case(67, n, dtype, residual, residual_dtype, True, False, quant_dtype, None)
    quant_case(67, n, dtype, residual, residual_dtype, False, True, quant_dtype, 64)


@pytest.mark.parametrize("group", [None, 32, 64, 128, 256])
@pytest.mark.parametrize("n", [31, 64, 1016, 4096, 4105, 20000, 40960])
def test_quant_groups(group, n):
    for bias in (False, True):
        quant_case(33, n, F16, F16, None, True, bias, I8, group)


def test_quant_affine_types_and_none():
    x = rand(70, 640, dtype=BF16)
    for wd in (BF16, F16, F32):
        w, b = (t.to(wd) for t in affine(640))
        q, s, _ = fused.rmsnorm_quant_fwd(x, w, b, group_size=128)
        _, _, y, size = ref.normalise(x, w, b, None)
        ref.check_quant(q, s, y, size, E4M3, 128)
    quant_case(70, 640, BF16, BF16, None, False, False, E4M3, None)


@pytest.mark.parametrize("n", [512, 4096])
def test_quant_unaligned_and_strided_inputs(n):
    quant_case(50, n, BF16, BF16, None, True, True, E4M3, 128, unaligned)
    x = rand(20, 3, 2 * n, dtype=BF16)[..., ::2]
    w, _ = affine(n)
    q, s, _ = fused.rmsnorm_quant_fwd(x, unaligned(w), group_size=64)
    _, _, y, size = ref.normalise(x, w, None, None)
    ref.check_quant(q, s, y, size, E4M3, 64)
    q2, s2, _ = fused.rmsnorm_quant_fwd(x, w, group_size=64, scales_column_major=True)
    assert s2.shape == s.shape and s2.stride() == (3, 1, 60)
    assert torch.equal(s2, s) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("n", [256, 1001, 4096, 32768])
@pytest.mark.parametrize("quant_dtype", [E4M3, I8])
@pytest.mark.parametrize("group", [None, 64])
def test_quant_special_values(n, quant_dtype, group):
    """Zero rows, NaN, infinities, tiny and huge values; other rows and groups stay exact."""
    x = rand(12, n, seed=3)
    x[1] = 0
    x[3, n // 2] = float("nan")
    x[5, n - 1] = float("inf")
    x[7] *= 1e-30
    x[8] *= 1e15
    q, s, _ = fused.rmsnorm_quant_fwd(x, quant_dtype=quant_dtype, group_size=group)
    _, _, y, size = ref.normalise(x, None, None, None)
    ok = [0, 1, 2, 4, 6, 7, 8, 9, 10, 11]
    ref.check_quant(q[ok], s[ok], y[ok], size[ok], quant_dtype, group)
    assert (s[1] == 2.0**-126).all() and (q[1].float() == 0).all()
    assert s[3].isnan().all()  # the whole row is NaN
    at = s[5] if group is None else s[5, (n - 1) // group]
    assert at.isnan()  # infinity / infinity
    if group:
        assert (s[5, : (n - 1) // group] == 2.0**-126).all()  # finite / infinity


def test_quant_empty():
    q, s, ro = fused.rmsnorm_quant_fwd(torch.zeros(0, 4096, device=DEV), group_size=128)
    assert q.shape == (0, 4096) and s.shape == (0, 32)


# ------------------------------------------------------------------ dropout
def drop_case(rows, n, dtype, residual, residual_dtype, out_dtype, weight, bias, p=0.3, rng=(0x123456789ABCDEF, 1 << 35),
              row_offset=0, change=lambda t: t, wd=F32):
    x = change(rand(rows, n, dtype=dtype, seed=1))
    r = change(rand(rows, n, dtype=residual, seed=2)) if residual else None
    w, b = (t.to(wd) for t in affine(n))
    w, b = (w if weight else None), (b if bias else None)
    keep = fused.dropout_mask((rows, n), p, rng, DEV, row_offset=row_offset)
    out, ro, rstd = fused.dropout_add_rmsnorm_fwd(
        x, w, b, r, p, rng, out_dtype, residual_dtype, store_rstd=True, row_offset=row_offset)
    h, r64, y, size = ref.normalise(x, w, b, r, keep=keep, p=p)
    ref.check(out, y, size, "out")
    ref.check(ro, h, h.abs() + (0 if r is None else r.double().abs()), "residual_out")
    ref.check(rstd, r64.squeeze(-1), 0.0, "rstd")
    if r is None:
        assert torch.equal(ro == 0, ~keep | (x == 0))
    assert out.dtype == (out_dtype or dtype) and ro.dtype == (residual_dtype or residual or dtype)


@pytest.mark.parametrize("n", WIDTHS)
def test_dropout_fwd_widths(n):
    drop_case(rows_for(n), n, BF16, BF16, None, None, True, True)


@pytest.mark.parametrize("rows", [1, 2, 64, 147, 149, 1000])
@pytest.mark.parametrize("n", [264, 4096])
def test_dropout_fwd_row_counts(rows, n):
    drop_case(rows, n, BF16, BF16, F32, None, True, False)


@pytest.mark.parametrize("dtype,residual,residual_dtype,out_dtype", [
    (BF16, None, None, None), (F16, None, None, F32), (F32, None, None, None), (F16, F16, None, None),
    (F32, F32, None, BF16), (BF16, F32, None, None), (F16, F32, F16, None), (BF16, BF16, F32, F16),
    (F32, BF16, None, None), (F16, BF16, F32, None)])
@pytest.mark.parametrize("n", [1000, 1001])
def test_dropout_fwd_types(dtype, residual, residual_dtype, out_dtype, n):
    drop_case(67, n, dtype, residual, residual_dtype, out_dtype, True, False)
    drop_case(67, n, dtype, residual, residual_dtype, out_dtype, False, True)


@pytest.mark.parametrize("n", [512, 1003])
def test_dropout_fwd_probabilities_rows_and_alignment(n):
    for p in (0.0, 1e-9, 0.5, 0.999):
        drop_case(40, n, F32, F32, None, None, True, True, p=p)
    drop_case(40, n, F16, F16, None, None, True, True, row_offset=(1 << 32) - 40)
    drop_case(40, n, BF16, BF16, None, None, True, True, change=unaligned)
    drop_case(40, n, BF16, BF16, None, None, True, True, wd=BF16, rng=((1 << 64) - 1, (1 << 64) - 1))


def test_dropped_values_do_not_reach_the_row():
    """NaN and infinities that the mask drops leave no trace, forward and backward."""
    n, rng = 4096, (3, 4)
    keep = fused.dropout_mask((9, n), 0.5, rng, DEV)
    x, r = rand(9, n), rand(9, n, seed=1)
    clean = torch.where(keep, x, 0.0)
    dirty = torch.where(keep, x, torch.where(rand(9, n, seed=2) > 0, float("nan"), float("inf")))
    a = fused.dropout_add_rmsnorm_fwd(clean, residual=r, p=0.5, rng=rng, store_rstd=True)
    b = fused.dropout_add_rmsnorm_fwd(dirty, residual=r, p=0.5, rng=rng, store_rstd=True)
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    dro = torch.where(keep, r, float("nan"))
    dx, _, _, dres = fused.dropout_add_rmsnorm_bwd(a[1], None, r, a[2], dro, 0.5, rng, has_residual=True)
    assert (dx[~keep] == 0).all() and dx.isfinite().all() and torch.equal(dres.isnan(), ~keep)


def bwd_case(rows, n, h_dtype, dtype, dro_dtype, weight, bias, has_residual=True, dx_dtype=None, dres_dtype=None, p=0.3,
             rng=(99, 7), row_offset=0, change=lambda t: t, wd=F32):
    h = change(rand(rows, n, dtype=h_dtype, seed=1))
    dout = change(rand(rows, n, dtype=dtype, seed=2))
    dro = change(rand(rows, n, dtype=dro_dtype, seed=3)) if dro_dtype else None
    w, b = (t.to(wd) for t in affine(n))
    w = w if weight else None
    rstd = (h.float().square().mean(-1) + 1e-6).rsqrt()
    keep = fused.dropout_mask((rows, n), p, rng, DEV, row_offset=row_offset)
    run = lambda: fused.dropout_add_rmsnorm_bwd(  # noqa: E731
        h, w, dout, rstd, dro, p, rng, bias, has_residual, b if bias else None, dx_dtype, dres_dtype,
        row_offset=row_offset)
    dx, dw, db, dres = run()
    e = ref.backward(h, w, dout, rstd, dro, keep, p)
    ref.check(dx, e["dx"], e["size"] / (1 - p), "dx")
    assert (dx[~keep] == 0).all()
    if has_residual:
        ref.check(dres, e["dh"], e["size"], "dresidual")
    else:
        assert dres is None
    if weight:
        ref.check(dw, e["dw"], e["dw_size"], "dweight")
    else:
        assert dw is None
    if bias:
        ref.check(db, e["db"], e["db_size"], "dbias")
    else:
        assert db is None
    for s, t in zip((dx, dw, db, dres), run()):  # the same bits every time
        assert s is None or torch.equal(s, t)


@pytest.mark.parametrize("n", WIDTHS)
def test_dropout_bwd_widths(n):
    bwd_case(rows_for(n), n, BF16, BF16, BF16, True, True)


@pytest.mark.parametrize("rows", [1, 2, 64, 147, 149, 1000, 5000])
@pytest.mark.parametrize("n", [264, 4096])
def test_dropout_bwd_row_counts(rows, n):
    bwd_case(rows, n, F32, BF16, F32, True, False)


@pytest.mark.parametrize("h_dtype,dtype,dro_dtype,dx_dtype,dres_dtype", [
    (BF16, BF16, None, None, None), (F16, F16, F16, None, None), (F32, F32, F32, None, None), (F32, F16, F32, None, F16),
    (F32, BF16, None, F32, BF16), (BF16, F32, BF16, BF16, F32), (F16, BF16, F32, F16, F32), (BF16, BF16, F32, None, F32)])
@pytest.mark.parametrize("n", [1000, 1001])
def test_dropout_bwd_types(h_dtype, dtype, dro_dtype, dx_dtype, dres_dtype, n):
    bwd_case(67, n, h_dtype, dtype, dro_dtype, True, True, True, dx_dtype, dres_dtype)
    bwd_case(67, n, h_dtype, dtype, dro_dtype, True, False, False, dx_dtype, dres_dtype)
    bwd_case(67, n, h_dtype, dtype, dro_dtype, False, True, True, dx_dtype, dres_dtype)
    bwd_case(67, n, h_dtype, dtype, dro_dtype, False, False, False, dx_dtype, dres_dtype)


@pytest.mark.parametrize("n", [512, 1003, 16384])
def test_dropout_bwd_alignment_rows_and_weights(n):
    bwd_case(40, n, BF16, BF16, BF16, True, True, change=unaligned)
    bwd_case(40, n, F32, BF16, F32, True, True, row_offset=(1 << 32) - 40, wd=BF16)


def test_dropout_rows_of_a_whole_tensor():
    """Two ranks' rows draw the mask of the whole tensor."""
    x, r = rand(100, 1024), rand(100, 1024, seed=1)
    whole = fused.dropout_add_rmsnorm_fwd(x, residual=r, p=0.2, rng=(5, 6))[1]
    parts = [fused.dropout_add_rmsnorm_fwd(x[a:z], residual=r[a:z], p=0.2, rng=(5, 6), row_offset=a)[1]
             for a, z in ((0, 37), (37, 100))]
    assert torch.equal(torch.cat(parts), whole)


@pytest.mark.parametrize("n", [512, 1003])
def test_dropout_bwd_of_zero_rows_with_a_tiny_eps(n):
    """rstd = eps^-1/2 = 1e16 and its cube does not fit fp32; dx = dout w rstd does."""
    h, dout = torch.zeros(40, n, device=DEV), rand(40, n, seed=1)
    w, _ = affine(n)
    rstd = torch.full((40,), 1e16, device=DEV)
    dx, dw, _, _ = fused.dropout_add_rmsnorm_bwd(h, w, dout, rstd)
    ref.check(dx, dout.double() * w.double() * 1e16, 0.0, "dx")
    assert (dw == 0).all()


def test_dropout_autograd_and_empty():
    x, r = (rand(6, 4, 128, dtype=BF16, seed=s).requires_grad_(True) for s in (1, 2))
    w, b = (t.requires_grad_(True) for t in affine(128))
    out, ro = fused.dropout_add_rmsnorm(x, w, b, r, 0.25, (1, 2), residual_dtype=F32, prenorm=True)
    g, gr = rand(6, 4, 128, dtype=BF16, seed=3), rand(6, 4, 128, seed=4)
    torch.autograd.backward((out, ro), (g, gr))
    keep = fused.dropout_mask((6, 4, 128), 0.25, (1, 2), DEV)
    rstd = (ro.double().square().mean(-1) + 1e-6).rsqrt().float()
    e = ref.backward(ro.detach(), w.detach(), g, rstd, gr, keep, 0.25)
    ref.check(x.grad, e["dx"], e["size"] / 0.75, "dx")
    ref.check(r.grad, e["dh"], e["size"], "dresidual")
    ref.check(w.grad, e["dw"], e["dw_size"], "dweight")
    ref.check(b.grad, e["db"], e["db_size"], "dbias")
    h = torch.zeros(0, 64, device=DEV)
    dx, dw, db, _ = fused.dropout_add_rmsnorm_bwd(h, torch.ones(64, device=DEV), h, torch.zeros(0, device=DEV),
                                                  has_bias=True)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_dropout_step_in_a_graph():
    """Replays of one captured call draw the masks of the step they run with; on a side stream."""
    x, r = rand(64, 1024), rand(64, 1024, seed=1)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    fused.dropout_add_rmsnorm_fwd(x, p=0.5, rng=(7, 100), rng_step=step)  # kernels are loaded before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, ro, _ = fused.dropout_add_rmsnorm_fwd(x, p=0.5, rng=(7, 100), rng_step=step)
    for i in (0, 5, -100, (1 << 63) - 1):
        step.fill_(i)
        graph.replay()
        assert torch.equal(ro == 0, ~fused.dropout_mask((64, 1024), 0.5, (7, (100 + i) % (1 << 64)), DEV)), i
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = fused.dropout_add_rmsnorm_fwd(x, residual=r, p=0.5, rng=(7, 1))
    torch.cuda.current_stream().wait_stream(side)
    for s, t in zip(other[:2], fused.dropout_add_rmsnorm_fwd(x, residual=r, p=0.5, rng=(7, 1))[:2]):
        assert torch.equal(s, t)


# ------------------------------------------------------------------ rotary positions
def rope_case(tokens, hq, hk, d, rd, sections, interleaved=False, norm=True, dtype=BF16, weights="shared", packed=True,
              inter_axes=False, pos_dtype=torch.int64, lead=None, wd=F32):
    width = hq + 2 * hk
    qkv = rand(tokens, width * d + (0 if packed else 1), dtype=dtype, seed=1)
    q = qkv[:, : hq * d].view(tokens, hq, d)
    k = qkv[:, hq * d: (hq + hk) * d].view(tokens, hk, d) if hk else None
    naxes = max(1, len(sections))
    table = fused.rope_table(5000, rd, device=DEV) if rd else torch.zeros(5000, 0, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    pos = torch.randint(0, 5000, (naxes, tokens), device=DEV, generator=g).to(pos_dtype)
    axes = fused.rope_axes(sections, inter_axes) if sections else ()
    shape = {"shared": lambda h: (d,), "heads": lambda h: (h, d)}.get(weights, lambda h: None)
    qw = (1 + 0.1 * rand(*shape(hq), seed=4)).to(wd) if shape(hq) else None
    kw = (1 + 0.1 * rand(*shape(hk), seed=5)).to(wd) if hk and shape(hk) else None
    if lead:
        q = q.unflatten(0, lead)
        k = k if k is None else k.unflatten(0, lead)
        pos = pos.unflatten(1, lead)
    cos, sin = ref.cos_sin(pos, table, axes)
    qo, ko = fused.qk_norm_rope_fwd(q, k, pos, table, qw, kw, axes, interleaved, norm)
    dqo = rand(*q.shape, dtype=dtype, seed=6)
    dko = rand(*k.shape, dtype=dtype, seed=7) if hk else None
    run = lambda: fused.qk_norm_rope_bwd(q, k, pos, table, dqo, dko, qw, kw, axes, interleaved, norm)  # noqa: E731
    dq, dk, dqw, dkw = run()
    for name, x, w, out, dout, dx, dw in (("q", q, qw, qo, dqo, dq, dqw), ("k", k, kw, ko, dko, dk, dkw)):
        if x is None:
            assert out is None and dx is None and dw is None
            continue
        want, size = ref.rope(x, w, cos, sin, interleaved, norm)
        ref.check(out, want, size, name)
        assert out.is_contiguous() and out.dtype == dtype
        want, size, gw, gw_size = ref.rope_backward(x, w, dout, cos, sin, interleaved, norm)
        ref.check(dx, want, size, "d" + name)
        if w is None:
            assert dw is None
        else:
            over = tuple(range(gw.dim() - w.dim()))
            ref.check(dw, gw.sum(over), gw_size.sum(over), f"d{name}_weight")
    for s, t in zip((dq, dk, dqw, dkw), run()):  # the same bits every time
        assert s is None or torch.equal(s, t)
    before = qkv.clone()
    iq, ik = fused.qk_norm_rope_fwd(q, k, pos, table, qw, kw, axes, interleaved, norm, inplace=True)
    assert iq is q and ik is k and torch.equal(iq, qo) and (k is None or torch.equal(ik, ko))
    assert torch.equal(qkv[:, (hq + hk) * d:], before[:, (hq + hk) * d:])  # v stays


@pytest.mark.parametrize("tokens", [1, 2, 7, 64, 999, 5001])
def test_rope_tokens(tokens):
    rope_case(tokens, 32, 8, 128, 128, (16, 24, 24))


@pytest.mark.parametrize("d,rd", [(1, 0), (2, 2), (7, 4), (8, 8), (10, 6), (16, 8), (24, 24), (64, 64), (72, 64), (80, 80),
                                  (80, 40), (96, 48), (100, 100), (128, 64), (160, 32), (192, 192), (256, 256), (256, 64),
                                  (248, 240), (250, 250)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_head_sizes(d, rd, interleaved):
    rope_case(133, 5, 2, d, rd, (rd // 2,) if rd else (), interleaved)
    rope_case(37, 3, 1, d, rd, (rd // 2,) if rd else (), interleaved, dtype=F32)


@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 1), (7, 1), (8, 8), (12, 4), (64, 8), (5, 0), (128, 1)])
@pytest.mark.parametrize("weights", ["shared", "heads", None])
def test_rope_heads_and_weights(hq, hk, weights):
    rope_case(130, hq, hk, 64, 64, (32,), dtype=F16, weights=weights)


@pytest.mark.parametrize("sections", [(64,), (32, 32), (16, 24, 24), (21, 21, 22), (1, 2, 3, 58), (0, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inter_axes", [False, True])
def test_rope_axes(sections, interleaved, inter_axes):
    rope_case(100, 4, 2, 128, 128, sections, interleaved, inter_axes=inter_axes)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("norm", [True, False])
def test_rope_types_norm_positions_and_layouts(dtype, norm):
    for weights in ("shared", "heads", None):
        rope_case(65, 6, 2, 128, 64, (10, 11, 11), norm=norm, dtype=dtype, weights=weights, pos_dtype=torch.int32)
    rope_case(65, 6, 2, 128, 128, (64,), norm=norm, dtype=dtype, wd=BF16, packed=False)  # odd token stride
    rope_case(66, 6, 2, 128, 128, (16, 24, 24), norm=norm, dtype=dtype, lead=(11, 6))


def test_rope_transposed_heads():
    """[heads, tokens, head_dim] seen as [tokens, heads, head_dim]."""
    q = rand(4, 50, 64, dtype=BF16).transpose(0, 1)
    table = fused.rope_table(64, 64, device=DEV)
    pos = torch.arange(50, device=DEV)
    out, _ = fused.qk_norm_rope_fwd(q, None, pos, table)
    cos, sin = ref.cos_sin(pos[None], table, (0,) * 32)
    want, size = ref.rope(q, None, cos, sin, False, True)
    ref.check(out, want, size, "q")
    fused.qk_norm_rope_fwd(q, None, pos, table, inplace=True)
    assert torch.equal(q, out)
    q4 = rand(2, 4, 50, 64, dtype=BF16).transpose(1, 2)
    with pytest.raises(ValueError, match="inplace"):
        fused.qk_norm_rope_fwd(q4, None, pos.expand(2, 50), table, inplace=True)
    out, _ = fused.qk_norm_rope_fwd(q4, None, pos.expand(2, 50), table)
    cos, sin = ref.cos_sin(pos.expand(1, 2, 50), table, (0,) * 32)
    want, size = ref.rope(q4, None, cos, sin, False, True)
    ref.check(out, want, size, "q")


@pytest.mark.parametrize("d", [64, 10])
def test_rope_position_outside_the_table(d):
    """The token's turned columns are NaN, the others are right, and the status word tells."""
    q = rand(6, 2, d)
    rd = d // 4 * 2
    table = fused.rope_table(100, rd, device=DEV)
    pos = torch.tensor([0, 99, 100, -1, 1 << 40, 5], device=DEV)
    out, _ = fused.qk_norm_rope_fwd(q, None, pos, table)
    torch.cuda.synchronize()
    assert _lib.device_status(DEV, clear=True) == (1, 10)
    for t in (2, 3, 4):
        assert out[t, :, :rd].isnan().all() and out[t, :, rd:].isfinite().all()
    assert out[[0, 1, 5]].isfinite().all()
    dq, _, _, _ = fused.qk_norm_rope_bwd(q, None, pos, table, rand(6, 2, d, seed=1), None)
    torch.cuda.synchronize()
    assert _lib.device_status(DEV, clear=True) == (1, 10)
    assert dq[[0, 1, 5]].isfinite().all() and dq[[2, 3, 4]].isnan().any(-1).all()


def test_rope_special_rows_autograd_and_empty():
    q = rand(8, 2, 64)
    q[1] = 0
    q[2, 0, 3] = float("nan")
    table = fused.rope_table(100, 64, device=DEV)
    pos = torch.arange(8, device=DEV)
    out, _ = fused.qk_norm_rope_fwd(q, None, pos, table)
    assert (out[1] == 0).all() and out[2, 0].isnan().all() and out[2, 1].isfinite().all() and out[3:].isfinite().all()
    x, y = rand(9, 3, 64, dtype=BF16).requires_grad_(True), rand(9, 1, 64, dtype=BF16, seed=1).requires_grad_(True)
    w = (1 + 0.1 * rand(64, seed=2)).requires_grad_(True)
    a, b = fused.qk_norm_rope(x, y, pos.new_tensor(range(9)), table, w, w)
    g, h = rand(9, 3, 64, dtype=BF16, seed=3), rand(9, 1, 64, dtype=BF16, seed=4)
    torch.autograd.backward((a, b), (g, h))
    cos, sin = ref.cos_sin(torch.arange(9, device=DEV)[None], table, (0,) * 32)
    d1 = ref.rope_backward(x.detach(), w.detach(), g, cos, sin, False, True)
    d2 = ref.rope_backward(y.detach(), w.detach(), h, cos, sin, False, True)
    ref.check(x.grad, d1[0], d1[1], "dq")
    ref.check(y.grad, d2[0], d2[1], "dk")
    ref.check(w.grad, d1[2].sum((0, 1)) + d2[2].sum((0, 1)), d1[3].sum((0, 1)) + d2[3].sum((0, 1)), "dweight")
    e = torch.zeros(0, 2, 64, device=DEV)
    out, none = fused.qk_norm_rope_fwd(e, None, pos[:0], table)
    assert out.shape == e.shape
    _, _, dw, _ = fused.qk_norm_rope_bwd(e, None, pos[:0], table, e, None, torch.ones(64, device=DEV))
    assert (dw == 0).all()


# ------------------------------------------------------------------ widths that 8 does not divide
# every remainder modulo 8, fewer rows than remainders, rows that end and begin inside a vector,
# one and several vector steps, groups of one and more warps, a cluster
ODD_WIDTHS = [2, 3, 5, 9, 250, 252, 1002, 1003, 1006, 1007, 2050, 4099, 5124, 8191, 12289, 16387, 33001]


@pytest.mark.parametrize("n", ODD_WIDTHS)
@pytest.mark.parametrize("rows", [1, 7, 301])
def test_odd_widths(n, rows):
    quant_case(rows, n, BF16, BF16, None, True, True, E4M3, None)
    quant_case(rows, n, F16, F16, F32, True, False, I8, 32)
    quant_case(rows, n, F32, None, None, True, True, E4M3, 256)
    drop_case(rows, n, BF16, BF16, None, None, True, True)
    drop_case(rows, n, F32, F32, None, None, True, False, row_offset=5)
    bwd_case(rows, n, BF16, BF16, BF16, True, True)
    bwd_case(rows, n, F32, BF16, F32, True, True)


@pytest.mark.parametrize("n", [9, 1003, 4100])
def test_odd_widths_keep_rows_apart(n):
    """A row's NaN and infinities stay in it, although it shares vectors with its neighbours."""
    x, dout, w = rand(61, n, dtype=BF16), rand(61, n, dtype=BF16, seed=1), rand(n, seed=2)
    bad = torch.arange(61, device=DEV) % 3 == 1
    dirty = torch.where(bad[:, None], torch.where(rand(61, n, seed=3) > 0, float("nan"), float("inf")).to(BF16), x)
    for group in (None, 32):
        a, b = (fused.rmsnorm_quant_fwd(t, w, group_size=group) for t in (x, dirty))
        assert torch.equal(a[0].view(torch.uint8)[~bad], b[0].view(torch.uint8)[~bad])
        assert torch.equal(a[1][~bad], b[1][~bad]) and not b[1][bad].isfinite().all()
    rng = (5, 6)
    a, b = (fused.dropout_add_rmsnorm_fwd(t, w, residual=dout, p=0.2, rng=rng, store_rstd=True) for t in (x, dirty))
    for s, t in zip(a, b):
        assert torch.equal(s[~bad], t[~bad])
    rstd = a[2]
    a, b = (fused.dropout_add_rmsnorm_bwd(t, w, dout, rstd, None, 0.2, rng, False, True) for t in (x, dirty))
    assert torch.equal(a[0][~bad], b[0][~bad]) and torch.equal(a[3][~bad], b[3][~bad])


@pytest.mark.parametrize("n", [520, 2368, 4160, 5120, 9216, 10240])
def test_widths_between_powers_of_two(n):
    """Row groups of every number of warps."""
    quant_case(601, n, BF16, BF16, None, True, True, E4M3, 64)
    drop_case(601, n, F16, F16, None, None, True, True)
    bwd_case(601, n, F16, F16, F16, True, True)
    bwd_case(601, n, F32, F32, F32, True, True)
    bwd_case(601, n, F32, BF16, None, True, False)


# ------------------------------------------------------------------ refusals that need a device
def test_refusals_on_device():
    x = rand(2, 64)
    with pytest.raises(ValueError, match="same device"):
        fused.rmsnorm_quant_fwd(x, torch.ones(64))
    with pytest.raises(ValueError, match="same device"):
        fused.dropout_add_rmsnorm_fwd(x, residual=torch.ones(2, 64))
    with pytest.raises(ValueError, match="rng_step"):
        fused.dropout_add_rmsnorm_fwd(x, rng_step=torch.tensor([1]))
    with pytest.raises(ValueError, match="same device"):
        fused.qk_norm_rope_fwd(x[:, None], None, torch.zeros(2, dtype=torch.int64), fused.rope_table(4, 64, device=DEV))
    w = torch.ones(64, device=DEV)
    args = _lib.DropoutBwdArgs(2, 64, x.data_ptr(), x.data_ptr(), x.data_ptr(), w.data_ptr(), None, x.data_ptr(), None,
                               w.data_ptr(), None, _lib.Dropout(0, 0, None, 0, 0.0), 2, 2, 2, 0, 2, 0, 2, 0)
    lib = _lib.load_library()
    n = ctypes.c_size_t(0)
    assert lib.rmsnorm_b200_dropout_rmsnorm_bwd_workspace_size(ctypes.byref(args), ctypes.byref(n)) == 0 and n.value > 0
    assert lib.rmsnorm_b200_dropout_rmsnorm_bwd(ctypes.byref(args), None, 0, None) == 3  # workspace missing
    ws = torch.empty(n.value + 8, dtype=torch.uint8, device=DEV)
    assert lib.rmsnorm_b200_dropout_rmsnorm_bwd(ctypes.byref(args), ws.data_ptr() + 4, n.value, None) == 3  # misaligned
