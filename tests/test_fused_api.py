# SPDX-License-Identifier: MIT
"""The fused operators without a GPU: refusals, host-tensor results against 64 bits, gradients
against differences, the generator against published vectors, the C ABI's layouts and checks."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

import fused_ref as ref
from rmsnorm import _host_fused, _lib, fused

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "rmsnorm_b200.h"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------ generator
@pytest.mark.parametrize("counter,key,words", [
    # the known-answer vectors that Salmon, Moraes, Dror and Shaw publish with Philox4x32-10
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(counter, key, words):
    if counter[0] == 0:
        got = _host_fused.philox_words(1, 4, key[0] | key[1] << 32, counter[2] | counter[3] << 32, counter[1], "cpu")
        assert got.tolist() == [list(words)]
    # any counter word: a tensor that reaches that quad would be too wide, so run the rounds
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 ^ c[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    assert tuple(c) == words


def test_philox_words_match_the_rounds_in_exact_integers():
    seed, offset, row0 = 0xFEDCBA9876543210, 0x89ABCDEF01234567, 0xFFFFFFF0
    got = _host_fused.philox_words(3, 11, seed, offset, row0, "cpu")
    for i in range(3):
        for j in range(11):
            c = [j // 4, row0 + i, offset & 0xFFFFFFFF, offset >> 32]
            k = [seed & 0xFFFFFFFF, seed >> 32]
            for _ in range(10):
                a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
                c = [b >> 32 ^ c[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ c[3] ^ k[1], a & 0xFFFFFFFF]
                k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
            assert got[i, j] == c[j % 4]


def test_mask_properties():
    m = fused.dropout_mask((256, 512), 0.25, (1, 2))
    # 131072 draws with probability 3/4: six standard deviations are 0.0072
    assert abs(m.double().mean().item() - 0.75) < 0.0072
    assert not torch.equal(m, fused.dropout_mask((256, 512), 0.25, (1, 3)))
    assert not torch.equal(m, fused.dropout_mask((256, 512), 0.25, (2, 2)))
    assert torch.equal(m[100:140], fused.dropout_mask((40, 512), 0.25, (1, 2), row_offset=100))
    assert torch.equal(m, fused.dropout_mask((256, 512), 0.25, (1, 0), rng_step=torch.tensor([2])))
    assert torch.equal(m, fused.dropout_mask((4, 64, 512), 0.25, (1, 2)).reshape(256, 512))
    assert fused.dropout_mask((64, 64), 0.0, (5, 6)).all()


# ------------------------------------------------------------------ host results
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("quant_dtype", [E4M3, torch.int8])
@pytest.mark.parametrize("n,group", [(1, None), (100, None), (100, 32), (257, 256), (256, 64)])
def test_quant_on_host(dtype, quant_dtype, n, group):
    torch.manual_seed(n)
    x, r = torch.randn(2, 3, n).to(dtype), torch.randn(2, 3, n).to(dtype)
    w, b = 1 + 0.1 * torch.randn(n), torch.randn(n)
    for args in ((w, None, None), (None, b, r), (w, b, r)):
        q, s, ro = fused.rmsnorm_quant_fwd(x, args[0], args[1], args[2], quant_dtype, group)
        h, _, y, size = ref.normalise(x, *args)
        ref.check_quant(q, s, y, size, quant_dtype, group)
        assert q.dtype == quant_dtype and q.shape == x.shape
        if args[2] is None:
            assert ro is x
        else:
            ref.check(ro, h, h.abs(), "residual_out")
    q2, s2, _ = fused.rmsnorm_quant_fwd(x, w, b, r, quant_dtype, group, scales_column_major=True)
    assert torch.equal(s2, s) and torch.equal(q2.float(), q.float())
    if group and n > group:
        assert s2.stride() == (3, 1, 6)


def test_quant_of_empty_zero_and_special_rows_on_host():
    q, s, _ = fused.rmsnorm_quant_fwd(torch.zeros(2, 64))
    assert (q.float() == 0).all() and (s == 2.0**-126).all()
    x = torch.randn(4, 64)
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    q, s, _ = fused.rmsnorm_quant_fwd(x, quant_dtype=torch.int8)
    assert s[1].isnan() and s[2].isnan() and s[0].isfinite() and s[3].isfinite()
    q, s, _ = fused.rmsnorm_quant_fwd(torch.zeros(0, 64), group_size=32)
    assert q.shape == (0, 64) and s.shape == (0, 2)


def _drop_inputs(shape, dtype=F32, seed=0):
    torch.manual_seed(seed)
    n = shape[-1]
    return (torch.randn(shape).to(dtype), 1 + 0.1 * torch.randn(n), torch.randn(n), torch.randn(shape).to(dtype))


@pytest.mark.parametrize("dtype,rdtype", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("shape", [(5, 33), (2, 3, 64), (1, 1)])
def test_dropout_on_host(dtype, rdtype, shape):
    x, w, b, r = _drop_inputs(shape, dtype)
    keep = fused.dropout_mask(shape, 0.3, (11, 12))
    out, ro, rstd = fused.dropout_add_rmsnorm_fwd(x, w, b, r, 0.3, (11, 12), residual_dtype=rdtype, store_rstd=True)
    h, r64, y, size = ref.normalise(x, w, b, r, keep=keep, p=0.3)
    ref.check(out, y, size, "out")
    ref.check(ro, h, h.abs() + r.double().abs(), "residual_out")
    ref.check(rstd, r64.squeeze(-1), 0.0, "rstd")
    dout, dro = torch.randn(shape).to(dtype), torch.randn(shape).to(rdtype)
    dx, dw, db, dres = fused.dropout_add_rmsnorm_bwd(ro, w, dout, rstd, dro, 0.3, (11, 12), True, True, b)
    e = ref.backward(ro, w, dout, rstd, dro, keep, 0.3)
    ref.check(dx, e["dx"], e["size"] / 0.7, "dx")
    ref.check(dres, e["dh"], e["size"], "dresidual")
    ref.check(dw, e["dw"], e["dw_size"], "dweight")
    ref.check(db, e["db"], e["db_size"], "dbias")


@pytest.mark.parametrize("prenorm", [False, True])
def test_dropout_gradients_against_differences(prenorm):
    """Central differences of the operator in 64 bits: the mask is fixed by rng, so the
    operator is smooth. Step 1e-6: truncation and rounding are both below 1e-8."""
    shape = (3, 10)
    x, w, b, r = _drop_inputs(shape)
    a, c = torch.randn(shape).double(), torch.randn(shape).double()
    keep = fused.dropout_mask(shape, 0.4, (3, 4))

    def loss(x, w, b, r):
        h, _, y, _ = ref.normalise(x, w, b, r, keep=keep, p=0.4)
        return (a * y).sum() + ((c * h).sum() if prenorm else 0)

    ts = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    got = fused.dropout_add_rmsnorm(ts[0], ts[1], ts[2], ts[3], 0.4, (3, 4), prenorm=prenorm)
    out, ro = got if prenorm else (got, None)
    ((a.float() * out).sum() + ((c.float() * ro).sum() if prenorm else 0)).backward()
    base = [t.double() for t in (x, w, b, r)]
    for i, t in enumerate(ts):
        want = torch.zeros_like(base[i])
        for j in range(want.numel()):
            d = torch.zeros_like(want)
            d.view(-1)[j] = 1e-6
            up = loss(*[v + d if m == i else v for m, v in enumerate(base)])
            down = loss(*[v - d if m == i else v for m, v in enumerate(base)])
            want.view(-1)[j] = (up - down) / 2e-6
        assert (t.grad.double() - want).abs().max() < 1e-4 * want.abs().max()


def test_dropout_without_residual_and_step():
    x, w, b, _ = _drop_inputs((4, 16))
    out, ro, rstd = fused.dropout_add_rmsnorm_fwd(x, w, p=0.5, rng=(1, 5), rng_step=torch.tensor(2))
    assert rstd is None and ro.dtype == x.dtype
    assert torch.equal(ro == 0, ~fused.dropout_mask((4, 16), 0.5, (1, 7)))
    x = x.clone().requires_grad_(True)
    step = torch.tensor([3])
    y = fused.dropout_add_rmsnorm(x, w, p=0.5, rng=(1, 5), rng_step=step)
    step += 1  # the backward keeps the mask of its forward
    y.sum().backward()
    assert torch.equal(x.grad == 0, ~fused.dropout_mask((4, 16), 0.5, (1, 8)))


ROPE = [(3, 2, 1, 8, 8, (4,), False), (5, 4, 2, 16, 8, (1, 1, 2), False), (2, 3, 3, 10, 6, (1, 2), True),
        (1, 1, 1, 7, 2, (1,), False), (4, 2, 1, 12, 12, (2, 2, 2), True), (2, 2, 1, 6, 0, (), False)]


def _rope_inputs(t, hq, hk, d, rd, sections, dtype=F32, seed=0):
    torch.manual_seed(seed)
    naxes = max(1, len(sections))
    table = fused.rope_table(50, rd) if rd else torch.zeros(50, 0)
    return (torch.randn(t, hq, d).to(dtype), torch.randn(t, hk, d).to(dtype), torch.randint(0, 50, (naxes, t)), table,
            1 + 0.1 * torch.randn(d), 1 + 0.1 * torch.randn(hk, d), fused.rope_axes(sections) if sections else ())


@pytest.mark.parametrize("case", ROPE)
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope_on_host(case, norm, dtype):
    t, hq, hk, d, rd, sections, inter = case
    q, k, pos, table, qw, kw, axes = _rope_inputs(t, hq, hk, d, rd, sections, dtype)
    cos, sin = ref.cos_sin(pos, table, axes)
    qo, ko = fused.qk_norm_rope_fwd(q, k, pos, table, qw, kw, axes, inter, norm)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    grads = fused.qk_norm_rope_bwd(q, k, pos, table, dq, dk, qw, kw, axes, inter, norm)
    for x, w, got, dout, gx, gw in ((q, qw, qo, dq, grads[0], grads[2]), (k, kw, ko, dk, grads[1], grads[3])):
        want, size = ref.rope(x, w, cos, sin, inter, norm)
        ref.check(got, want, size, "out")
        dx, size, dw, dw_size = ref.rope_backward(x, w, dout, cos, sin, inter, norm)
        ref.check(gx, dx, size, "dx")
        over = (0, 1) if w.dim() == 1 else (0,)
        ref.check(gw, dw.sum(over), dw_size.sum(over), "dweight")
    a, b = q.clone(), k.clone()
    r = fused.qk_norm_rope_fwd(a, b, pos, table, qw, kw, axes, inter, norm, inplace=True)
    assert r[0] is a and r[1] is b and torch.equal(a, qo) and torch.equal(b, ko)


@pytest.mark.parametrize("norm", [True, False])
def test_rope_gradients_against_differences(norm):
    q, k, pos, table, qw, kw, axes = _rope_inputs(2, 2, 1, 8, 4, (1, 1))
    a, b = torch.randn(q.shape).double(), torch.randn(k.shape).double()
    cos, sin = ref.cos_sin(pos, table, axes)

    def loss(q, k, qw, kw):
        return (a * ref.rope(q, qw, cos, sin, False, norm)[0]).sum() + (b * ref.rope(k, kw, cos, sin, False, norm)[0]).sum()

    ts = [t.clone().requires_grad_(True) for t in (q, k, qw, kw)]
    qo, ko = fused.qk_norm_rope(ts[0], ts[1], pos, table, ts[2], ts[3], axes, norm=norm)
    ((a.float() * qo).sum() + (b.float() * ko).sum()).backward()
    base = [t.double() for t in (q, k, qw, kw)]
    for i, t in enumerate(ts):
        want = torch.zeros_like(base[i])
        for j in range(want.numel()):
            d = torch.zeros_like(want)
            d.view(-1)[j] = 1e-6
            up = loss(*[v + d if m == i else v for m, v in enumerate(base)])
            down = loss(*[v - d if m == i else v for m, v in enumerate(base)])
            want.view(-1)[j] = (up - down) / 2e-6
        assert (t.grad.double() - want).abs().max() < 1e-4 * want.abs().max()


def test_rope_helpers_and_positions_outside_the_table():
    assert fused.rope_axes((1, 2)) == (0, 1, 1)
    assert fused.rope_axes((2, 1, 1), interleaved=True) == (0, 1, 2, 0)
    assert fused.rope_axes((0, 2)) == (1, 1)
    with pytest.raises(ValueError, match="sections"):
        fused.rope_axes(())
    with pytest.raises(ValueError, match="sections"):
        fused.rope_axes((1, -1))
    with pytest.raises(ValueError, match="rope_table"):
        fused.rope_table(4, 3)
    t = fused.rope_table(100, 8)
    assert t[0, :4].tolist() == [1.0] * 4 and t[0, 4:].tolist() == [0.0] * 4
    q = torch.randn(2, 1, 8)
    out, none = fused.qk_norm_rope_fwd(q, None, torch.tensor([3, 100]), t[:, [0, 1, 4, 5]])
    assert none is None and out[0].isfinite().all() and out[1, 0, :4].isnan().all() and out[1, 0, 4:].isfinite().all()


def test_under_torch_compile():
    """The operators break the graph and compute what they compute in eager mode."""
    torch._dynamo.reset()
    x, r, w = torch.randn(4, 64), torch.randn(4, 64), torch.ones(64)
    q, pos, table = torch.randn(4, 2, 16), torch.arange(4), fused.rope_table(8, 16)

    def f(x, q):
        h, res = fused.dropout_add_rmsnorm(x * 2, w, residual=r, p=0.25, rng=(1, 2), prenorm=True)
        a, _ = fused.qk_norm_rope(q + 1, None, pos, table)
        v, s, _ = fused.rmsnorm_quant_fwd(h, w)
        return (h + res) * 3, a - 1, v.float() * s[:, None]

    x1, x2 = (x.clone().requires_grad_(True) for _ in range(2))
    want, got = f(x1, q), torch.compile(f, backend="eager")(x2, q)
    for s, t in zip(want, got):
        assert torch.equal(s, t)
    want[0].sum().backward()
    got[0].sum().backward()
    assert torch.equal(x1.grad, x2.grad)


# ------------------------------------------------------------------ refusals
def test_quant_refusals():
    x = torch.randn(2, 64)
    with pytest.raises(AssertionError, match="Unsupported dtype"):
        fused.rmsnorm_quant_fwd(x.int())
    with pytest.raises(AssertionError, match="quant_dtype"):
        fused.rmsnorm_quant_fwd(x, quant_dtype=torch.uint8)
    with pytest.raises(AssertionError, match="residual_dtype"):
        fused.rmsnorm_quant_fwd(x, residual_dtype=torch.int8)
    with pytest.raises(AssertionError, match="Weight must"):
        fused.rmsnorm_quant_fwd(x, torch.ones(64, dtype=torch.int32))
    for g in (0, 16, 48, 512, -128):
        with pytest.raises(ValueError, match="group_size"):
            fused.rmsnorm_quant_fwd(x, group_size=g)
    with pytest.raises(ValueError, match="weight shape"):
        fused.rmsnorm_quant_fwd(x, torch.ones(63))
    with pytest.raises(ValueError, match="weight shape"):
        fused.rmsnorm_quant_fwd(x, torch.ones(2, 64))
    with pytest.raises(ValueError, match="bias shape"):
        fused.rmsnorm_quant_fwd(x, None, torch.ones(1))
    with pytest.raises(ValueError, match="residual shape"):
        fused.rmsnorm_quant_fwd(x, residual=torch.randn(1, 64))
    with pytest.raises(ValueError, match="nonzero"):
        fused.rmsnorm_quant_fwd(torch.zeros(2, 0))
    with pytest.raises(ValueError, match="at least one dimension"):
        fused.rmsnorm_quant_fwd(torch.tensor(1.0))


def test_dropout_refusals():
    x = torch.randn(2, 64)
    for p in (-0.1, 1.0, float("nan")):
        with pytest.raises(ValueError, match="p must be"):
            fused.dropout_add_rmsnorm(x, p=p)
    for rng in ((-1, 0), (0, 1 << 64)):
        with pytest.raises(ValueError, match="rng must"):
            fused.dropout_add_rmsnorm(x, p=0.1, rng=rng)
    for row in (-1, (1 << 32) - 1):
        with pytest.raises(ValueError, match="row_offset"):
            fused.dropout_add_rmsnorm(x, p=0.1, row_offset=row)
    for step in (torch.tensor([1, 2]), torch.tensor([1.0])):
        with pytest.raises(ValueError, match="rng_step"):
            fused.dropout_add_rmsnorm(x, p=0.1, rng_step=step)
    with pytest.raises(AssertionError, match="out_dtype"):
        fused.dropout_add_rmsnorm(x, out_dtype=torch.int8)
    with pytest.raises(ValueError, match="residual shape"):
        fused.dropout_add_rmsnorm(x, residual=x[:1])
    rstd = torch.ones(2)
    with pytest.raises(ValueError, match="rstd must be float32"):
        fused.dropout_add_rmsnorm_bwd(x, None, x, rstd.double())
    with pytest.raises(ValueError, match="one element per row"):
        fused.dropout_add_rmsnorm_bwd(x, None, x, rstd[:1])
    with pytest.raises(ValueError, match="dout shape"):
        fused.dropout_add_rmsnorm_bwd(x, None, x[:1], rstd)
    with pytest.raises(ValueError, match="dresidual_out shape"):
        fused.dropout_add_rmsnorm_bwd(x, None, x, rstd, x[:1])
    with pytest.raises(AssertionError, match="dx_dtype"):
        fused.dropout_add_rmsnorm_bwd(x, None, x, rstd, dx_dtype=torch.int8)


def test_rope_refuses_more_heads_than_the_kernels_count():
    q, table, pos = torch.zeros(1, 65537, 2), torch.ones(1, 2), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="65536"):
        fused.qk_norm_rope_fwd(q, None, pos, table)
    with pytest.raises(ValueError, match="65536"):
        fused.qk_norm_rope_fwd(q[:, :1], q, pos, table)
    fused.qk_norm_rope_fwd(q[:, 1:], q[:, :1], pos, table)


def test_rope_refusals():
    q, k, pos, table, qw, kw, axes = _rope_inputs(4, 2, 1, 8, 8, (2, 2))
    ok = dict(q=q, k=k, positions=pos, table=table, q_weight=qw, k_weight=kw, axes=axes)
    fused.qk_norm_rope_fwd(**ok)
    for change, error, match in [
        (dict(q=q.int(), k=k.int()), AssertionError, "Unsupported"),
        (dict(k=k.half()), AssertionError, "same dtype"),
        (dict(k=k[:3]), ValueError, "q's shape"),
        (dict(k=k[..., :4]), ValueError, "q's shape"),
        (dict(q=q[:, :0]), ValueError, "at least one head"),
        (dict(table=table.double()), ValueError, "table must"),
        (dict(table=torch.zeros(9, 10)), ValueError, "table must"),
        (dict(table=torch.zeros(9, 3)), ValueError, "table must"),
        (dict(positions=pos.float()), ValueError, "int32 or int64"),
        (dict(positions=pos[:, :3]), ValueError, "positions must"),
        (dict(positions=pos[0]), ValueError, "axes must"),
        (dict(axes=axes[:3]), ValueError, "axes must"),
        (dict(axes=(0, 0, 2, 0)), ValueError, "axes must"),
        (dict(q_weight=qw[:4]), ValueError, "q_weight shape"),
        (dict(k_weight=kw.expand(3, 8)), ValueError, "k_weight shape"),
        (dict(k=None), ValueError, "k_weight needs k"),
        (dict(k_weight=kw.bfloat16()), AssertionError, "same dtype"),
    ]:
        with pytest.raises(error, match=match):
            fused.qk_norm_rope_fwd(**{**ok, **change})
    with pytest.raises(ValueError, match="head_dim"):
        fused.qk_norm_rope_fwd(torch.randn(1, 1, 257), None, torch.zeros(1, dtype=torch.int64), table)
    with pytest.raises(ValueError, match="dk_out"):
        fused.qk_norm_rope_bwd(q, k, pos, table, q, None, qw, kw, axes)
    with pytest.raises(ValueError, match="dq_out"):
        fused.qk_norm_rope_bwd(q, k, pos, table, q[:2], k, qw, kw, axes)


# ------------------------------------------------------------------ C ABI
@pytest.mark.parametrize("cls,cname", [
    (_lib.QuantArgs, "rmsnorm_b200_quant_args"), (_lib.Dropout, "rmsnorm_b200_dropout"),
    (_lib.DropoutFwdArgs, "rmsnorm_b200_dropout_fwd_args"), (_lib.DropoutBwdArgs, "rmsnorm_b200_dropout_bwd_args"),
    (_lib.RopeTensor, "rmsnorm_b200_rope_tensor"), (_lib.RopeArgs, "rmsnorm_b200_rope_args"),
    (_lib.RopeGrads, "rmsnorm_b200_rope_grads")])
def test_struct_layouts(cls, cname, tmp_path):
    fields = [f[0] for f in cls._fields_]
    src = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{HEADER}"', "int main(void) {",
           f'  printf("%zu\\n", sizeof({cname}));', *[f'  printf("%zu\\n", offsetof({cname}, {f}));' for f in fields],
           "  return 0;", "}"]
    (tmp_path / "probe.c").write_text("\n".join(src))
    subprocess.run(["gcc", "-o", str(tmp_path / "probe"), str(tmp_path / "probe.c")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(cls), *[getattr(cls, f).offset for f in fields]]


def test_entry_points_refuse_bad_arguments_without_a_device():
    lib = _lib.load_library()
    bad = 1  # RMSNORM_B200_ERR_INVALID_ARGUMENT

    def quant(**kw):
        a = dict(rows=4, hidden=64, x=16, q=16, scales=16, q_dtype=3)
        return lib.rmsnorm_b200_quant_fwd(ctypes.byref(_lib.QuantArgs(**{**a, **kw})), None)

    assert lib.rmsnorm_b200_quant_fwd(None, None) == bad
    for kw in (dict(rows=-1), dict(hidden=0), dict(x=None), dict(q=None), dict(scales=None), dict(q_dtype=1),
               dict(x_dtype=3), dict(group=16), dict(residual=16, residual_dtype=4), dict(scale_row_stride=-1)):
        assert quant(**kw) == bad, kw
    assert quant(rows=0, x=None, q=None, scales=None) == 0

    def drop(p=0.1, row_offset=0, **kw):
        a = dict(rows=4, hidden=64, x=16, out=16, drop=_lib.Dropout(1, 2, None, row_offset, p))
        return lib.rmsnorm_b200_dropout_rmsnorm_fwd(ctypes.byref(_lib.DropoutFwdArgs(**{**a, **kw})), None)

    assert lib.rmsnorm_b200_dropout_rmsnorm_fwd(None, None) == bad
    for kw in (dict(p=1.0), dict(p=-0.5), dict(p=float("nan")), dict(row_offset=-1), dict(row_offset=(1 << 32) - 3),
               dict(x=None), dict(out=None), dict(out_dtype=3), dict(weight=16, weight_dtype=9)):
        assert drop(**kw) == bad, kw
    assert drop(rows=0) == 0

    def drop_bwd(p=0.1, **kw):
        a = dict(rows=4, hidden=64, h=16, dout=16, rstd=16, dx=16, drop=_lib.Dropout(1, 2, None, 0, p))
        return lib.rmsnorm_b200_dropout_rmsnorm_bwd(ctypes.byref(_lib.DropoutBwdArgs(**{**a, **kw})), None, 0, None)

    assert lib.rmsnorm_b200_dropout_rmsnorm_bwd(None, None, 0, None) == bad
    assert lib.rmsnorm_b200_dropout_rmsnorm_bwd_workspace_size(None, None) == bad
    for kw in (dict(p=2.0), dict(h=None), dict(rstd=None), dict(dx_dtype=7), dict(dweight=16, dweight_dtype=5)):
        assert drop_bwd(**kw) == bad, kw

    tensor = _lib.RopeTensor(16, 64, 8)

    def rope(axis_word=0, **kw):
        words = (ctypes.c_uint64 * 4)(axis_word, 0, 0, 0)
        a = dict(tokens=4, table_rows=9, positions=16, table=16, q=tensor, k=tensor, axis_of_pair=words, q_heads=2,
                 k_heads=1, head_dim=8, rotary_dim=8, axes=1, q_weight_heads=1, k_weight_heads=1)
        return lib.rmsnorm_b200_rope_fwd(ctypes.byref(_lib.RopeArgs(**{**a, **kw})), ctypes.byref(tensor),
                                         ctypes.byref(tensor), None)

    assert lib.rmsnorm_b200_rope_fwd(None, None, None, None) == bad
    for kw in (dict(tokens=-1), dict(q_heads=0), dict(k_heads=-1), dict(head_dim=257), dict(head_dim=0),
               dict(rotary_dim=7), dict(rotary_dim=16), dict(axes=0), dict(axes=5), dict(axis_word=1), dict(dtype=3),
               dict(q=_lib.RopeTensor(None, 0, 0)), dict(q=_lib.RopeTensor(16, -1, 0)), dict(positions=None),
               dict(table=None), dict(q_weight=16, q_weight_heads=3), dict(k_weight=16, weight_dtype=8)):
        assert rope(**kw) == bad, kw
    assert rope(tokens=0) == 0
    grads = _lib.RopeGrads(tensor, tensor, tensor, tensor, 16, None)  # a gradient without its weight
    a = _lib.RopeArgs(tokens=4, table_rows=9, positions=16, table=16, q=tensor, k=tensor, q_heads=2, k_heads=1,
                      head_dim=8, rotary_dim=8, axes=1)
    assert lib.rmsnorm_b200_rope_bwd(ctypes.byref(a), ctypes.byref(grads), None, 0, None) == bad
