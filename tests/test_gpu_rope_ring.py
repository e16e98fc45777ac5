# SPDX-License-Identifier: MIT
"""The rotary kernels that stream a warp's heads through a ring, where their data or layout is
out of the ordinary: positions outside the table beside ordinary ones, heads that are not
neighbours, head sizes with lanes to spare, eps 0 with heads that do not fill a warp."""

from __future__ import annotations

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import fused_ref as ref
from rmsnorm import _lib, fused
from test_gpu_fused import BF16, DEV, F16, F32, rand

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


@pytest.fixture(autouse=True)
def _status_stays_clear():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status(DEV) == (0, 0)


def on_the_ring() -> bool:
    """Whether the last call of this thread ran with a ring (its plan has ring slots)."""
    plan = _lib.last_plan()
    return plan.startswith("rope_") and "generic" not in plan and not plan.endswith("S=0")


def same(a, b):
    return all(s is t or torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("axes", [(0,) * 32, (0, 1) * 16])
def test_positions_outside_the_table_leave_the_rest_alone(dtype, axes):
    """Few bad positions in a long prompt: their tokens' turned columns are NaN, everything else
    of that call, and of calls after it with the status not cleared, is bit for bit what it is
    without them. The columns turned are the first 64 of 128."""
    tokens, rd = 6000, 64
    q, k = rand(tokens, 32, 128, dtype=dtype, seed=1), rand(tokens, 8, 128, dtype=dtype, seed=2)
    dq, dk = rand(tokens, 32, 128, dtype=dtype, seed=3), rand(tokens, 8, 128, dtype=dtype, seed=4)
    w, u = 1 + 0.1 * rand(128, seed=5), 1 + 0.1 * rand(128, seed=6)
    table = fused.rope_table(500, rd, device=DEV)
    good = torch.randint(0, 500, (2, tokens), device=DEV, generator=torch.Generator(device=DEV).manual_seed(7))
    at = torch.arange(tokens, device=DEV) % 97 == 5
    bad = torch.where(at, torch.tensor([[-1], [500]], device=DEV), good)

    def forward(pos):
        out = fused.qk_norm_rope_fwd(q, k, pos, table, w, u, axes)
        assert on_the_ring()
        return out

    def backward(pos):
        out = fused.qk_norm_rope_bwd(q, k, pos, table, dq, dk, w, u, axes)
        assert on_the_ring()
        return out

    want, want_grads = forward(good), backward(good)
    got, got_grads = forward(bad), backward(bad)
    again, again_grads = forward(good), backward(good)
    torch.cuda.synchronize()
    assert _lib.device_status(DEV, clear=True) == (1, 10)
    assert same(want, again) and same(want_grads, again_grads)
    for s, t in zip(want, got):
        assert torch.equal(s[~at], t[~at])
        assert t[at][..., :rd].isnan().all() and torch.equal(s[at][..., rd:], t[at][..., rd:])
    for s, t in zip(want_grads[:2], got_grads[:2]):
        assert torch.equal(s[~at], t[~at]) and t[at].isnan().all()  # a head's mean reaches all its columns
    for s, t in zip(want_grads[2:], got_grads[2:]):
        assert t[:rd].isnan().all() and torch.equal(s[rd:], t[rd:])


def test_a_wait_that_ran_out_is_told_before_a_position():
    q, table = rand(4, 2, 64), fused.rope_table(8, 64, device=DEV)
    fused.qk_norm_rope_fwd(q, None, torch.full((4,), 8, device=DEV), table)
    torch.cuda.synchronize()
    assert _lib.device_status(DEV) == (1, 10)
    _lib.selftest_wait_timeout(DEV, 5_000_000)
    assert _lib.device_status(DEV, clear=True) == (_lib.ERR_DEVICE_TIMEOUT, 8)


# ------------------------------------------------------------------ heads that are not neighbours
def apart(tokens, heads, d, gap, dtype, seed):
    """[tokens, heads, d] with a head stride of `gap` head sizes; 0: [heads, tokens, d] transposed."""
    if gap == 0:
        return rand(heads, tokens, d, dtype=dtype, seed=seed).transpose(0, 1)
    return rand(tokens, heads, gap * d, dtype=dtype, seed=seed)[..., :d]


def apart_case(tokens, hq, hk, d, gap, dtype=BF16, weights="shared", interleaved=False, grad_gap=None, ring=True):
    grad_gap = gap if grad_gap is None else grad_gap
    q, k = apart(tokens, hq, d, gap, dtype, 1), apart(tokens, hk, d, gap, dtype, 2)
    dq, dk = apart(tokens, hq, d, grad_gap, dtype, 3), apart(tokens, hk, d, grad_gap, dtype, 4)
    table = fused.rope_table(3000, d, device=DEV)
    pos = torch.randint(0, 3000, (1, tokens), device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    axes = (0,) * (d // 2)
    cos, sin = ref.cos_sin(pos, table, axes)
    shape = (lambda h: (h, d)) if weights == "heads" else (lambda h: (d,))
    qw, kw = 1 + 0.1 * rand(*shape(hq), seed=6), 1 + 0.1 * rand(*shape(hk), seed=7)
    qo, ko = fused.qk_norm_rope_fwd(q, k, pos, table, qw, kw, axes, interleaved)
    assert on_the_ring() == ring
    gx, gy, gw, gu = fused.qk_norm_rope_bwd(q, k, pos, table, dq, dk, qw, kw, axes, interleaved)
    assert on_the_ring()
    for name, x, w, out, dout, dx, dw in (("q", q, qw, qo, dq, gx, gw), ("k", k, kw, ko, dk, gy, gu)):
        want, size = ref.rope(x, w, cos, sin, interleaved, True)
        ref.check(out, want, size, name)
        want, size, each, each_size = ref.rope_backward(x, w, dout, cos, sin, interleaved, True)
        ref.check(dx, want, size, "d" + name)
        over = tuple(range(each.dim() - w.dim()))
        ref.check(dw, each.sum(over), each_size.sum(over), f"d{name}_weight")


# a lane copies a head: more heads than a warp has lanes, at head sizes of which a warp could hold
# 128, 64, 32, 16 and 8 (half of that with a weight a head)
@pytest.mark.parametrize("d,hq,hk", [(8, 130, 33), (8, 200, 64), (16, 64, 33), (16, 65, 1), (32, 40, 33), (64, 33, 2),
                                     (128, 33, 8), (24, 64, 40), (48, 35, 4)])
@pytest.mark.parametrize("gap", [0, 2, 3])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_heads_apart(d, hq, hk, gap, dtype):
    apart_case(1500, hq, hk, d, gap, dtype)


@pytest.mark.parametrize("d,hq,hk", [(8, 130, 33), (16, 64, 33), (16, 65, 1), (32, 40, 33), (128, 33, 8)])
@pytest.mark.parametrize("gap", [0, 3])
def test_heads_apart_with_a_weight_a_head(d, hq, hk, gap):
    apart_case(1200, hq, hk, d, gap, F16, "heads", interleaved=True)


@pytest.mark.parametrize("tokens", [1, 3, 50])
@pytest.mark.parametrize("d", [8, 16])
def test_few_tokens_with_heads_apart(tokens, d):
    """The forward without a ring, the backward with one."""
    apart_case(tokens, 130, 33, d, 2, ring=False)
    apart_case(tokens, 64, 40, d, 3, F16, "heads", ring=False)


def test_inputs_and_gradients_laid_out_differently():
    apart_case(1300, 64, 33, 16, 1, grad_gap=3)
    apart_case(1300, 64, 33, 16, 3, grad_gap=1)
    apart_case(1300, 130, 33, 8, 2, F32, grad_gap=0)


# ------------------------------------------------------------------ head sizes with lanes to spare
@pytest.mark.parametrize("d", [24, 40, 48, 72, 80, 96, 112, 136, 160, 192, 248])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_a_weight_a_head_with_lanes_to_spare(d, dtype, interleaved):
    """Lanes beside the head's columns have no weight of their own and must not reach its sums."""
    apart_case(1200, 7, 3, d, 1, dtype, "heads", interleaved)
    apart_case(1200, 33, 8, d, 1, dtype, "heads", interleaved)


# ------------------------------------------------------------------ eps 0
@pytest.mark.parametrize("d,hq,hk", [(8, 5, 1), (16, 33, 2), (64, 5, 3), (80, 7, 1), (128, 5, 1), (128, 9, 2), (256, 3, 5)])
@pytest.mark.parametrize("weights", ["shared", "heads"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_eps_zero_where_heads_do_not_fill_a_warp(d, hq, hk, weights, dtype):
    """Lanes without a head, whose rstd would be infinite, leave nothing in the weights' gradients."""
    tokens = 1200
    q, k = rand(tokens, hq, d, dtype=dtype, seed=1), rand(tokens, hk, d, dtype=dtype, seed=2)
    dq, dk = rand(tokens, hq, d, dtype=dtype, seed=3), rand(tokens, hk, d, dtype=dtype, seed=4)
    shape = (lambda h: (h, d)) if weights == "heads" else (lambda h: (d,))
    qw, kw = 1 + 0.1 * rand(*shape(hq), seed=5), 1 + 0.1 * rand(*shape(hk), seed=6)
    table, pos = fused.rope_table(tokens, d, device=DEV), torch.arange(tokens, device=DEV)
    cos, sin = ref.cos_sin(pos[None], table, (0,) * (d // 2))
    outs = fused.qk_norm_rope_fwd(q, k, pos, table, qw, kw, eps=0.0)
    gx, gy, gw, gu = fused.qk_norm_rope_bwd(q, k, pos, table, dq, dk, qw, kw, eps=0.0)
    assert on_the_ring()
    for name, x, w, out, dout, dx, dw in (("q", q, qw, outs[0], dq, gx, gw), ("k", k, kw, outs[1], dk, gy, gu)):
        want, size = ref.rope(x, w, cos, sin, False, True, 0.0)
        ref.check(out, want, size, name)
        want, size, each, each_size = ref.rope_backward(x, w, dout, cos, sin, False, True, 0.0)
        ref.check(dx, want, size, "d" + name)
        over = tuple(range(each.dim() - w.dim()))
        ref.check(dw, each.sum(over), each_size.sum(over), f"d{name}_weight")


def on_the_bounds_checked_build(calls):
    """Runs lines of code that use this module as `t` on librmsnorm_b200_debug.so, in a process of
    its own: no access out of range, no wait that ran out."""
    here = Path(__file__).resolve().parent
    lib = here.parent / "rmsnorm-h100_b200" / "rmsnorm" / "lib" / "librmsnorm_b200_debug.so"
    assert lib.exists(), "librmsnorm_b200_debug.so is missing: run __graft_entry__.build()"
    code = """
import json, sys
sys.path[:0] = [%r, %r, %r]
import torch
import test_gpu_rope_ring as t
from rmsnorm import _lib
%s
torch.cuda.synchronize()
print(json.dumps({"build": _lib.debug_bounds_build(), "report": _lib.debug_report(t.DEV), "status": _lib.device_status(t.DEV)}))
""" % (str(here), str(here.parent), str(here.parent / "rmsnorm-h100_b200"), calls)
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, RMSNORM_B200_LIBRARY=str(lib)), capture_output=True,
                       text=True, timeout=600)
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith("{")]
    assert lines, f"no summary (exit {r.returncode}):\n{r.stdout[-2000:]}\n{r.stderr[-2000:]}"
    summary = json.loads(lines[-1])
    assert summary["build"] and summary["report"]["violations"] == 0 and summary["status"] == [0, 0], summary


def test_heads_apart_on_the_bounds_checked_build():
    on_the_bounds_checked_build("""
for c in ((1200, 130, 33, 8, 2), (1200, 64, 33, 16, 3), (1200, 33, 8, 128, 2), (3, 64, 33, 16, 0)):
    t.apart_case(*c, ring=c[0] > 3)
    t.apart_case(*c, t.F16, "heads", ring=c[0] > 3)
""")


def test_a_ring_of_one_slot_on_the_bounds_checked_build():
    """fp32 gradients of heads that leave lanes idle: the lanes without a head reach the next wait
    first, while lane 0 may still have to issue the copy that it is for."""
    on_the_bounds_checked_build("""
for c in ((9215, 5, 5, 8), (2759, 1, 1, 8), (5479, 7, 2, 64), (4227, 3, 1, 64), (6696, 8, 20, 32), (3001, 5, 1, 128)):
    t.apart_case(*c, 1, t.F32)
    assert t._lib.last_plan().endswith("S=1")
    t.apart_case(*c, 1, t.F32, "heads")
""")
