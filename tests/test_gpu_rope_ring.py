# SPDX-License-Identifier: MIT
"""The rotary kernels that stream a warp's heads through a ring, where their data or layout is
out of the ordinary: positions outside the table beside ordinary ones."""

from __future__ import annotations

import pytest
import torch

from rmsnorm import _lib, fused
from test_gpu_fused import BF16, DEV, F32, rand

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
