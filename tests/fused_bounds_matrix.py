# SPDX-License-Identifier: MIT
"""Cases of the fused operators run through the bounds-checked build (selected with
RMSNORM_B200_LIBRARY by tests/test_gpu_fused_bounds.py, which starts this script as a child
process). Every case is checked against 64 bits as in tests/test_gpu_fused.py, then the
build's report and the device status word are read. A last case registers an output one row
short, so that the checker has something to find. Prints one JSON summary line."""

from __future__ import annotations

import json
import os
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
for p in (str(HERE), str(HERE.parent), str(HERE.parent / "rmsnorm-h100_b200")):
    if p not in sys.path:
        sys.path.insert(0, p)

import torch  # noqa: E402

import test_gpu_fused as t  # noqa: E402
from rmsnorm import _lib, fused  # noqa: E402

BF16, F16, F32, E4M3, I8 = t.BF16, t.F16, t.F32, t.E4M3, t.I8


def cases():
    for n in (8, 100, 256, 264, 1001, 2048, 4100, 5120, 8192, 16384, 16392, 24576, 32768, 65536, 270000):
        rows = t.rows_for(n)
        yield f"quant {n}", lambda n=n, r=rows: t.quant_case(r, n, BF16, BF16, None, True, True, E4M3, 128)
        yield f"quant row {n}", lambda n=n, r=rows: t.quant_case(r, n, F16, None, None, True, False, I8, None)
        yield f"dropout fwd {n}", lambda n=n, r=rows: t.drop_case(r, n, BF16, BF16, F32, None, True, True)
        yield f"dropout bwd {n}", lambda n=n, r=rows: t.bwd_case(r, n, BF16, BF16, BF16, True, True)
        yield f"dropout bwd f32 {n}", lambda n=n, r=rows: t.bwd_case(r, n, F32, BF16, F32, True, False)
    for n in (3, 9, 252, 1003, 1006, 4099, 16387):  # vectors shared by neighbouring rows
        for r in (1, 5, 301):
            yield f"odd quant {n} {r}", lambda n=n, r=r: t.quant_case(r, n, BF16, BF16, None, True, True, E4M3, 32)
            yield f"odd quant row {n} {r}", lambda n=n, r=r: t.quant_case(r, n, F32, None, None, True, False, I8, None)
            yield f"odd dropout fwd {n} {r}", lambda n=n, r=r: t.drop_case(r, n, F16, F16, F32, None, True, True)
            yield f"odd dropout bwd {n} {r}", lambda n=n, r=r: t.bwd_case(r, n, F32, BF16, F32, True, True)
    for rows in (1, 147, 149):
        yield f"quant rows {rows}", lambda r=rows: t.quant_case(r, 4096, F32, F32, None, True, False, E4M3, None)
        yield f"dropout rows {rows}", lambda r=rows: t.bwd_case(r, 4096, F16, F16, None, True, True)
    yield "quant unaligned", lambda: t.quant_case(50, 512, BF16, BF16, None, True, True, E4M3, 64, t.unaligned)
    yield "dropout unaligned", lambda: t.drop_case(50, 1003, F32, F32, None, None, True, True, change=t.unaligned)
    yield "dropout bwd unaligned", lambda: t.bwd_case(50, 1003, BF16, BF16, BF16, True, True, change=t.unaligned)
    yield "quant mixed types", lambda: t.quant_case(67, 1001, F32, BF16, F16, True, True, I8, 32)
    for tokens in (1, 64, 999):
        for weights in ("shared", "heads"):
            yield f"rope {tokens} {weights}", lambda n=tokens, w=weights: t.rope_case(n, 32, 8, 128, 128, (16, 24, 24), weights=w)
    for d, rd in ((10, 6), (64, 32), (80, 80), (256, 256)):
        yield f"rope {d}", lambda d=d, rd=rd: t.rope_case(133, 5, 2, d, rd, (rd // 2,), d == 80, dtype=F32)
    yield "rope odd stride", lambda: t.rope_case(65, 6, 2, 128, 128, (64,), packed=False)


def main() -> int:
    failures, n = [], 0
    for name, case in cases():
        n += 1
        try:
            case()
        except Exception as exc:  # noqa: BLE001
            failures.append([name, repr(exc)[:300]])
        torch.cuda.synchronize()
        report = _lib.debug_report(t.DEV, clear=True)
        status = _lib.device_status(t.DEV, clear=True)
        if report["violations"] or status != (0, 0):
            failures.append([name, report, status])
    x = t.rand(20, 512, dtype=BF16)
    want = fused.rmsnorm_quant_fwd(x)[0].view(torch.uint8)
    torch.cuda.synchronize()
    fill = torch.full_like(want, 0x55)
    os.environ["RMSNORM_B200_DEBUG_CLIP_OUT"] = "512"
    original = torch.empty_like
    torch.empty_like = lambda *a, **k: fill.view(torch.float8_e4m3fn) if k.get("dtype") == torch.float8_e4m3fn else original(*a, **k)
    got = fused.rmsnorm_quant_fwd(x)[0].view(torch.uint8)
    torch.empty_like = original
    torch.cuda.synchronize()
    report = _lib.debug_report(t.DEV, clear=True)
    clip = {"violations": report["violations"], "site": report["site"], "last_row_untouched": bool((got[-1] == 0x55).all()),
            "rest_ok": bool((got[:-1] == want[:-1]).all())}
    print(json.dumps({"cases": n, "failures": failures, "clip": clip, "debug_build": _lib.debug_bounds_build()}))
    return 1 if failures else 0


if __name__ == "__main__":
    sys.exit(main())
