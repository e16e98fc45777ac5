# SPDX-License-Identifier: MIT
"""Cases of the 8-bit products and the quantised cache run through the bounds-checked build
(selected with RMSNORM_B200_LIBRARY by tests/test_gpu_block_bounds.py, which starts this script
as a child process). Every case is checked against 64 bits as in the tests it comes from, then
the build's report and the device status word are read. A last case registers an output short,
so that the checker has something to find. Prints one JSON summary line."""

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

import test_gpu_block as b  # noqa: E402
import test_gpu_cache as c  # noqa: E402
from rmsnorm import _lib, fused  # noqa: E402

BF16, F16, F32, E4M3, I8 = c.BF16, c.F16, c.F32, c.E4M3, c.I8


def cases():
    for rows, cols in ((1, 1), (3, 7), (127, 129), (129, 127), (300, 1001), (1, 5000), (2000, 16), (1000, 4096)):
        for dtype in (BF16, F32):
            for block_rows in (1, 128):
                yield f"quantize {rows} {cols}", lambda r=rows, n=cols, d=dtype, br=block_rows: b.test_quantize(r, n, d, br)
    for m in (1, 17, 33, 100, 129, 500):
        for n, k in ((1, 1), (127, 129), (520, 2049), (4100, 512)):
            yield f"product {m} {n} {k}", lambda m=m, n=n, k=k: b.product_case(m, n, k, 128 if n > 200 else 1, F32)
    for m, n, k in ((1000, 1040, 640), (777, 4100, 384), (64, 16384, 300)):
        for out in (BF16, F16):
            yield f"product {m} {n} {k} {out}", lambda m=m, n=n, k=k, o=out: b.product_case(m, n, k, 128, o)
    for m, n, k in ((1000, 4096, 640), (2300, 5000, 300), (300, 12345, 130)):
        yield f"powers {m} {n} {k}", lambda m=m, n=n, k=k: b.power_case(m, n, k, 1, BF16)
    for m in (1, 130, 600):
        yield f"product off 16 bytes {m}", lambda m=m: b.product_case(m, 1300, 1001, 128, F32, True, b.shifted, b.padded)
    for t, n, k in ((7, 100, 300), (333, 520, 1001), (1500, 1300, 640)):
        yield f"linear {t}", lambda t=t, n=n, k=k: b.test_linear(t, n, k, BF16, F32)
    for d in (1, 7, 64, 80, 128, 255, 256):
        for kept in (E4M3, I8):
            yield f"cache write {d}", lambda d=d, q=kept: c.write_case(700, 5, d, 16, BF16, q)
            yield f"cache read {d}", lambda d=d, q=kept: c.read_case([5, 0, 333, 1], 5, d, 17, q, F16, 3)
    for d in (7, 72, 128, 200):
        yield f"cache write of many {d}", lambda d=d: c.write_case(16001, 5, d, 16, BF16, E4M3)
    yield "cache strides", c.test_write_strided_inputs_and_caches
    yield "cache far", c.test_write_leading_dimensions_and_none
    yield "cache one", lambda: c.write_case(1, 1, 128, 64, F32, E4M3)


def main() -> int:
    failures, n = [], 0
    for name, case in cases():
        n += 1
        try:
            case()
        except Exception as exc:  # noqa: BLE001
            failures.append([name, repr(exc)[:300]])
        torch.cuda.synchronize()
        report = _lib.debug_report(c.DEV, clear=True)
        status = _lib.device_status(c.DEV, clear=True)
        if report["violations"] or status != (0, 0):
            failures.append([name, report, status])
    a, sa = b.operand(200, 256, 1, 1)
    w, sw = b.operand(9600, 256, 128, 2)
    want = fused.block_mm(a, sa, w, sw)
    torch.cuda.synchronize()
    fill = torch.full_like(want, 7.0)
    os.environ["RMSNORM_B200_DEBUG_CLIP_OUT"] = str(9600 * 2)
    original = torch.empty
    torch.empty = lambda *s, **k: fill if s == (200, 9600) else original(*s, **k)
    got = fused.block_mm(a, sa, w, sw)
    torch.empty = original
    torch.cuda.synchronize()
    report = _lib.debug_report(c.DEV, clear=True)
    clip = {"violations": report["violations"], "site": report["site"], "last_row_untouched": bool((got[-1] == 7).all()),
            "rest_ok": bool(torch.equal(got[:-1], want[:-1]))}
    print(json.dumps({"cases": n, "failures": failures, "clip": clip, "debug_build": _lib.debug_bounds_build()}))
    return 1 if failures else 0


if __name__ == "__main__":
    sys.exit(main())
