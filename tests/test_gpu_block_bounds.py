# SPDX-License-Identifier: MIT
"""The 8-bit products and the quantised cache on the bounds-checked build
(librmsnorm_b200_debug.so): no failed check over tests/block_bounds_matrix.py, and the checker
finds an output registered a row short."""

from __future__ import annotations

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

HERE = Path(__file__).resolve().parent
DEBUG_LIB = HERE.parent / "rmsnorm-h100_b200" / "rmsnorm" / "lib" / "librmsnorm_b200_debug.so"


def test_block_matrix_is_clean_under_the_bounds_checked_build():
    assert DEBUG_LIB.exists(), "librmsnorm_b200_debug.so is missing: run __graft_entry__.build()"
    env = dict(os.environ, RMSNORM_B200_LIBRARY=str(DEBUG_LIB))
    r = subprocess.run([sys.executable, str(HERE / "block_bounds_matrix.py")], env=env, capture_output=True, text=True,
                       timeout=1200)
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith("{")]
    assert lines, f"no summary (exit {r.returncode}):\n{r.stdout[-2000:]}\n{r.stderr[-2000:]}"
    summary = json.loads(lines[-1])
    assert summary["debug_build"] and summary["cases"] >= 90
    assert not summary["failures"], json.dumps(summary["failures"][:5], indent=1)
    clip = summary["clip"]
    assert clip["violations"] > 0 and clip["site"] == 2 and clip["last_row_untouched"] and clip["rest_ok"], clip
