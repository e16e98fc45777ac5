# SPDX-License-Identifier: MIT
"""Waits in the kernels' sources: a wait that whole warps make brings them together first
(mbar_wait_warp). A plain mbar_wait is for single threads: the drain after a failure and the
self test."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "rmsnorm-h100_b200" / "csrc"
SOURCES = sorted(p for p in [*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")] if p.name != "device_common.cuh")


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_plain_waits_are_for_single_threads(path):
    code = "\n".join(line.split("//")[0] for line in path.read_text().splitlines())
    for m in re.finditer(r"\bmbar_(?:try_)?wait(?:_cluster|_slow)?(?:<\w+>)?\s*\(", code):
        call = code[m.start():code.index(";", m.start())]
        assert "kSiteDrain" in call or path.name == "generic_kernels.cuh", f"{path.name}: {call}"


def test_every_site_has_a_number_of_its_own():
    """rmsnorm_b200_device_status tells where something went wrong by a site's number."""
    found = re.findall(r"\b(kSite\w+) = (\d+)", "\n".join(p.read_text() for p in [*SOURCES, CSRC / "device_common.cuh"]))
    assert len(found) > 12
    numbers = [n for _, n in found]
    assert len(set(numbers)) == len(numbers), found
