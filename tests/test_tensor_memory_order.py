# SPDX-License-Identifier: MIT
"""Kernels that take tensor memory, by their sources: a launch that follows one of them with
programmatic dependent launch may ask for tensor memory itself and then wait for the kernel before
it, so a kernel lets its dependents start only once it holds its own. Were the order the other way
round, both could wait for one another without an end, which no run may show."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "rmsnorm-h100_b200" / "csrc"


def body_at(text: str, at: int) -> str:
    """The block in braces that begins behind `at`."""
    first = text.index("{", at)
    depth = 0
    for i in range(first, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[first: i + 1]
    raise AssertionError("no end")


def kernels():
    for path in sorted([*CSRC.glob("*.cuh"), *CSRC.glob("*.cu")]):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__.*?\b(\w+_kernel)\s*\(", text, re.S):
            yield m.group(1), body_at(text, m.end()), text


TAKING = [(name, body) for name, body, _ in kernels() if "tmem_alloc" in body]


def test_the_kernels_that_take_tensor_memory_are_found():
    assert {n for n, _ in TAKING} >= {"block_mm_wide_kernel", "block_mm_scaled_kernel", "block_mm_few_kernel", "shift_bwd_kernel",
                                      "fused_bwd_kernel", "bwd_stream_kernel"}
    assert "__syncthreads" in body_at(*next((t, t.index("void init_barriers")) for _, _, t in kernels() if "void init_barriers" in t))


@pytest.mark.parametrize("name,body", TAKING, ids=[n for n, _ in TAKING])
def test_dependents_start_once_tensor_memory_is_held(name, body):
    taken = [m.end() for m in re.finditer(r"tmem_alloc\w*\(", body)]
    assert len(taken) == 1
    let = [m.start() for m in re.finditer(r"pdl_launch_dependents\(", body)]
    assert let
    for at in let:
        if "} else {" in body[taken[0]: at] and body[taken[0]: at].rstrip().endswith("} else {"):
            continue  # the variant that takes none
        assert at > taken[0], "before tensor memory is taken"
        between = body[taken[0]: at]
        # a barrier of the CTA, or the warp that took it, in the same block
        assert "__syncthreads" in between or "init_barriers(" in between or "}" not in between


def test_warps_come_together_before_they_read_tensor_memory():
    """tcgen05.ld takes a whole warp, converged. In a loop that a warp leaves some of its lanes behind
    in (stores of rows inside the matrix, returns of columns outside it), it comes together first."""
    found = 0
    for name, body in TAKING:
        for m in re.finditer(r"\bfor\s*\([^{;]*;[^{;]*;[^{;]*\)\s*\{", body):
            loop = body_at(body, m.end() - 1)
            read = loop.find("tmem_ld(")
            if read < 0 or not re.search(r"store_turned\(|if \(row < p\.m\)", loop) or re.search(r"\bfor\s*\([^{]*\)\s*\{[^}]*tmem_ld\(", loop):
                continue
            found += 1
            assert "__syncwarp();" in loop[:read], f"{name}: {loop[:read]}"
    assert found == 1
