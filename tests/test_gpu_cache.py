# SPDX-License-Identifier: MIT
"""The quantised cache's kernels against 64 bits (tests/block_ref.py has the error bounds)."""

from __future__ import annotations

import pytest
import torch

import block_ref as ref
from fused_ref import TINY, UNIT
from rmsnorm import _lib, fused

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3, I8 = torch.float8_e4m3fn, torch.int8
TOP = {E4M3: 448.0, I8: 127.0}
INVALID = 1


def rand(*shape, dtype=F32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def new_cache(pages, page_size, heads, d, kept, seed=7):
    """Caches and scales that hold something already (numbers: no NaN)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for _ in range(2):
        b = torch.randint(-119, 120, (pages, page_size, heads, d), device=DEV, generator=g)
        out.append(b.to(I8) if kept == I8 else (b.abs() + (b < 0) * 128).to(torch.uint8).view(E4M3))
    return (*out, torch.rand(pages, page_size, heads, device=DEV, generator=g), torch.rand(pages, page_size, heads, device=DEV, generator=g))


def bits(t):
    return t.contiguous().view(torch.uint8)


def check_write(k, v, cache, slots, before, clear=True):
    """Written slots hold k and v, all others what they held."""
    pages, page_size, heads, d = cache[0].shape
    written = torch.zeros(pages * page_size, dtype=torch.bool, device=DEV)
    keep = (slots >= 0) & (slots < pages * page_size)
    at = slots[keep].long()
    written[at] = True
    for x, q, s, q0, s0 in ((k, cache[0], cache[2], before[0], before[2]), (v, cache[1], cache[3], before[1], before[3])):
        flat, held = q.reshape(-1, heads, d), s.reshape(-1, heads)
        ref.check_cached(flat[at], held[at], x.reshape(-1, heads, d)[keep.reshape(-1)], TOP[q.dtype])
        assert torch.equal(bits(flat[~written]), bits(q0.reshape(-1, heads, d)[~written]))
        assert torch.equal(held[~written], s0.reshape(-1, heads)[~written])
    torch.cuda.synchronize()
    if clear:
        assert _lib.device_status(DEV) == (0, 0)


def write_case(tokens, heads, d, page_size, dtype, kept, slot_dtype=torch.int64, change=lambda t: t):
    pages = tokens // page_size + 3
    cache = new_cache(pages, page_size, heads, d, kept)
    before = [t.clone() for t in cache]
    g = torch.Generator(device=DEV).manual_seed(1)
    slots = torch.randperm(pages * page_size, device=DEV, generator=g)[:tokens].to(slot_dtype)
    slots[tokens // 2 + 1:: 5] = -1
    k, v = change(rand(tokens, heads, d, dtype=dtype, seed=2)), change(3 * rand(tokens, heads, d, dtype=dtype, seed=3))
    fused.cache_write(k, v, *cache, slots)
    check_write(k, v, cache, slots, before)


@pytest.mark.parametrize("d", [1, 7, 8, 64, 65, 80, 96, 127, 128, 136, 192, 255, 256])
@pytest.mark.parametrize("kept", [E4M3, I8])
def test_write_head_sizes(d, kept):
    for tokens, heads in ((1, 1), (5, 3), (700, 4)):
        write_case(tokens, heads, d, 16, BF16, kept)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("slot_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("page_size", [1, 17, 64])
def test_write_types_and_pages(dtype, slot_dtype, page_size):
    write_case(1, 8, 128, page_size, dtype, E4M3, slot_dtype)
    write_case(3000, 8, 128, page_size, dtype, E4M3, slot_dtype)


@pytest.mark.parametrize("d", [1, 7, 64, 65, 72, 128, 129, 136, 200, 256])
@pytest.mark.parametrize("dtype,kept", [(BF16, E4M3), (F16, E4M3), (BF16, I8)])
def test_write_of_many_tokens(d, dtype, kept):
    """So many that a lane takes two octets of a head; bits as when they are written few at a time."""
    tokens, heads = 16001, 5
    write_case(tokens, heads, d, 16, dtype, kept)
    k, v = rand(tokens, heads, d, dtype=dtype, seed=4), rand(tokens, heads, d, dtype=dtype, seed=5)
    k[3, 1, d // 2], k[4, 2, d - 1], v[5, 0, 0], v[6] = float("nan"), float("inf"), float("-inf"), 0
    k[100:200] *= 2.0 ** (-130 if dtype == BF16 else -20)
    slots = torch.randperm(16 * 1001, device=DEV)[:tokens]
    one, other = new_cache(1001, 16, heads, d, kept), new_cache(1001, 16, heads, d, kept)
    fused.cache_write(k, v, *one, slots)
    for at in range(0, tokens, 1000):
        fused.cache_write(k[at: at + 1000], v[at: at + 1000], *other, slots[at: at + 1000])
    assert all(torch.equal(bits(x), bits(y)) for x, y in zip(one, other))


def test_write_strided_inputs_and_caches():
    odd = lambda t: torch.cat([t, t], -1)[..., 1: 1 + t.shape[-1]]  # noqa: E731 -- off any 16 bytes
    for d in (64, 128):
        write_case(300, 4, d, 16, BF16, E4M3, change=odd)
        write_case(300, 4, d, 16, F32, I8, change=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1))
        write_case(300, 4, d, 16, BF16, I8, change=lambda t: t.mT.contiguous().mT)
        write_case(40, 4, d, 16, BF16, E4M3, change=lambda t: t[:, :1].expand(-1, 4, -1))
    # a packed projection; heads before slots in the cache; a cache that begins off 8 bytes
    for shift in (0, 3):
        packed = rand(50, 3 * 4 * 64, dtype=BF16)
        k, v = packed[:, 256:512].view(50, 4, 64), packed[:, 512:].view(50, 4, 64)
        whole = torch.zeros(2, 9 * 4 * 8 * 64 + shift, dtype=torch.uint8, device=DEV)
        cache = [w[shift:].view(9, 4, 8, 64).transpose(1, 2).view(E4M3) for w in whole]
        cache += [torch.zeros(4, 8, 9, device=DEV).permute(2, 1, 0) for _ in range(2)]
        before = [t.clone() for t in cache]
        slots = torch.randperm(72, device=DEV)[:50]
        fused.cache_write(k, v, *cache, slots)
        check_write(k, v, cache, slots, before)
        table, starts = torch.arange(9, dtype=torch.int32, device=DEV)[None], torch.tensor([0, 72], dtype=torch.int32, device=DEV)
        rk, rv = fused.cache_read(*cache, table, starts, 72, F32)
        assert torch.equal(rk, (cache[0].float() * cache[2][..., None]).reshape(72, 4, 64))
        assert torch.equal(rv, (cache[1].float() * cache[3][..., None]).reshape(72, 4, 64))


def test_write_leading_dimensions_and_none():
    cache = new_cache(8, 16, 2, 64, E4M3)
    before = [t.clone() for t in cache]
    k, v = rand(3, 7, 2, 64), rand(3, 7, 2, 64, seed=1)
    slots = torch.randperm(128, device=DEV)[:21].view(3, 7)
    versions = [t._version for t in cache]
    fused.cache_write(k, v, *cache, slots)
    assert all(t._version > n for t, n in zip(cache, versions))
    check_write(k, v, cache, slots, before)
    fused.cache_write(k[:0], v[:0], *cache, slots[:0])
    fused.cache_write(k, v, *cache, torch.full_like(slots, -5))
    check_write(k, v, cache, slots, before)
    one = rand(2, 64)
    fused.cache_write(one, one, *cache, torch.tensor(3, device=DEV))
    ref.check_cached(cache[0].view(-1, 2, 64)[3], cache[2].view(-1, 2)[3], one, 448.0)


def test_write_slots_beyond_the_cache_are_left_out_and_told():
    cache = new_cache(4, 16, 2, 64, E4M3)
    before = [t.clone() for t in cache]
    k, v = rand(6, 2, 64), rand(6, 2, 64, seed=1)
    slots = torch.tensor([3, 64, 5, 1 << 40, 63, 65], device=DEV)
    fused.cache_write(k, v, *cache, slots)
    check_write(k, v, cache, slots, before, clear=False)
    assert _lib.device_status(DEV, clear=True) == (INVALID, 11)
    fused.cache_write(k[:3], v[:3], *cache, torch.tensor([1, 2, 3], device=DEV))
    torch.cuda.synchronize()
    assert _lib.device_status(DEV) == (0, 0)


@pytest.mark.parametrize("kept", [E4M3, I8])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_write_ties_go_to_even(kept, dtype):
    """16-bit x: q is the number nearest to Q x / max |x| in exact arithmetic, ties to even."""
    k = rand(4000, 2, 128, dtype=dtype, seed=5)
    k[:1000] = k[:1000] * torch.exp2(torch.arange(1000, device=DEV) % 20 - 10.0)[:, None, None]
    cache = new_cache(4000, 1, 2, 128, kept)
    fused.cache_write(k, k, *cache, torch.arange(4000, device=DEV))
    x = k.double()
    most = x.abs().amax(-1, keepdim=True)
    v = x * TOP[kept] / most  # a tie has few bits: 53 give it exactly, and keep what is none apart
    want = v.round() if kept == I8 else ref.nearest_e4m3(v)
    assert torch.equal(cache[0].view(4000, 2, 128).double(), want)


@pytest.mark.parametrize("kept", [E4M3, I8])
@pytest.mark.parametrize("power", [-135, -118, -100, 0, 100, 120])
def test_write_at_the_ends_of_the_range(kept, power):
    k = (rand(50, 1, 64, seed=6).double() * 2.0**power).float()
    k[0, 0, 0], k[1, 0, 5] = torch.finfo(F32).max, -torch.finfo(F32).max
    cache = new_cache(50, 1, 1, 64, kept)
    fused.cache_write(k, k, *cache, torch.arange(50, device=DEV))
    ref.check_cached(cache[0].view(50, 1, 64), cache[2].view(50, 1), k, TOP[kept])


@pytest.mark.parametrize("kept", [E4M3, I8])
def test_write_zeros_nan_and_infinity(kept):
    cache = new_cache(1, 8, 1, 64, kept)
    k = torch.zeros(5, 1, 64, device=DEV)
    k[1, 0, 3], k[2, 0, 4], k[3, 0, 5], k[4, 0, :2] = float("nan"), float("inf"), float("-inf"), 1e-44
    k[1:4, 0, 9] = 2.0
    fused.cache_write(k, k, *cache, torch.arange(5, device=DEV))
    s = cache[2][0, :5, 0]
    assert s[0] == 2.0**-126 and s[1].isnan() and s[2].isinf() and s[3].isinf() and s[4] == 2.0**-126
    q = cache[0][0, :5, 0].double()
    assert (q[0] == 0).all() and q[2, 9] == 0 and q[3, 9] == 0 and (q[4] == 0).all()


def read_case(lengths, heads, d, page_size, kept, dtype, extra_rows=0, out=False):
    """Sequences of these lengths at any pages; unused entries of the table name no page."""
    starts = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    each = [-(-n // page_size) for n in lengths]
    pages = sum(each) + 2
    cache = new_cache(pages, page_size, heads, d, kept)
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist()
    table = torch.full((len(lengths), max(each, default=0) + 1), -7, dtype=torch.int32)
    at = 0
    for i, n in enumerate(each):
        table[i, :n] = torch.tensor(free[at: at + n], dtype=torch.int32)
        at += n
    table = table.to(DEV)
    total = sum(lengths)
    into = None
    if out:
        into = tuple(torch.full((total + extra_rows, heads, d), 5.0, dtype=dtype, device=DEV) for _ in range(2))
    got = fused.cache_read(*cache, table, starts, total + extra_rows, dtype, into)
    for which in range(2):
        parts = []
        for i, n in enumerate(lengths):
            p = table[i, : each[i]].long()
            parts.append((cache[which][p].double() * cache[2 + which][p].double()[..., None]).flatten(0, 1)[:n])
        want = torch.cat(parts) if parts else torch.zeros(0, heads, d, device=DEV, dtype=torch.float64)
        r = got[which]
        assert r.shape == (total + extra_rows, heads, d) and r.dtype == dtype
        # a product of two numbers in fp32, rounded to the type: half a step of each
        off = (r[:total].double() - want).abs()
        assert (off <= (UNIT[dtype] + 2.0**-23) * want.abs() + TINY[dtype]).all()
        assert (r[total:] == (5.0 if out else 0.0)).all()
        if out:
            assert r is into[which]
    torch.cuda.synchronize()
    assert _lib.device_status(DEV) == (0, 0)


@pytest.mark.parametrize("d", [1, 7, 8, 64, 65, 80, 128, 192, 255, 256])
@pytest.mark.parametrize("kept", [E4M3, I8])
def test_read_head_sizes(d, kept):
    for heads in (1, 3, 8):
        read_case([5, 0, 33, 1], heads, d, 16, kept, BF16, 3)


@pytest.mark.parametrize("lengths", [[1], [0], [0, 0, 3], [16], [17, 15], [1000], [1] * 300, [0] * 40 + [7] + [0] * 40,
                                     [3000, 1, 2000, 0, 77]])
@pytest.mark.parametrize("page_size", [1, 16, 17])
def test_read_lengths(lengths, page_size):
    read_case(lengths, 4, 128, page_size, E4M3, BF16, 2)
    read_case(lengths, 2, 64, page_size, I8, F32, 200, out=True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_read_types(dtype):
    read_case([100, 300], 8, 128, 64, E4M3, dtype, 5, out=True)
    read_case([40000, 3], 1, 96, 64, I8, dtype)


def test_read_of_no_sequences_and_no_rows():
    cache = new_cache(2, 16, 2, 64, E4M3)
    none = torch.zeros(0, 4, dtype=torch.int32, device=DEV)
    starts = torch.zeros(1, dtype=torch.int32, device=DEV)
    k, v = fused.cache_read(*cache, none, starts, 5)
    assert (k == 0).all() and (v == 0).all()
    k, v = fused.cache_read(*cache, none, starts, 0)
    assert k.shape == (0, 2, 64)


def test_read_bad_pages_are_nan_and_told():
    cache = new_cache(4, 16, 2, 64, E4M3)
    table = torch.tensor([[0, 1], [2, 9], [-1, 3]], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 20, 52, 68], dtype=torch.int32, device=DEV)
    k, v = fused.cache_read(*cache, table, starts, 70, F32)
    for t in (k, v):
        assert t[36:68].isnan().all() and not t[:36].isnan().any() and (t[68:] == 0).all()
    assert _lib.device_status(DEV, clear=True) == (INVALID, 12)
    # a sequence longer than its row of the table, and rows before the first
    long = torch.tensor([1, 40], dtype=torch.int32, device=DEV)
    k, v = fused.cache_read(*cache, table[:1], long, 40, F32)
    assert k[0].isnan().all() and not k[1:33].isnan().any() and k[33:].isnan().all()
    assert _lib.device_status(DEV, clear=True) == (INVALID, 12)


def test_far_slots_of_a_long_cache():
    """Offsets beyond 32 bits: 5 GiB of keys."""
    pages, page_size, heads, d = 5 * 1024, 512, 8, 256
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GiB")
    k_cache = torch.zeros(pages, page_size, heads, d, dtype=torch.uint8, device=DEV).view(E4M3)
    scales = [torch.zeros(pages, page_size, heads, device=DEV) for _ in range(2)]
    v_cache = torch.zeros_like(k_cache.view(torch.uint8)).view(E4M3)
    k, v = rand(40, heads, d, dtype=BF16), rand(40, heads, d, dtype=BF16, seed=1)
    slots = torch.arange(40, device=DEV) * 65000 + 17
    slots[-1] = pages * page_size - 1
    fused.cache_write(k, v, k_cache, v_cache, *scales, slots)
    ref.check_cached(k_cache.view(-1, heads, d).view(torch.uint8)[slots].view(E4M3), scales[0].view(-1, heads)[slots], k, 448.0)
    table = (slots // page_size).to(torch.int32)[:, None]
    starts = torch.arange(0, 41 * page_size, page_size, dtype=torch.int32, device=DEV)
    rk, rv = fused.cache_read(k_cache, v_cache, *scales, table, starts, 40 * page_size)
    at = torch.arange(40, device=DEV) * page_size + slots % page_size
    assert (rk[at].float() - k.float()).abs().max() < 0.3 and (rv[at].float() - v.float()).abs().max() < 0.3
    assert int((rk != 0).any(-1).any(-1).sum()) == 40


def test_cache_in_graphs_and_on_streams():
    """A captured step that writes one token of each sequence and reads all of them back."""
    sequences, page_size, heads, d = 6, 16, 4, 128
    cache = new_cache(40, page_size, heads, d, E4M3)
    table = torch.randperm(40, device=DEV)[: sequences * 6].view(sequences, 6).to(torch.int32)
    k, v = rand(sequences, heads, d, dtype=BF16), rand(sequences, heads, d, dtype=BF16, seed=1)
    slots = torch.zeros(sequences, dtype=torch.int64, device=DEV)
    starts = torch.zeros(sequences + 1, dtype=torch.int32, device=DEV)
    out = tuple(torch.zeros(400, heads, d, dtype=BF16, device=DEV) for _ in range(2))

    def step():
        fused.cache_write(k, v, *cache, slots)
        return fused.cache_read(*cache, table, starts, 400, BF16, out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for n in (1, 16, 17, 60):
        length = torch.tensor([n, n, 1, n, 2, n], dtype=torch.int32, device=DEV)
        starts[1:] = length.cumsum(0)
        pos = length.long() - 1
        slots.copy_(table[torch.arange(sequences), pos // page_size].long() * page_size + pos % page_size)
        k.copy_(rand(sequences, heads, d, dtype=BF16, seed=n))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = fused.cache_read(*cache, table, starts, 400, BF16)
        total = int(starts[-1])
        assert all(torch.equal(a[:total], b[:total]) for a, b in zip(got, want))
        last = starts[1:].long() - 1
        assert (got[0][last].float() - k.float()).abs().max() < 0.3
    assert _lib.device_status(DEV) == (0, 0)
