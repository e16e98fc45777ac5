# SPDX-License-Identifier: MIT
"""A cache of keys and values in 8 bits, in pages (`rmsnorm.fused` offers it)."""

from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _host_fused as _host
from . import _lib
from .rmsnorm import _check_optional_dtype

_CODE = _lib._DTYPE_CODES
_MAX_HEADS, _MAX_HEAD_DIM = 65536, 256
_TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
_is_compiling = torch.compiler.is_dynamo_compiling

_CACHE = struct.Struct("qQ3qQ3qQ3qQ3q4i")
_WRITE = struct.Struct("qQ2qQ2qQ2i")
_READ = struct.Struct("4q4Q2i")
for _s, _c in ((_CACHE, _lib.CacheArgs), (_WRITE, _lib.CacheWriteArgs), (_READ, _lib.CacheReadArgs)):
    assert _s.size == ctypes.sizeof(_c), _c.__name__

_BYTES, _STREAM = ctypes.c_char_p, ctypes.c_void_p


def _check_cache(k_cache: Tensor, v_cache: Tensor, k_scales: Tensor, v_scales: Tensor) -> bytes:
    """The cache as the library takes it, checked."""
    code = _lib._QUANT_CODES.get(k_cache.dtype)
    if code is None or v_cache.dtype != k_cache.dtype:
        raise AssertionError("k_cache and v_cache must both be float8_e4m3fn or int8")
    shape = k_cache.shape
    if len(shape) != 4:
        raise ValueError(f"k_cache must be (pages, page_size, heads, head_dim), got {tuple(shape)}")
    if v_cache.shape != shape:
        raise ValueError(f"v_cache must have k_cache's shape {tuple(shape)}, got {tuple(v_cache.shape)}")
    pages, page_size, heads, d = shape
    if not 1 <= heads <= _MAX_HEADS or not 1 <= d <= _MAX_HEAD_DIM or page_size < 1:
        raise ValueError(f"a cache has 1 to {_MAX_HEADS} heads of 1 to {_MAX_HEAD_DIM} columns and pages of at least one "
                         f"slot, got {tuple(shape)}")
    f32, lead, device = torch.float32, shape[:3], k_cache.device
    if k_scales.dtype != f32 or v_scales.dtype != f32 or k_scales.shape != lead or v_scales.shape != lead:
        for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
            if t.dtype != f32 or t.shape != lead:
                raise ValueError(f"{name} must be float32 {tuple(lead)}, got {t.dtype} {tuple(t.shape)}")
    if v_cache.device != device or k_scales.device != device or v_scales.device != device:
        raise ValueError("v_cache, k_scales and v_scales must be on the same device as k_cache")
    ks, vs = k_cache.stride(), v_cache.stride()
    if d > 1 and (ks[3] != 1 or vs[3] != 1):
        raise ValueError("a cache's heads must be contiguous")
    return _CACHE.pack(
        pages, k_cache.data_ptr(), *ks[:3], k_scales.data_ptr(), *k_scales.stride(), v_cache.data_ptr(), *vs[:3],
        v_scales.data_ptr(), *v_scales.stride(), page_size, heads, d, code)


def _repeats(t: Tensor) -> bool:
    stride = t.stride()
    return 0 in stride and any(s == 0 and n > 1 for s, n in zip(stride, t.shape))


def _meet(apart: int, dims, width: int) -> bool:
    """Whether two places of one layout, `apart` from each other, share some of `width` elements:
    dims has (stride, most steps), the largest stride first. Where places do not overlap by
    themselves at most two numbers of steps of a stride bring them near enough to look further."""
    if not dims:
        return -width < apart < width
    (stride, most), rest = dims[0], dims[1:]
    reach = sum(s * n for s, n in rest) + width - 1
    low, high = max(-(-(apart - reach) // stride), -most), min((apart + reach) // stride, most)
    return any(_meet(apart - i * stride, rest, width) for i in range(low, high + 1))


def _overlap(t: Tensor, u: Tensor, lead: Tuple[int, int, int], width: int) -> bool:
    """Whether tensors of one layout (`lead` places of `width` elements) share memory. Of tensors
    with other strides than one another nothing is told but that they begin at the same place."""
    stride, size = t.stride(), t.element_size()
    apart = t.data_ptr() - u.data_ptr()
    a, b, c = lead
    if abs(apart) >= size * ((a - 1) * stride[0] + (b - 1) * stride[1] + (c - 1) * stride[2] + width) or not a:
        return False
    if apart == 0:
        return True
    if stride != u.stride() or apart % size:
        return False
    dims = sorted(((s, n - 1) for s, n in zip(stride, lead) if n > 1), reverse=True)
    return _meet(apart // size, dims, width)


def _heads_of(name: str, t: Tensor, shape: torch.Size, device: torch.device) -> Tuple[Tensor, Tuple[int, int, int]]:
    """t as [tokens, heads, head_dim], a view wherever the strides allow one; its address, token
    stride and head stride."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on the same device as k_cache")
    stride = t.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        t = t.contiguous()
        stride = t.stride()
    if len(stride) != 3:
        t = t.reshape(shape[:-2].numel(), *shape[-2:])
        stride = t.stride()
    return t, (t.data_ptr(), stride[0], stride[1])


def cache_write(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, k_scales: Tensor, v_scales: Tensor,
                slots: Tensor) -> None:
    """Writes tokens into a cache in 8 bits: the heads of k and v (..., heads, head_dim), which
    may be strided views such as slices of a packed projection, as q * scale with q in the
    caches' dtype (float8_e4m3fn or int8; (pages, page_size, heads, head_dim), any strides but
    the last) and an fp32 scale for every head (k_scales, v_scales: (pages, page_size, heads)).
    The four may share a buffer, but no bytes: of two of one kind with the same strides that is an
    error, of others it is not looked at.

    A scale is max |x| / 448 (e4m3) or / 127 (int8), at least 2^-126; q is x over that quotient as
    it is before it is rounded to fp32, rounded to nearest even. A NaN makes its head's scale NaN, an infinity infinite.

    slots (int32 or int64, k's leading shape) has each token's place, page * page_size + place
    in the page. A negative slot leaves its token out. One beyond the cache does too and, on
    CUDA, the device status tells of an invalid argument (on the host it is an IndexError). Slots
    named twice hold bytes of either token. Outside autograd."""
    if _is_compiling():
        return _write_untraced(k, v, k_cache, v_cache, k_scales, v_scales, slots)
    cache = _check_cache(k_cache, v_cache, k_scales, v_scales)
    code = _CODE.get(k.dtype)
    if code is None or v.dtype != k.dtype:
        raise AssertionError("k and v must have the same dtype, float16, bfloat16 or float32")
    if k.dim() < 2:
        raise ValueError("k must have at least two dimensions (heads, head_dim)")
    if slots.dtype != torch.int64 and slots.dtype != torch.int32:
        raise ValueError("slots must be int32 or int64")
    lead = k.shape[:-2]
    if slots.shape != lead:
        raise ValueError(f"slots must have k's leading shape {tuple(lead)}, got {tuple(slots.shape)}")
    if slots.device != k_cache.device:
        raise ValueError("slots must be on the same device as k_cache")
    shape = lead + k_cache.shape[2:]
    kf, k_place = _heads_of("k", k, shape, k_cache.device)
    vf, v_place = _heads_of("v", v, shape, k_cache.device)
    written = (k_cache, v_cache, k_scales, v_scales)
    for t in written:
        if _repeats(t):
            raise ValueError("caches and scales must have places of their own, not be expanded views")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("cache_write is outside autograd: caches and scales must not require gradients")
    *places, d = k_cache.shape
    if _overlap(k_cache, v_cache, places, d) and slots.numel():
        raise ValueError("k_cache and v_cache must be different tensors that do not overlap")
    if _overlap(k_scales, v_scales, places, 1) and slots.numel():
        raise ValueError("k_scales and v_scales must be different tensors that do not overlap")
    if len(lead) != 1:
        slots = slots.reshape(-1)
    if not k_cache.is_cuda:
        keep = slots >= 0
        at = slots[keep].long()
        if at.numel() and int(at.max()) >= k_cache.shape[0] * k_cache.shape[1]:
            raise IndexError("a slot lies beyond the cache")
        page, place = at // k_cache.shape[1], at % k_cache.shape[1]
        with torch.no_grad():
            _host.cache_write(kf[keep], k_cache, k_scales, page, place, _TOP[k_cache.dtype])
            _host.cache_write(vf[keep], v_cache, v_scales, page, place, _TOP[k_cache.dtype])
        return
    slots = slots.contiguous()
    args = _WRITE.pack(slots.shape[0], *k_place, *v_place, slots.data_ptr(), slots.dtype == torch.int64, code)
    name = "rmsnorm_b200_cache_write"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _BYTES, _STREAM), name, k_cache.device.index, cache, args)
    torch.autograd.graph.increment_version(written)


def cache_read(k_cache: Tensor, v_cache: Tensor, k_scales: Tensor, v_scales: Tensor, page_table: Tensor, starts: Tensor,
               tokens: int, dtype: torch.dtype = torch.bfloat16,
               out: Optional[Tuple[Tensor, Tensor]] = None) -> Tuple[Tensor, Tensor]:
    """(k, v), (tokens, heads, head_dim) in `dtype`: sequences read back from a cache that
    `cache_write` filled, one after the other. starts (int32, sequences + 1, ascending from 0)
    has the row where each begins and, last, where they end; row s of page_table (int32,
    (sequences, pages of the longest)) the pages of sequence s in order. Entries behind a
    sequence's last page are not read.

    Rows from starts[-1] on are zeros, or left as they are in `out`, a pair of contiguous
    tensors to write into. Rows before starts[0], and rows whose page lies outside the table or the
    cache, are NaN and, on CUDA, the device status tells of an invalid argument (on the host it is
    an IndexError)."""
    if _is_compiling():
        return _read_untraced(k_cache, v_cache, k_scales, v_scales, page_table, starts, tokens, dtype, out)
    cache = _check_cache(k_cache, v_cache, k_scales, v_scales)
    device = k_cache.device
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise ValueError("page_table must be int32 (sequences, pages)")
    sequences = page_table.shape[0]
    if starts.dtype != torch.int32 or starts.shape != (sequences + 1,):
        raise ValueError(f"starts must be int32 ({sequences + 1},), got {starts.dtype} {tuple(starts.shape)}")
    for name, t in (("page_table", page_table), ("starts", starts)):
        if t.device != device:
            raise ValueError(f"{name} must be on the same device as k_cache")
    if tokens < 0:
        raise ValueError(f"tokens must not be negative, got {tokens}")
    code = _CODE.get(dtype)
    if code is None:
        _check_optional_dtype("dtype", dtype)
    shape = (tokens, *k_cache.shape[2:])
    if out is None:
        k, v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
    else:
        k, v = out
        for t in out:
            if t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
                raise ValueError(f"out must be two contiguous {dtype} tensors of shape {shape} on {device}")
            if t.requires_grad and torch.is_grad_enabled():
                raise ValueError("cache_read is outside autograd: out must not require gradients")
        if abs(k.data_ptr() - v.data_ptr()) < k.numel() * k.element_size():
            raise ValueError("out must be two different tensors that do not overlap")
    if not k_cache.is_cuda:
        if out is None:
            k.zero_()
            v.zero_()
        at = starts.tolist()
        if tokens and at[0] != 0 and at[-1] > 0:
            raise IndexError(f"the first sequence must begin at row 0, got starts[0] = {at[0]}")
        page_size = k_cache.shape[1]
        with torch.no_grad():
            for s in range(sequences):
                n = min(at[s + 1], tokens) - at[s]
                if n <= 0:
                    continue
                pages = page_table[s, : -(-n // page_size)].long()
                if pages.numel() * page_size < n or int(pages.min()) < 0 or int(pages.max()) >= k_cache.shape[0]:
                    raise IndexError("a sequence's page lies outside the table or the cache")
                page = pages.repeat_interleave(page_size)[:n]
                place = torch.arange(page_size).repeat(pages.numel())[:n]
                k[at[s]: at[s] + n] = _host.cache_read(k_cache, k_scales, page, place, dtype)
                v[at[s]: at[s] + n] = _host.cache_read(v_cache, v_scales, page, place, dtype)
        return k, v
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    starts = starts.contiguous()
    args = _READ.pack(tokens, sequences, page_table.shape[1], page_table.stride(0), page_table.data_ptr(),
                      starts.data_ptr(), k.data_ptr(), v.data_ptr(), code, out is None)
    name = "rmsnorm_b200_cache_read"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _BYTES, _STREAM), name, device.index, cache, args)
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return k, v


_write_untraced = torch.compiler.disable(cache_write)
_read_untraced = torch.compiler.disable(cache_read)
