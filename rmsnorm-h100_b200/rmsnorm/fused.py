# SPDX-License-Identifier: MIT
"""Operators fused with the norm, on the kernels of librmsnorm_b200:

* `rmsnorm_quant_fwd` -- residual addition + RMSNorm with an 8-bit output and scales;
* `dropout_add_rmsnorm` (`_fwd`, `_bwd`) -- dropout from a counter-based generator, residual
  addition and RMSNorm; the mask is never stored;
* `qk_norm_rope` (`_fwd`, `_bwd`) -- per-head RMSNorm of q and k with rotary positions on one
  to four axes (`rope_table`, `rope_axes`).

They follow the conventions of `rmsnorm.rmsnorm`: arguments are checked before anything
runs, CUDA tensors go to the native library on the current stream of their device, tensors
on the host are computed in plain PyTorch. Under `torch.compile` they run as graph breaks.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _host_fused as _host
from . import _lib
from .rmsnorm import (
    _check_optional_dtype,
    _check_same_device,
    _check_tensor_dtype,
    _check_x_shape,
    _contig,
    _SUPPORTED_DTYPES,
)

__all__ = [
    "DropoutAddRMSNormFunction",
    "QKNormRopeFunction",
    "dropout_add_rmsnorm",
    "dropout_add_rmsnorm_bwd",
    "dropout_add_rmsnorm_fwd",
    "dropout_mask",
    "qk_norm_rope",
    "qk_norm_rope_bwd",
    "qk_norm_rope_fwd",
    "rmsnorm_quant_fwd",
    "rope_axes",
    "rope_table",
]

_CODE = _lib._DTYPE_CODES
_GROUP_SIZES = (None, 32, 64, 128, 256)


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _code(t: Optional[Tensor]) -> int:
    return 0 if t is None else _CODE[t.dtype]


def _check_affine(name: str, t: Optional[Tensor], n: int, device: torch.device) -> None:
    if t is None:
        return
    if t.dtype not in _SUPPORTED_DTYPES:
        _check_tensor_dtype(name.capitalize(), t)
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} shape must be (N,) with N={n}, got {tuple(t.shape)}")
    if t.device != device:
        _check_same_device(name, t, device)


def _check_like(name: str, t: Optional[Tensor], x: Tensor) -> None:
    if t is None:
        return
    if t.dtype not in _SUPPORTED_DTYPES:
        _check_tensor_dtype(name.capitalize(), t)
    if t.shape != x.shape:
        raise ValueError(f"{name} shape must match x shape {tuple(x.shape)}, got {tuple(t.shape)}")
    if t.device != x.device:
        _check_same_device(name, t, x.device)


def _check_row_input(x: Tensor, weight, bias, residual) -> None:
    if x.dtype not in _SUPPORTED_DTYPES:
        raise AssertionError("Unsupported dtype")
    _check_x_shape(x.shape)
    n = x.shape[-1]
    _check_affine("weight", weight, n, x.device)
    _check_affine("bias", bias, n, x.device)
    _check_like("residual", residual, x)


# ---------------------------------------------------------------------------------------
# Residual addition + RMSNorm with an 8-bit output
# ---------------------------------------------------------------------------------------
@torch.compiler.disable
def rmsnorm_quant_fwd(
    x: Tensor,
    weight: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    residual: Optional[Tensor] = None,
    quant_dtype: torch.dtype = torch.float8_e4m3fn,
    group_size: Optional[int] = None,
    residual_dtype: Optional[torch.dtype] = None,
    eps: float = 1e-6,
    scales_column_major: bool = False,
) -> Tuple[Tensor, Tensor, Tensor]:
    """(q, scales, residual_out): y = RMSNorm(x + residual) * weight + bias in fp32, held as
    q * scales with q in `quant_dtype` (float8_e4m3fn or int8) and fp32 scales, one per row
    (shape x.shape[:-1]) or, with `group_size` 32, 64, 128 or 256, one per group of that
    many columns (shape x.shape[:-1] + (groups,), the last group possibly shorter).

    A scale is max |y| / 448 (e4m3) or / 127 (int8), at least 2^-126; q is rounded to nearest
    even. NaN in a group makes its scale NaN. `scales_column_major` lays grouped scales out
    column by column (the strides of a transposed tensor), as block-scaled products take
    them. residual_out as in `rmsnorm_fwd`."""
    _check_row_input(x, weight, bias, residual)
    if residual_dtype is not None:
        _check_optional_dtype("residual_dtype", residual_dtype)
    if quant_dtype not in _lib._QUANT_CODES:
        raise AssertionError("quant_dtype must be float8_e4m3fn or int8")
    if group_size not in _GROUP_SIZES:
        raise ValueError(f"group_size must be None, 32, 64, 128 or 256, got {group_size}")
    shape = x.shape
    n = shape[-1]
    rows = x.numel() // n
    row_stride, group_stride = 1, 0
    if group_size is None:
        scales = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    else:
        groups = -(-n // group_size)
        if scales_column_major:
            scales = torch.empty((groups, *shape[:-1]), dtype=torch.float32, device=x.device).movedim(0, -1)
            row_stride, group_stride = 1, rows
        else:
            scales = torch.empty((*shape[:-1], groups), dtype=torch.float32, device=x.device)
            row_stride, group_stride = groups, 1
    if not x.is_cuda:
        q, residual_out = _host.rmsnorm_quant_fwd(
            x, weight, bias, residual, quant_dtype, group_size, residual_dtype, eps, scales)
        return q, scales, residual_out
    x = _contig(x)
    residual = _contig(residual)
    weight = _contig(weight)
    bias = _contig(bias)
    q = torch.empty(shape, dtype=quant_dtype, device=x.device)
    residual_out = None
    if residual is not None:
        residual_out = torch.empty(shape, dtype=residual_dtype or residual.dtype, device=x.device)
    elif residual_dtype is not None and residual_dtype != x.dtype:
        residual_out = torch.empty(shape, dtype=residual_dtype, device=x.device)
    args = _lib.QuantArgs(
        rows, n, x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(bias), q.data_ptr(), scales.data_ptr(),
        _ptr(residual_out), row_stride, group_stride, _CODE[x.dtype], _code(residual), _code(weight), _code(bias),
        _lib._QUANT_CODES[quant_dtype], _code(residual_out), group_size or 0, eps)
    _lib.enqueue("rmsnorm_b200_quant_fwd", x.device, ctypes.byref(args))
    return q, scales, x if residual_out is None else residual_out


# ---------------------------------------------------------------------------------------
# Dropout + residual addition + RMSNorm
# ---------------------------------------------------------------------------------------
def _check_dropout(p: float, rng, step: Optional[Tensor], row_offset: int, rows: int, device) -> Tuple[int, int]:
    if not 0.0 <= p < 1.0:
        raise ValueError(f"p must be at least 0 and below 1, got {p}")
    seed, offset = rng
    if not 0 <= seed < 1 << 64 or not 0 <= offset < 1 << 64:
        raise ValueError("rng must be a (seed, offset) pair of integers in [0, 2^64)")
    if row_offset < 0 or row_offset + rows > 1 << 32:
        raise ValueError(f"row_offset must keep every row in [0, 2^32), got {row_offset} with {rows} rows")
    if step is not None and (step.dtype != torch.int64 or step.numel() != 1 or step.device != device):
        raise ValueError("rng_step must be an int64 tensor of one element on the same device as x")
    return seed, offset


def dropout_mask(shape: Sequence[int], p: float, rng: Tuple[int, int], device=None, rng_step: Optional[Tensor] = None,
                 row_offset: int = 0) -> Tensor:
    """The mask (True: kept) that `dropout_add_rmsnorm` draws for x of this shape, as a bool
    tensor; plain PyTorch, for tests and inspection."""
    shape = tuple(shape)
    _check_x_shape(torch.Size(shape))
    device = torch.device(device or "cpu")
    rows = 1
    for d in shape[:-1]:
        rows *= d
    if rng_step is not None and device.type == "cuda" and device.index is None:
        device = rng_step.device
    seed, offset = _check_dropout(p, rng, rng_step, row_offset, rows, device)
    return _host.dropout_mask(shape, p, seed, _with_step(offset, rng_step), row_offset, device)


def _with_step(offset: int, step: Optional[Tensor]) -> int:
    return offset if step is None else (offset + int(step)) % (1 << 64)


@torch.compiler.disable
def dropout_add_rmsnorm_fwd(
    x: Tensor,
    weight: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    residual: Optional[Tensor] = None,
    p: float = 0.0,
    rng: Tuple[int, int] = (0, 0),
    out_dtype: Optional[torch.dtype] = None,
    residual_dtype: Optional[torch.dtype] = None,
    eps: float = 1e-6,
    store_rstd: bool = False,
    rng_step: Optional[Tensor] = None,
    row_offset: int = 0,
) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
    """(out, residual_out, rstd): h = dropout(x) / (1 - p) + residual, out = RMSNorm(h) *
    weight + bias; residual_out is h in residual_dtype (default: residual's dtype, else x's);
    rstd (fp32, x.shape[:-1]) when store_rstd.

    The mask is a function of `rng` = (seed, offset), the row and the column alone (see
    `dropout_mask`): calls that must differ take another offset. `rng_step`, an int64 CUDA
    tensor of one element, is added to the offset when the kernel runs, so that replays of a
    CUDA graph can draw new masks. `row_offset` is the row of the whole tensor's mask that x
    begins with, for tensors whose rows are spread over ranks."""
    _check_row_input(x, weight, bias, residual)
    if out_dtype is not None:
        _check_optional_dtype("out_dtype", out_dtype)
    if residual_dtype is not None:
        _check_optional_dtype("residual_dtype", residual_dtype)
    shape = x.shape
    n = shape[-1]
    rows = x.numel() // n
    device = x.device
    seed, offset = _check_dropout(p, rng, rng_step, row_offset, rows, device)
    out_dtype = out_dtype or x.dtype
    residual_dtype = residual_dtype or (x.dtype if residual is None else residual.dtype)
    if not x.is_cuda:
        mask = _host.dropout_mask(shape, p, seed, _with_step(offset, rng_step), row_offset, device)
        return _host.dropout_add_rmsnorm_fwd(
            x, weight, bias, residual, mask, p, out_dtype, residual_dtype, eps, store_rstd)
    x = _contig(x)
    residual = _contig(residual)
    weight = _contig(weight)
    bias = _contig(bias)
    out = torch.empty(shape, dtype=out_dtype, device=device)
    residual_out = torch.empty(shape, dtype=residual_dtype, device=device)
    rstd = torch.empty(shape[:-1], dtype=torch.float32, device=device) if store_rstd else None
    args = _lib.DropoutFwdArgs(
        rows, n, x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(bias), out.data_ptr(), residual_out.data_ptr(),
        _ptr(rstd), _lib.Dropout(seed, offset, _ptr(rng_step), row_offset, p), _CODE[x.dtype], _code(residual),
        _code(weight), _code(bias), _CODE[out_dtype], _CODE[residual_dtype], eps, 0)
    _lib.enqueue("rmsnorm_b200_dropout_rmsnorm_fwd", device, ctypes.byref(args))
    return out, residual_out, rstd


@torch.compiler.disable
def dropout_add_rmsnorm_bwd(
    residual_out: Tensor,
    weight: Optional[Tensor],
    dout: Tensor,
    rstd: Tensor,
    dresidual_out: Optional[Tensor] = None,
    p: float = 0.0,
    rng: Tuple[int, int] = (0, 0),
    has_bias: bool = False,
    has_residual: bool = False,
    bias: Optional[Tensor] = None,
    dx_dtype: Optional[torch.dtype] = None,
    dresidual_dtype: Optional[torch.dtype] = None,
    rng_step: Optional[Tensor] = None,
    row_offset: int = 0,
) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """(dx, dweight, dbias, dresidual) from the forward's residual_out and rstd; p, rng,
    rng_step and row_offset as in the forward. dx is in dx_dtype (default: dout's), dresidual
    (None unless has_residual) in dresidual_dtype (default: residual_out's); dweight and dbias
    follow the affine tensors (dbias without a bias tensor: weight's dtype, else dout's)."""
    h = residual_out
    if h.dtype not in _SUPPORTED_DTYPES:
        raise AssertionError("Unsupported dtype")
    _check_x_shape(h.shape)
    shape = h.shape
    n = shape[-1]
    rows = h.numel() // n
    device = h.device
    _check_affine("weight", weight, n, device)
    _check_affine("bias", bias, n, device)
    _check_like("dout", dout, h)
    _check_like("dresidual_out", dresidual_out, h)
    if dx_dtype is not None:
        _check_optional_dtype("dx_dtype", dx_dtype)
    if dresidual_dtype is not None:
        _check_optional_dtype("dresidual_dtype", dresidual_dtype)
    if rstd.dtype != torch.float32:
        raise ValueError("rstd must be float32")
    if rstd.numel() != rows:
        raise ValueError(f"rstd must have one element per row, got {rstd.numel()} for {rows} rows")
    if rstd.device != device:
        _check_same_device("rstd", rstd, device)
    seed, offset = _check_dropout(p, rng, rng_step, row_offset, rows, device)
    dx_dtype = dx_dtype or dout.dtype
    dresidual_dtype = dresidual_dtype or h.dtype
    if not h.is_cuda:
        mask = _host.dropout_mask(shape, p, seed, _with_step(offset, rng_step), row_offset, device)
        dx, dw, db, dh = _host.dropout_add_rmsnorm_bwd(
            h, weight, dout, rstd, dresidual_out, mask, p, has_bias, bias, dx_dtype)
        return dx, dw, db, dh.to(dresidual_dtype) if has_residual else None
    h = _contig(h)
    dout = _contig(dout)
    rstd = rstd.contiguous()
    weight = _contig(weight)
    dresidual_out = _contig(dresidual_out)
    dx = torch.empty(shape, dtype=dx_dtype, device=device)
    dresidual = torch.empty(shape, dtype=dresidual_dtype, device=device) if has_residual else None
    dw = torch.empty_like(weight) if weight is not None else None
    db = None
    if has_bias:
        like = bias if bias is not None else weight
        db = torch.empty((n,), dtype=like.dtype if like is not None else dout.dtype, device=device)
    args = _lib.DropoutBwdArgs(
        rows, n, h.data_ptr(), dout.data_ptr(), rstd.data_ptr(), _ptr(weight), _ptr(dresidual_out), dx.data_ptr(),
        _ptr(dresidual), _ptr(dw), _ptr(db), _lib.Dropout(seed, offset, _ptr(rng_step), row_offset, p),
        _CODE[h.dtype], _CODE[dout.dtype], _code(weight), _code(dresidual_out), _CODE[dx_dtype],
        _CODE[dresidual_dtype], _code(dw), _code(db))
    a = ctypes.byref(args)
    nbytes = _lib.workspace_bytes("rmsnorm_b200_dropout_rmsnorm_bwd_workspace_size", device, a)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _lib.enqueue("rmsnorm_b200_dropout_rmsnorm_bwd", device, a, _ptr(ws), nbytes)
    return dx, dw, db, dresidual


class DropoutAddRMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, p, rng, out_dtype, residual_dtype, eps, prenorm, rng_step, row_offset):
        need_grad = any(ctx.needs_input_grad[:4])
        # the backward draws the mask of this call again: it keeps the step's value, not the
        # caller's tensor, which may have moved on by then
        step = rng_step.clone() if (rng_step is not None and need_grad) else rng_step
        out, residual_out, rstd = dropout_add_rmsnorm_fwd(
            x, weight, bias, residual, p, rng, out_dtype, residual_dtype, eps, need_grad, step, row_offset)
        ctx.save_for_backward(residual_out, weight, bias, rstd, step)
        ctx.p, ctx.rng, ctx.row_offset, ctx.prenorm = p, rng, row_offset, prenorm
        ctx.x_dtype = x.dtype
        ctx.residual_dtype = residual.dtype if residual is not None else None
        return (out, residual_out) if prenorm else out

    @staticmethod
    def backward(ctx, dout, dresidual_out=None):
        h, weight, bias, rstd, step = ctx.saved_tensors
        dx, dw, db, dresidual = dropout_add_rmsnorm_bwd(
            h, weight, dout, rstd, dresidual_out, ctx.p, ctx.rng, bias is not None, ctx.residual_dtype is not None,
            bias, ctx.x_dtype, ctx.residual_dtype, step, ctx.row_offset)
        return dx, dw, db, dresidual, *([None] * 8)


@torch.compiler.disable
def dropout_add_rmsnorm(
    x: Tensor,
    weight: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    residual: Optional[Tensor] = None,
    p: float = 0.0,
    rng: Tuple[int, int] = (0, 0),
    out_dtype: Optional[torch.dtype] = None,
    residual_dtype: Optional[torch.dtype] = None,
    eps: float = 1e-6,
    prenorm: bool = False,
    rng_step: Optional[Tensor] = None,
    row_offset: int = 0,
):
    """`dropout_add_rmsnorm_fwd` with autograd: out, or (out, residual_out) when prenorm."""
    return DropoutAddRMSNormFunction.apply(
        x, weight, bias, residual, p, tuple(rng), out_dtype, residual_dtype, eps, prenorm, rng_step, row_offset)


# ---------------------------------------------------------------------------------------
# Per-head RMSNorm of q and k with rotary positions
# ---------------------------------------------------------------------------------------
def rope_table(max_position: int, rotary_dim: int, base: float = 10000.0, device=None) -> Tensor:
    """fp32 [max_position, rotary_dim]: row t holds cos(t f_i) for every pair i, then
    sin(t f_i), with f_i = base^(-2 i / rotary_dim). Computed in 64 bits."""
    if max_position < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rope_table needs max_position >= 1 and an even rotary_dim >= 2, got {max_position}, {rotary_dim}")
    f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * f
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def rope_axes(sections: Sequence[int], interleaved: bool = False) -> Tuple[int, ...]:
    """The position axis of each rotary pair for `sections` pairs per axis: consecutive runs,
    or (interleaved) the axes in turn, each until its pairs are used up."""
    left = [int(s) for s in sections]
    if not 1 <= len(left) <= 4 or min(left) < 0:
        raise ValueError(f"sections must be 1 to 4 counts of pairs, got {tuple(sections)}")
    if not interleaved:
        return tuple(a for a, n in enumerate(left) for _ in range(n))
    out = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return tuple(out)


@functools.lru_cache(maxsize=64)
def _axis_words(axes: Tuple[int, ...]) -> Tuple[int, ...]:
    words = [0, 0, 0, 0]
    for i, a in enumerate(axes):
        words[i // 32] |= a << (2 * (i % 32))
    return tuple(words)


def _check_rope(q, k, positions, table, q_weight, k_weight, axes) -> Tuple[Tuple[int, ...], int]:
    """(axis of each pair, number of axes)."""
    if q.dtype not in _SUPPORTED_DTYPES:
        raise AssertionError("Unsupported dtype")
    if q.dim() < 2:
        raise ValueError("q must have at least two dimensions (heads, head_dim)")
    d = q.shape[-1]
    device = q.device
    if not 1 <= d <= 256:
        raise ValueError(f"head_dim must be 1 to 256, got {d}")
    if q.shape[-2] < 1:
        raise ValueError("q must have at least one head")
    if k is not None:
        if k.dtype != q.dtype:
            raise AssertionError("q and k must have the same dtype")
        if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != d:
            raise ValueError(f"k must have q's shape apart from the heads, got {tuple(k.shape)} for {tuple(q.shape)}")
        if k.device != device:
            raise ValueError("k must be on the same device as q")
    if table.dtype != torch.float32 or table.dim() != 2 or table.shape[1] % 2 or table.shape[1] > d:
        raise ValueError(f"table must be float32 [positions, rotary_dim] with an even rotary_dim of at most {d}")
    tokens = q.shape[:-2]
    pairs = table.shape[1] // 2
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    if positions.shape == tokens:
        naxes = 1
    elif positions.dim() == len(tokens) + 1 and positions.shape[1:] == tokens and 1 <= positions.shape[0] <= 4:
        naxes = positions.shape[0]
    else:
        raise ValueError(f"positions must be q's leading shape {tuple(tokens)}, or 1 to 4 axes of it, got "
                         f"{tuple(positions.shape)}")
    for name, t in (("positions", positions), ("table", table)):
        if t.device != device:
            raise ValueError(f"{name} must be on the same device as q")
    for name, w, heads in (("q_weight", q_weight, q.shape[-2]), ("k_weight", k_weight, k.shape[-2] if k is not None else 0)):
        if w is None:
            continue
        if name == "k_weight" and k is None:
            raise ValueError("k_weight needs k")
        _check_tensor_dtype(name, w)
        if tuple(w.shape) != (d,) and tuple(w.shape) != (heads, d):
            raise ValueError(f"{name} shape must be ({d},) or ({heads}, {d}), got {tuple(w.shape)}")
        if w.device != device:
            raise ValueError(f"{name} must be on the same device as q")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise AssertionError("q_weight and k_weight must have the same dtype")
    if axes is None:
        axes = (0,) * pairs
    axes = tuple(axes)
    if len(axes) != pairs or (axes and not 0 <= min(axes) <= max(axes) < naxes):
        raise ValueError(f"axes must name one of the {naxes} position axes for each of the {pairs} pairs")
    return axes, naxes


def _flat(t: Tensor) -> Tensor:
    """[tokens, heads, head_dim] with a contiguous last dimension; a view wherever the strides
    allow one (q and k as slices of a packed projection)."""
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        t = t.contiguous()
    return t if t.dim() == 3 else t.reshape(-1, t.shape[-2], t.shape[-1])


def _tensor(t: Optional[Tensor]) -> _lib.RopeTensor:
    if t is None:
        return _lib.RopeTensor(None, 0, 0)
    s = t.stride()
    return _lib.RopeTensor(t.data_ptr(), s[0], s[1])


def _weight_heads(w: Optional[Tensor]) -> int:
    return w.shape[0] if (w is not None and w.dim() == 2) else 1


def _rope_args(q, k, positions, table, q_weight, k_weight, axes, naxes, interleaved, norm, eps):
    words = (ctypes.c_uint64 * 4)(*_axis_words(axes))
    tokens = q.shape[0]
    w = q_weight if q_weight is not None else k_weight
    return _lib.RopeArgs(
        tokens, table.shape[0], positions.data_ptr(), tokens, table.data_ptr(), _ptr(q_weight), _ptr(k_weight),
        _tensor(q), _tensor(k), words, q.shape[1], 0 if k is None else k.shape[1], q.shape[2], table.shape[1], naxes,
        bool(interleaved), bool(norm), positions.dtype == torch.int64, _CODE[q.dtype], _code(w),
        _weight_heads(q_weight), _weight_heads(k_weight), eps, 0)


@torch.compiler.disable
def qk_norm_rope_fwd(
    q: Tensor,
    k: Optional[Tensor],
    positions: Tensor,
    table: Tensor,
    q_weight: Optional[Tensor] = None,
    k_weight: Optional[Tensor] = None,
    axes: Optional[Sequence[int]] = None,
    interleaved: bool = False,
    norm: bool = True,
    eps: float = 1e-6,
    inplace: bool = False,
) -> Tuple[Tensor, Optional[Tensor]]:
    """(q_out, k_out): every head of q (..., q_heads, head_dim) and k (..., k_heads, head_dim;
    may be None) normalised over head_dim (unless norm is False), multiplied by its weight
    ((head_dim,) or (heads, head_dim)), and its first rotary_dim columns turned by the
    token's positions. q and k may be strided views, such as slices of a packed projection;
    `inplace` writes into them, otherwise the outputs are new and contiguous.

    positions (int32 or int64) has the leading shape of q, or (axes, ...) of it; `axes` names
    the axis of each of the rotary_dim / 2 pairs (`rope_axes`; default: axis 0). Pair i is the
    columns (i, i + rotary_dim / 2), or (2 i, 2 i + 1) when `interleaved`. `table` is
    `rope_table`'s. A position outside the table gives NaN columns, and on CUDA an
    invalid-argument entry in the device status word."""
    axes, naxes = _check_rope(q, k, positions, table, q_weight, k_weight, axes)
    if not q.is_cuda:
        pos = positions.reshape(naxes, *q.shape[:-2])
        cos, sin = _host.rope_cos_sin(pos, table, axes)
        outs = [t if t is None else _host.qk_norm_rope_fwd(t, w, cos, sin, interleaved, norm, eps)
                for t, w in ((q, q_weight), (k, k_weight))]
        if inplace:
            for t, o in zip((q, k), outs):
                if t is not None:
                    t.copy_(o)
            return q, k
        return tuple(outs)
    qf = _flat(q)
    kf = None if k is None else _flat(k)
    q_out, k_out = q, k
    if inplace:
        for t, f in ((q, qf), (k, kf)):
            if t is not None and f.data_ptr() != t.data_ptr():
                raise ValueError("inplace needs q and k whose leading dimensions collapse to one stride")
        qo, ko = qf, kf
    else:
        q_out = qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if k is not None:
            k_out = ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        else:
            ko = None
        if q.dim() != 3:
            qo = qo.view(qf.shape)
            ko = None if ko is None else ko.view(kf.shape)
    positions = positions.contiguous()
    table = table.contiguous()
    q_weight = _contig(q_weight)
    k_weight = _contig(k_weight)
    args = _rope_args(qf, kf, positions, table, q_weight, k_weight, axes, naxes, interleaved, norm, eps)
    _lib.enqueue("rmsnorm_b200_rope_fwd", q.device, ctypes.byref(args), ctypes.byref(_tensor(qo)),
                 ctypes.byref(_tensor(ko)))
    return q_out, k_out


@torch.compiler.disable
def qk_norm_rope_bwd(
    q: Tensor,
    k: Optional[Tensor],
    positions: Tensor,
    table: Tensor,
    dq_out: Tensor,
    dk_out: Optional[Tensor],
    q_weight: Optional[Tensor] = None,
    k_weight: Optional[Tensor] = None,
    axes: Optional[Sequence[int]] = None,
    interleaved: bool = False,
    norm: bool = True,
    eps: float = 1e-6,
) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """(dq, dk, dq_weight, dk_weight) from the forward's inputs and the gradients of its
    outputs; the weights' gradients (None without a weight) are summed in a fixed order."""
    axes, naxes = _check_rope(q, k, positions, table, q_weight, k_weight, axes)
    for name, g, t in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        if (g is None) != (t is None):
            raise ValueError(f"{name} is needed exactly when its input is given")
        if g is not None and (g.shape != t.shape or g.dtype != q.dtype or g.device != q.device):
            raise ValueError(f"{name} must have its input's shape, dtype and device")
    if not q.is_cuda:
        pos = positions.reshape(naxes, *q.shape[:-2])
        cos, sin = _host.rope_cos_sin(pos, table, axes)
        dq, dqw = _host.qk_norm_rope_bwd(q, q_weight, dq_out, cos, sin, interleaved, norm, eps)
        dk = dkw = None
        if k is not None:
            dk, dkw = _host.qk_norm_rope_bwd(k, k_weight, dk_out, cos, sin, interleaved, norm, eps)
        return dq, dk, dqw, dkw
    device = q.device
    qf = _flat(q)
    kf = None if k is None else _flat(k)
    dq = torch.empty(q.shape, dtype=q.dtype, device=device)
    dk = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=device)
    q_weight = _contig(q_weight)
    k_weight = _contig(k_weight)
    dqw = None if q_weight is None else torch.empty_like(q_weight)
    dkw = None if k_weight is None else torch.empty_like(k_weight)
    positions = positions.contiguous()
    table = table.contiguous()
    dqo = _flat(dq_out)
    dko = None if k is None else _flat(dk_out)
    args = _rope_args(qf, kf, positions, table, q_weight, k_weight, axes, naxes, interleaved, norm, eps)
    grads = _lib.RopeGrads(_tensor(dqo), _tensor(dko), _tensor(dq.view(qf.shape)),
                           _tensor(None if k is None else dk.view(kf.shape)), _ptr(dqw), _ptr(dkw))
    a, g = ctypes.byref(args), ctypes.byref(grads)
    nbytes = _lib.workspace_bytes("rmsnorm_b200_rope_bwd_workspace_size", device, a, g)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _lib.enqueue("rmsnorm_b200_rope_bwd", device, a, g, _ptr(ws), nbytes)
    return dq, dk, dqw, dkw


class QKNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, table, q_weight, k_weight, axes, interleaved, norm, eps):
        ctx.save_for_backward(q, k, positions, table, q_weight, k_weight)
        ctx.rest = (axes, interleaved, norm, eps)
        return qk_norm_rope_fwd(q, k, positions, table, q_weight, k_weight, *ctx.rest)

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        q, k, positions, table, q_weight, k_weight = ctx.saved_tensors
        dq, dk, dqw, dkw = qk_norm_rope_bwd(q, k, positions, table, dq_out, dk_out, q_weight, k_weight, *ctx.rest)
        return dq, dk, None, None, dqw, dkw, None, None, None, None


@torch.compiler.disable
def qk_norm_rope(
    q: Tensor,
    k: Optional[Tensor],
    positions: Tensor,
    table: Tensor,
    q_weight: Optional[Tensor] = None,
    k_weight: Optional[Tensor] = None,
    axes: Optional[Sequence[int]] = None,
    interleaved: bool = False,
    norm: bool = True,
    eps: float = 1e-6,
) -> Tuple[Tensor, Optional[Tensor]]:
    """`qk_norm_rope_fwd` with autograd (for q, k and the weights)."""
    return QKNormRopeFunction.apply(
        q, k, positions, table, q_weight, k_weight, None if axes is None else tuple(axes), interleaved, norm, eps)
