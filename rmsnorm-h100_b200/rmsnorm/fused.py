# SPDX-License-Identifier: MIT
"""Operators fused with the norm, on the kernels of librmsnorm_b200:

* `rmsnorm_quant_fwd` -- residual addition + RMSNorm with an 8-bit output and scales;
* `dropout_add_rmsnorm` (`_fwd`, `_bwd`) -- dropout from a counter-based generator, residual
  addition and RMSNorm; the mask is never stored;
* `qk_norm_rope` (`_fwd`, `_bwd`) -- per-head RMSNorm of q and k with rotary positions on one
  to four axes (`rope_table`, `rope_axes`);

and, on what these leave behind:

* `block_mm` -- products of 8-bit matrices with a scale for every block of 128,
  `block_quantize`, which makes their operands, and `block_linear`, a linear layer on both with
  gradients;
* `cache_write`, `cache_read` -- keys and values in the pages of an 8-bit cache.

They follow the conventions of `rmsnorm.rmsnorm`: arguments are checked before anything
runs, CUDA tensors go to the native library on the current stream of their device, tensors
on the host are computed in plain PyTorch. Under `torch.compile` they run as graph breaks (so
`fullgraph=True` refuses them, unlike `rmsnorm`).
"""

from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _host_fused as _host
from . import _lib
from ._autograd import first_order
from ._block import BlockLinearFunction, block_linear, block_mm, block_quantize
from ._cache import cache_read, cache_write
from .rmsnorm import (
    _check_optional_dtype,
    _check_same_device,
    _check_tensor_dtype,
    _check_x_shape,
    _contig,
)

__all__ = [
    "BlockLinearFunction",
    "DropoutAddRMSNormFunction",
    "QKNormRopeFunction",
    "block_linear",
    "block_mm",
    "block_quantize",
    "cache_read",
    "cache_write",
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
_MAX_HEADS = 65536
_GROUP_SIZES = (None, 32, 64, 128, 256)
# Dynamo alone breaks its graph at the untraced functions; a non-strict export runs their code.
_is_compiling = torch.compiler.is_dynamo_compiling

# The C argument structs as packed bytes, field by field as _lib declares them (null pointers
# are 0). A decoding step calls these operators with microseconds of work, so the checks and
# the call are kept short.
_QUANT = struct.Struct("2q7Q2q7if")
_DROP_FWD = struct.Struct("2q7Q3Qqd6ifi")
_DROP_BWD = struct.Struct("2q9Q3Qqd8i")
_ROPE_TENSOR = struct.Struct("Q2q")
_ROPE = struct.Struct("2qQq3QQ2qQ2q4Q12ifi")
_ROPE_GRADS = struct.Struct("Q2qQ2qQ2qQ2q2Q")
for _s, _c in ((_QUANT, _lib.QuantArgs), (_DROP_FWD, _lib.DropoutFwdArgs), (_DROP_BWD, _lib.DropoutBwdArgs),
               (_ROPE_TENSOR, _lib.RopeTensor), (_ROPE, _lib.RopeArgs), (_ROPE_GRADS, _lib.RopeGrads)):
    assert _s.size == ctypes.sizeof(_c), _c.__name__

_BYTES, _STREAM, _SIZE, _OUT = ctypes.c_char_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)


def _affine_code(name: str, t: Optional[Tensor], n: int, device: torch.device) -> int:
    if t is None:
        return 0
    code = _CODE.get(t.dtype)
    if code is None:
        _check_tensor_dtype(name.capitalize(), t)
    if t.shape != (n,):
        raise ValueError(f"{name} shape must be (N,) with N={n}, got {tuple(t.shape)}")
    if t.device != device:
        _check_same_device(name, t, device)
    return code


def _like_code(name: str, t: Optional[Tensor], x: Tensor, shape, device: torch.device) -> int:
    if t is None:
        return 0
    code = _CODE.get(t.dtype)
    if code is None:
        _check_tensor_dtype(name.capitalize(), t)
    if t.shape != shape:
        raise ValueError(f"{name} shape must match x shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        _check_same_device(name, t, device)
    return code


def _dtype_code(name: str, dtype: torch.dtype) -> int:
    code = _CODE.get(dtype)
    if code is None:
        _check_optional_dtype(name, dtype)
    return code


def _row_codes(x: Tensor, weight, bias, residual):
    """Checks the inputs of a row operator; (shape, hidden, device, their dtype codes)."""
    code = _CODE.get(x.dtype)
    if code is None:
        raise AssertionError("Unsupported dtype")
    shape = x.shape
    if not shape or not shape[-1]:
        _check_x_shape(shape)
    n = shape[-1]
    device = x.device
    return (shape, n, device, code, _affine_code("weight", weight, n, device), _affine_code("bias", bias, n, device),
            _like_code("residual", residual, x, shape, device))


# ---------------------------------------------------------------------------------------
# Residual addition + RMSNorm with an 8-bit output
# ---------------------------------------------------------------------------------------
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

    A scale is max |y| / 448 (e4m3) or / 127 (int8), at least 2^-126; q is y / scale rounded to
    nearest even (on CUDA y times the reciprocal of the scale: within one part in 2^22 of the
    midpoint of two values either is possible). A NaN among a group's y makes its scale NaN, an
    infinite y infinite. `scales_column_major` lays grouped scales out
    column by column (the strides of a transposed tensor), as block-scaled products take
    them. residual_out as in `rmsnorm_fwd`."""
    if _is_compiling():
        return _quant_untraced(
            x, weight, bias, residual, quant_dtype, group_size, residual_dtype, eps, scales_column_major)
    shape, n, device, xc, wc, bc, rc = _row_codes(x, weight, bias, residual)
    roc = 0 if residual_dtype is None else _dtype_code("residual_dtype", residual_dtype)
    qc = _lib._QUANT_CODES.get(quant_dtype)
    if qc is None:
        raise AssertionError("quant_dtype must be float8_e4m3fn or int8")
    if group_size not in _GROUP_SIZES:
        raise ValueError(f"group_size must be None, 32, 64, 128 or 256, got {group_size}")
    rows = x.numel() // n
    row_stride, group_stride = 1, 0
    if group_size is None:
        scales = torch.empty(*shape[:-1], dtype=torch.float32, device=device) if len(shape) > 1 else torch.empty(
            (), dtype=torch.float32, device=device)
    else:
        groups = -(-n // group_size)
        if scales_column_major:
            scales = torch.empty(groups, *shape[:-1], dtype=torch.float32, device=device).movedim(0, -1)
            row_stride, group_stride = 1, rows
        else:
            scales = torch.empty(*shape[:-1], groups, dtype=torch.float32, device=device)
            row_stride, group_stride = groups, 1
    if not x.is_cuda:
        q, residual_out = _host.rmsnorm_quant_fwd(
            x, weight, bias, residual, quant_dtype, group_size, residual_dtype, eps, scales)
        return q, scales, residual_out
    x = _contig(x)
    residual = _contig(residual)
    weight = _contig(weight)
    bias = _contig(bias)
    q = torch.empty_like(x, dtype=quant_dtype)
    residual_out = None
    if residual is not None:
        if residual_dtype is None:
            residual_out, roc = torch.empty_like(residual), rc
        else:
            residual_out = torch.empty_like(x, dtype=residual_dtype)
    elif residual_dtype is not None and residual_dtype != x.dtype:
        residual_out = torch.empty_like(x, dtype=residual_dtype)
    args = _QUANT.pack(
        rows, n, x.data_ptr(), 0 if residual is None else residual.data_ptr(),
        0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(), q.data_ptr(),
        scales.data_ptr(), 0 if residual_out is None else residual_out.data_ptr(), row_stride, group_stride, xc, rc, wc,
        bc, qc, roc, group_size or 0, eps)
    name = "rmsnorm_b200_quant_fwd"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _STREAM), name, device.index, args)
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
    if _is_compiling():
        return _drop_fwd_untraced(
            x, weight, bias, residual, p, rng, out_dtype, residual_dtype, eps, store_rstd, rng_step, row_offset)
    shape, n, device, xc, wc, bc, rc = _row_codes(x, weight, bias, residual)
    if out_dtype is None:
        out_dtype, oc = x.dtype, xc
    else:
        oc = _dtype_code("out_dtype", out_dtype)
    if residual_dtype is None:
        residual_dtype, roc = (x.dtype, xc) if residual is None else (residual.dtype, rc)
    else:
        roc = _dtype_code("residual_dtype", residual_dtype)
    rows = x.numel() // n
    seed, offset = _check_dropout(p, rng, rng_step, row_offset, rows, device)
    if not x.is_cuda:
        mask = _host.dropout_mask(shape, p, seed, _with_step(offset, rng_step), row_offset, device)
        return _host.dropout_add_rmsnorm_fwd(
            x, weight, bias, residual, mask, p, out_dtype, residual_dtype, eps, store_rstd)
    x = _contig(x)
    residual = _contig(residual)
    weight = _contig(weight)
    bias = _contig(bias)
    out = torch.empty_like(x, dtype=out_dtype)
    residual_out = torch.empty_like(x, dtype=residual_dtype)
    rstd = torch.empty(shape[:-1], dtype=torch.float32, device=device) if store_rstd else None
    args = _DROP_FWD.pack(
        rows, n, x.data_ptr(), 0 if residual is None else residual.data_ptr(),
        0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(), out.data_ptr(),
        residual_out.data_ptr(), 0 if rstd is None else rstd.data_ptr(), seed, offset,
        0 if rng_step is None else rng_step.data_ptr(), row_offset, p, xc, rc, wc, bc, oc, roc, eps, 0)
    name = "rmsnorm_b200_dropout_rmsnorm_fwd"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _STREAM), name, device.index, args)
    return out, residual_out, rstd


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
    if _is_compiling():
        return _drop_bwd_untraced(
            residual_out, weight, dout, rstd, dresidual_out, p, rng, has_bias, has_residual, bias, dx_dtype,
            dresidual_dtype, rng_step, row_offset)
    h = residual_out
    shape, n, device, hc, wc, bc, _ = _row_codes(h, weight, bias, None)
    yc = _like_code("dout", dout, h, shape, device)
    doc = _like_code("dresidual_out", dresidual_out, h, shape, device)
    if dx_dtype is None:
        dx_dtype, dxc = dout.dtype, yc
    else:
        dxc = _dtype_code("dx_dtype", dx_dtype)
    if dresidual_dtype is None:
        dresidual_dtype, dresc = h.dtype, hc
    else:
        dresc = _dtype_code("dresidual_dtype", dresidual_dtype)
    rows = h.numel() // n
    if rstd.dtype != torch.float32:
        raise ValueError("rstd must be float32")
    if rstd.numel() != rows:
        raise ValueError(f"rstd must have one element per row, got {rstd.numel()} for {rows} rows")
    if rstd.device != device:
        _check_same_device("rstd", rstd, device)
    seed, offset = _check_dropout(p, rng, rng_step, row_offset, rows, device)
    if not h.is_cuda:
        mask = _host.dropout_mask(shape, p, seed, _with_step(offset, rng_step), row_offset, device)
        dx, dw, db, dh = _host.dropout_add_rmsnorm_bwd(
            h, weight, dout, rstd, dresidual_out, mask, p, has_bias, bias, dx_dtype)
        return dx, dw, db, dh.to(dresidual_dtype) if has_residual else None
    h = _contig(h)
    dout = _contig(dout)
    rstd = _contig(rstd)
    weight = _contig(weight)
    dresidual_out = _contig(dresidual_out)
    dx = torch.empty_like(h, dtype=dx_dtype)
    dresidual = torch.empty_like(h, dtype=dresidual_dtype) if has_residual else None
    dw = torch.empty_like(weight) if weight is not None else None
    db = None
    if has_bias:
        if bias is None:
            db = torch.empty(n, dtype=dout.dtype, device=device) if weight is None else torch.empty_like(weight)
            bc = yc if weight is None else wc
        else:
            db = torch.empty_like(bias, memory_format=torch.contiguous_format)
    args = _DROP_BWD.pack(
        rows, n, h.data_ptr(), dout.data_ptr(), rstd.data_ptr(), 0 if weight is None else weight.data_ptr(),
        0 if dresidual_out is None else dresidual_out.data_ptr(), dx.data_ptr(),
        0 if dresidual is None else dresidual.data_ptr(), 0 if dw is None else dw.data_ptr(),
        0 if db is None else db.data_ptr(), seed, offset, 0 if rng_step is None else rng_step.data_ptr(), row_offset, p,
        hc, yc, wc, doc, dxc, dresc, wc, bc)
    nbytes = 0
    if dw is not None or db is not None:
        name = "rmsnorm_b200_dropout_rmsnorm_bwd_workspace_size"
        nbytes = _lib.workspace_bytes(_lib.packed_entry(name, _BYTES, _OUT), name, device.index, args)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    name = "rmsnorm_b200_dropout_rmsnorm_bwd"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _STREAM, _SIZE, _STREAM), name, device.index, args,
                 None if ws is None else ws.data_ptr(), nbytes)
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
        # on the host too: what the forward saved of its sum and rstd has no graph
        return *first_order("dropout_add_rmsnorm", (dx, dw, db, dresidual)), *([None] * 8)


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
    """`dropout_add_rmsnorm_fwd` with autograd: out, or (out, residual_out) when prenorm. Its
    gradients cannot be differentiated again: that is an error."""
    if _is_compiling():
        return _drop_untraced(
            x, weight, bias, residual, p, rng, out_dtype, residual_dtype, eps, prenorm, rng_step, row_offset)
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


@functools.lru_cache(maxsize=256)
def _axis_words(axes: Optional[Tuple[int, ...]], pairs: int, naxes: int):
    """(axes, two bits per pair in four words), checked."""
    if axes is None:
        axes = (0,) * pairs
    if len(axes) != pairs or (axes and not 0 <= min(axes) <= max(axes) < naxes):
        raise ValueError(f"axes must name one of the {naxes} position axes for each of the {pairs} pairs")
    words = [0, 0, 0, 0]
    for i, a in enumerate(axes):
        words[i // 32] |= a << (2 * (i % 32))
    return axes, tuple(words)


def _rope_weight_code(name: str, w: Optional[Tensor], heads: int, d: int, device: torch.device) -> Tuple[int, int]:
    """(dtype code, heads) of a weight."""
    if w is None:
        return 0, 1
    code = _CODE.get(w.dtype)
    if code is None:
        _check_tensor_dtype(name, w)
    shape = w.shape
    if shape != (d,) and (heads < 1 or shape != (heads, d)):
        raise ValueError(f"{name} shape must be ({d},) or ({heads}, {d}), got {tuple(shape)}")
    if w.device != device:
        raise ValueError(f"{name} must be on the same device as q")
    return code, 1 if len(shape) == 1 else heads


def _check_rope(q, k, positions, table, q_weight, k_weight, axes):
    """(axis of each pair, packed axes, number of axes, device, dtype code, weights' dtype
    code, q's and k's weight heads)."""
    dt = q.dtype
    code = _CODE.get(dt)
    if code is None:
        raise AssertionError("Unsupported dtype")
    shape = q.shape
    if len(shape) < 2:
        raise ValueError("q must have at least two dimensions (heads, head_dim)")
    d = shape[-1]
    device = q.device
    if not 1 <= d <= 256:
        raise ValueError(f"head_dim must be 1 to 256, got {d}")
    if not 1 <= shape[-2] <= _MAX_HEADS:
        raise ValueError(f"q must have at least one head and at most {_MAX_HEADS}, got {shape[-2]}")
    tokens = shape[:-2]
    k_heads = 0
    if k is not None:
        if k.dtype != dt:
            raise AssertionError("q and k must have the same dtype")
        kshape = k.shape
        if len(kshape) != len(shape) or kshape[:-2] != tokens or kshape[-1] != d:
            raise ValueError(f"k must have q's shape apart from the heads, got {tuple(kshape)} for {tuple(shape)}")
        if k.device != device:
            raise ValueError("k must be on the same device as q")
        k_heads = kshape[-2]
        if k_heads > _MAX_HEADS:
            raise ValueError(f"k must have at most {_MAX_HEADS} heads, got {k_heads}")
    elif k_weight is not None:
        raise ValueError("k_weight needs k")
    tshape = table.shape
    if table.dtype != torch.float32 or len(tshape) != 2 or tshape[1] % 2 or tshape[1] > d:
        raise ValueError(f"table must be float32 [positions, rotary_dim] with an even rotary_dim of at most {d}")
    if positions.dtype != torch.int64 and positions.dtype != torch.int32:
        raise ValueError("positions must be int32 or int64")
    pshape = positions.shape
    if pshape == tokens:
        naxes = 1
    elif len(pshape) == len(tokens) + 1 and pshape[1:] == tokens and 1 <= pshape[0] <= 4:
        naxes = pshape[0]
    else:
        raise ValueError(f"positions must be q's leading shape {tuple(tokens)}, or 1 to 4 axes of it, got "
                         f"{tuple(pshape)}")
    if positions.device != device:
        raise ValueError("positions must be on the same device as q")
    if table.device != device:
        raise ValueError("table must be on the same device as q")
    qwc, qwh = _rope_weight_code("q_weight", q_weight, shape[-2], d, device)
    kwc, kwh = _rope_weight_code("k_weight", k_weight, k_heads, d, device)
    if q_weight is not None and k_weight is not None and qwc != kwc:
        raise AssertionError("q_weight and k_weight must have the same dtype")
    axes, words = _axis_words(None if axes is None else tuple(axes), tshape[1] // 2, naxes)
    return axes, words, naxes, device, code, kwc if q_weight is None else qwc, qwh, kwh


_NOWHERE = (0, 0, 0)


def _place(t: Optional[Tensor]) -> Tuple[Optional[Tensor], Tuple[int, int, int]]:
    """t as [tokens, heads, head_dim] with a contiguous last dimension, a view wherever the
    strides allow one (q and k as slices of a packed projection); its address, token stride
    and head stride."""
    if t is None:
        return None, _NOWHERE
    stride = t.stride()
    if stride[-1] != 1 and t.shape[-1] > 1:
        t = t.contiguous()
        stride = t.stride()
    if len(stride) != 3:
        t = t.reshape(t.shape[:-2].numel(), t.shape[-2], t.shape[-1])  # no -1: k may have no heads
        stride = t.stride()
    return t, (t.data_ptr(), stride[0], stride[1])


def _repeats(t: Tensor) -> bool:
    """Whether t is an expanded view: a dimension that stays at one place."""
    stride = t.stride()
    return 0 in stride and any(s == 0 and n > 1 for s, n in zip(stride, t.shape))


def _new_like(t: Optional[Tensor]) -> Tuple[Optional[Tensor], Tuple[int, int, int]]:
    """A contiguous tensor of t's shape, and its place as _place gives it."""
    if t is None:
        return None, _NOWHERE
    new = torch.empty_like(t, memory_format=torch.contiguous_format)
    d = t.shape[-1]
    return new, (new.data_ptr(), t.shape[-2] * d, d)


def _rope_args(q, q_place, k, k_place, positions, table, q_weight, k_weight, checked, interleaved, norm, eps) -> bytes:
    _, words, naxes, _, code, wc, qwh, kwh = checked
    tokens, heads, d = q.shape
    return _ROPE.pack(
        tokens, table.shape[0], positions.data_ptr(), tokens, table.data_ptr(),
        0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(), *q_place,
        *k_place, *words, heads, 0 if k is None else k.shape[1], d, table.shape[1], naxes, bool(interleaved),
        bool(norm), positions.dtype == torch.int64, code, wc, qwh, kwh, eps, 0)


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
    `inplace` writes into them, otherwise the outputs are new and contiguous. On CUDA `inplace`
    is outside autograd: it refuses q and k that require gradients while those are recorded.

    positions (int32 or int64) has the leading shape of q, or (axes, ...) of it; `axes` names
    the axis of each of the rotary_dim / 2 pairs (`rope_axes`; default: axis 0). Pair i is the
    columns (i, i + rotary_dim / 2), or (2 i, 2 i + 1) when `interleaved`. `table` is
    `rope_table`'s. A position outside the table makes its token's turned columns NaN, and on
    CUDA the device status tells of an invalid argument; nothing else changes."""
    if _is_compiling():
        return _rope_fwd_untraced(
            q, k, positions, table, q_weight, k_weight, axes, interleaved, norm, eps, inplace)
    checked = _check_rope(q, k, positions, table, q_weight, k_weight, axes)
    if inplace and (_repeats(q) or k is not None and _repeats(k)):
        raise ValueError("inplace needs q and k whose elements have places of their own, not expanded views")
    if not q.is_cuda:
        cos, sin = _host.rope_cos_sin(positions.reshape(checked[2], *q.shape[:-2]), table, checked[0])
        outs = [t if t is None else _host.qk_norm_rope_fwd(t, w, cos, sin, interleaved, norm, eps)
                for t, w in ((q, q_weight), (k, k_weight))]
        if inplace:
            for t, o in zip((q, k), outs):
                if t is not None:
                    t.copy_(o)
            return q, k
        return tuple(outs)
    qf, q_place = _place(q)
    kf, k_place = _place(k)
    if inplace:
        for t, place in ((q, q_place), (k, k_place)):
            if t is None:
                continue
            if place[0] != t.data_ptr():
                raise ValueError("inplace needs q and k whose leading dimensions collapse to one stride")
            if t.requires_grad and torch.is_grad_enabled():
                raise ValueError("inplace on CUDA is outside autograd: q and k must not require gradients "
                                 "(qk_norm_rope has them; torch.no_grad() leaves them out)")
        q_out, k_out, qo_place, ko_place = q, k, q_place, k_place
    else:
        q_out, qo_place = _new_like(q)
        k_out, ko_place = _new_like(k)
    positions = positions.contiguous()
    table = table.contiguous()
    q_weight = _contig(q_weight)
    k_weight = _contig(k_weight)
    args = _rope_args(qf, q_place, kf, k_place, positions, table, q_weight, k_weight, checked, interleaved, norm, eps)
    name = "rmsnorm_b200_rope_fwd"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _BYTES, _BYTES, _STREAM), name, checked[3].index, args,
                 _ROPE_TENSOR.pack(*qo_place), _ROPE_TENSOR.pack(*ko_place))
    if inplace:  # as torch's own in-place operations: what autograd saved of q and k is no longer valid
        torch.autograd.graph.increment_version(q if k is None else (q, k))
    return q_out, k_out


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
    if _is_compiling():
        return _rope_bwd_untraced(
            q, k, positions, table, dq_out, dk_out, q_weight, k_weight, axes, interleaved, norm, eps)
    checked = _check_rope(q, k, positions, table, q_weight, k_weight, axes)
    for name, g, t in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        if (g is None) != (t is None):
            raise ValueError(f"{name} is needed exactly when its input is given")
        if g is not None and (g.shape != t.shape or g.dtype != q.dtype or g.device != q.device):
            raise ValueError(f"{name} must have its input's shape, dtype and device")
    if not q.is_cuda:
        cos, sin = _host.rope_cos_sin(positions.reshape(checked[2], *q.shape[:-2]), table, checked[0])
        dq, dqw = _host.qk_norm_rope_bwd(q, q_weight, dq_out, cos, sin, interleaved, norm, eps)
        dk = dkw = None
        if k is not None:
            dk, dkw = _host.qk_norm_rope_bwd(k, k_weight, dk_out, cos, sin, interleaved, norm, eps)
        return dq, dk, dqw, dkw
    device = checked[3]
    qf, q_place = _place(q)
    kf, k_place = _place(k)
    dqo, dqo_place = _place(dq_out)  # named, so that copies live until the launch
    dko, dko_place = _place(dk_out)
    dq, dq_place = _new_like(q)
    dk, dk_place = _new_like(k)
    q_weight = _contig(q_weight)
    k_weight = _contig(k_weight)
    dqw = None if q_weight is None else torch.empty_like(q_weight)
    dkw = None if k_weight is None else torch.empty_like(k_weight)
    positions = positions.contiguous()
    table = table.contiguous()
    args = _rope_args(qf, q_place, kf, k_place, positions, table, q_weight, k_weight, checked, interleaved, norm, eps)
    grads = _ROPE_GRADS.pack(
        *dqo_place, *dko_place, *dq_place, *dk_place, 0 if dqw is None else dqw.data_ptr(),
        0 if dkw is None else dkw.data_ptr())
    nbytes = 0
    if dqw is not None or dkw is not None:
        name = "rmsnorm_b200_rope_bwd_workspace_size"
        nbytes = _lib.workspace_bytes(_lib.packed_entry(name, _BYTES, _BYTES, _OUT), name, device.index, args, grads)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    name = "rmsnorm_b200_rope_bwd"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _BYTES, _STREAM, _SIZE, _STREAM), name, device.index, args, grads,
                 None if ws is None else ws.data_ptr(), nbytes)
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
        if q.is_cuda:  # the host's are plain PyTorch
            dq, dk, dqw, dkw = first_order("qk_norm_rope", (dq, dk, dqw, dkw))
        return dq, dk, None, None, dqw, dkw, None, None, None, None


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
    """`qk_norm_rope_fwd` with autograd (for q, k and the weights). On CUDA its gradients cannot
    be differentiated again: that is an error."""
    if _is_compiling():
        return _rope_untraced(
            q, k, positions, table, q_weight, k_weight, axes, interleaved, norm, eps)
    return QKNormRopeFunction.apply(
        q, k, positions, table, q_weight, k_weight, None if axes is None else tuple(axes), interleaved, norm, eps)


# The same functions as torch.compile calls them: untraced, a graph break each.
_quant_untraced = torch.compiler.disable(rmsnorm_quant_fwd)
_drop_fwd_untraced = torch.compiler.disable(dropout_add_rmsnorm_fwd)
_drop_bwd_untraced = torch.compiler.disable(dropout_add_rmsnorm_bwd)
_drop_untraced = torch.compiler.disable(dropout_add_rmsnorm)
_rope_fwd_untraced = torch.compiler.disable(qk_norm_rope_fwd)
_rope_bwd_untraced = torch.compiler.disable(qk_norm_rope_bwd)
_rope_untraced = torch.compiler.disable(qk_norm_rope)
