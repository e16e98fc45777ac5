# SPDX-License-Identifier: MIT
"""8-bit products with a scale for every block of 128 (`rmsnorm.fused` offers them)."""

from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _host_fused as _host
from . import _lib
from ._autograd import first_order
from .rmsnorm import _check_optional_dtype, _check_same_device, _check_tensor_dtype, _check_x_shape

_CODE = _lib._DTYPE_CODES
_BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_is_compiling = torch.compiler.is_dynamo_compiling

_QUANT = struct.Struct("2qQqQqQ2qQq2Q4i")
_MM = struct.Struct("3qQqQqQ2qQ2q2Q4i")
for _s, _c in ((_QUANT, _lib.BlockQuantArgs), (_MM, _lib.BlockMmArgs)):
    assert _s.size == ctypes.sizeof(_c), _c.__name__

_BYTES, _STREAM, _SIZE, _OUT = ctypes.c_char_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)


def _rows_of(t: Tensor) -> Tensor:
    """t as a matrix over its last dimension, whose values lie side by side: a view wherever
    the strides allow one."""
    if t.dim() != 2:
        t = t.reshape(t.shape[:-1].numel(), t.shape[-1])
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t


def _bytes_empty(shape, device) -> Tensor:
    """e4m3 values whose rows begin at multiples of 16 bytes, as the product reads them."""
    k = shape[-1]
    pitch = -(-k // 16) * 16
    if pitch == k:
        return torch.empty(shape, dtype=_E4M3, device=device)
    return torch.empty(*shape[:-1], pitch, dtype=_E4M3, device=device)[..., :k]


def _quantize(x: Tensor, rows: int, want: bool, want_t: bool, sums_dtype=None):
    """On the host, (q, scales, q_t, scales_t, column sums) of a matrix, those that are wanted."""
    none = (None, None)
    sums = None if sums_dtype is None else x.float().sum(0).to(sums_dtype)
    return (*(_host.block_quantize(x, rows) if want else none), *(_host.block_quantize(x.t(), rows) if want_t else none), sums)


def _quantize_cuda(x: Tensor, rows: int, want_t: bool, column_major: bool):
    """(q, scales, q_t, scales_t) of a matrix, the last two where they are wanted."""
    n, k = x.shape
    device = x.device
    gn, gk = -(-n // rows), -(-k // _BLOCK)
    q, q_t, scales_t = _bytes_empty((n, k), device), None, None
    if column_major:
        scales = torch.empty(gk, gn, dtype=torch.float32, device=device).t()
        sr, sg = 1, gn
    else:
        scales = torch.empty(gn, gk, dtype=torch.float32, device=device)
        sr, sg = gk, 1
    if want_t:
        q_t = _bytes_empty((k, n), device)
        scales_t = torch.empty(-(-n // _BLOCK), gk if rows > 1 else k, dtype=torch.float32, device=device).t()
    _enqueue_quantize(x, rows, q.data_ptr(), scales.data_ptr(), sr, sg, q_t.data_ptr() if want_t else 0,
                      scales_t.data_ptr() if want_t else 0, None)
    return q, scales, q_t, scales_t


def _enqueue_quantize(x: Tensor, rows: int, q: int, scales: int, sr: int, sg: int, q_t: int, scales_t: int, sums) -> None:
    """Into what lies at these addresses (0: is not wanted), rows at multiples of 16 bytes."""
    n, k = x.shape
    device = x.device
    args = _QUANT.pack(
        n, k, x.data_ptr(), x.stride(0), q, -(-k // 16) * 16, scales, sr, sg, q_t, -(-n // 16) * 16, scales_t,
        0 if sums is None else sums.data_ptr(), _CODE[x.dtype], rows, 0 if sums is None else _CODE[sums.dtype], 0)
    nbytes, ws = 0, None
    if sums is not None:
        name = "rmsnorm_b200_block_quant_workspace_size"
        nbytes = _lib.workspace_bytes(_lib.packed_entry(name, _BYTES, _OUT), name, device.index, args)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    name = "rmsnorm_b200_block_quant"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _STREAM, _SIZE, _STREAM), name, device.index, args,
                 None if ws is None else ws.data_ptr(), nbytes)


def block_quantize(x: Tensor, block_rows: int = 1, transposed: bool = False, scales_column_major: bool = False):
    """(q, scales): x (..., K) held as q * scales, q in float8_e4m3fn and fp32 scales, one for
    every 128 columns of a row (block_rows 1, scales x.shape[:-1] + (ceil(K / 128),)) or, of a
    matrix, for every 128 x 128 block (block_rows 128, scales (ceil(N / 128), ceil(K / 128)));
    the last ones may be shorter. With `transposed` (q, scales, q_t, scales_t): from the same
    read also those of x transposed, the matrix (K, rows of x).

    A scale is the smallest power of two that brings the largest |x| to 448 or below, at least
    2^-126; q is x / scale, which is exact, rounded to nearest even. A NaN makes its scale NaN,
    an infinity infinite. `scales_column_major` lays q's scales out column by column, as scales_t
    are: large products read them faster so. The rows of q and q_t begin at multiples of 16 bytes:
    where their length is none, they are views of wider rows. Outside autograd."""
    if _is_compiling():
        return _quantize_untraced(x, block_rows, transposed, scales_column_major)
    if x.dtype not in _CODE:
        raise AssertionError("Unsupported dtype")
    if not x.shape or not x.shape[-1]:
        _check_x_shape(x.shape)
    if block_rows not in (1, _BLOCK):
        raise ValueError(f"block_rows must be 1 or 128, got {block_rows}")
    if block_rows > 1 and x.dim() != 2:
        raise ValueError(f"128 x 128 blocks need a matrix, got shape {tuple(x.shape)}")
    if x.requires_grad:
        x = x.detach()
    if x.is_cuda:
        q, scales, q_t, scales_t = _quantize_cuda(_rows_of(x), block_rows, transposed, scales_column_major)
    else:
        q, scales, q_t, scales_t, _ = _quantize(_rows_of(x), block_rows, True, transposed)
        if scales_column_major:
            scales = scales.t().contiguous().t()
    if x.dim() != 2:
        lead = x.shape[:-1]
        q = q.view(*lead, x.shape[-1]) if q.is_contiguous() else q.unflatten(0, lead) if lead else q[0]
        scales = scales.unflatten(0, lead) if lead else scales[0]
    return (q, scales, q_t, scales_t) if transposed else (q, scales)


def _check_bias(bias: Optional[Tensor], n: int, device: torch.device) -> int:
    """Its dtype code."""
    if bias is None:
        return 0
    code = _CODE.get(bias.dtype)
    if code is None:
        _check_tensor_dtype("Bias", bias)
    if bias.shape != (n,):
        raise ValueError(f"bias shape must be (N,) with N={n}, got {tuple(bias.shape)}")
    if bias.device != device:
        _check_same_device("bias", bias, device)
    return code


def block_mm(a: Tensor, a_scales: Tensor, b: Tensor, b_scales: Tensor, bias: Optional[Tensor] = None,
             out_dtype: torch.dtype = torch.bfloat16, power_of_two: bool = False) -> Tensor:
    """The product of 8-bit matrices with scales, (a * a_scales) (b * b_scales)^T + bias, in
    out_dtype: a (..., K) and b (N, K) in float8_e4m3fn, fp32 scales for groups of 128 columns,
    a_scales a.shape[:-1] + (ceil(K / 128),) as `rmsnorm_quant_fwd` with group_size 128 and
    `block_quantize` leave them, b_scales (N, ceil(K / 128)) or, a scale per 128 x 128 block,
    (ceil(N / 128), ceil(K / 128)). Scales may have any strides. The sums are held in fp32,
    rounded once at the end; on CUDA so is the product of a's and b's scale for a group, which has
    to be a normal number there.

    `power_of_two` tells that every scale is a power of two, as `block_quantize` makes them: large
    products with 16-bit results then leave the scales to the tensor cores, which is a fifth to a
    half faster. They add all of K themselves then, in fp32 but not rounded to nearest: a sum may lose
    up to 2^-23 of its magnitudes with each of K / 32 additions (in registers the groups' sums are
    added rounded to nearest). Of scales that are none only the exponent may be used; an infinite one
    counts as NaN.

    Operands whose rows begin at multiples of 16 bytes are read as they are, others copied by
    every call. Outside autograd: `block_linear` has gradients."""
    if _is_compiling():
        return _mm_untraced(a, a_scales, b, b_scales, bias, out_dtype, power_of_two)
    if a.dtype != _E4M3 or b.dtype != _E4M3:
        raise AssertionError("a and b must be float8_e4m3fn")
    if a_scales.dtype != torch.float32 or b_scales.dtype != torch.float32:
        raise AssertionError("scales must be float32")
    oc = _CODE.get(out_dtype)
    if oc is None:
        _check_optional_dtype("out_dtype", out_dtype)
    shape, b_shape = a.shape, b.shape
    if not shape or not shape[-1]:
        _check_x_shape(shape)
    k, device = shape[-1], a.device
    if len(b_shape) != 2 or b_shape[1] != k or not b_shape[0]:
        raise ValueError(f"b must be (N, K) with K={k} and at least one row, got {tuple(b_shape)}")
    n, groups = b_shape[0], -(-k // _BLOCK)
    matrix = len(shape) == 2
    s_shape = a_scales.shape
    if len(s_shape) != len(shape) or s_shape[-1] != groups or s_shape[:-1] != shape[:-1]:
        raise ValueError(f"a_scales must be {tuple(shape[:-1] + (groups,))}, got {tuple(s_shape)}")
    bs_rows = b_scales.shape[0] if b_scales.dim() == 2 and b_scales.shape[1] == groups else -1
    if bs_rows == -(-n // _BLOCK):
        b_rows = _BLOCK
    elif bs_rows == n:
        b_rows = 1
    else:
        raise ValueError(f"b_scales must be {(n, groups)} or {(-(-n // _BLOCK), groups)}, got {tuple(b_scales.shape)}")
    if a_scales.device != device or b.device != device or b_scales.device != device:
        for name, t in (("a_scales", a_scales), ("b", b), ("b_scales", b_scales)):
            _check_same_device(name, t, device)
    bias_code = 0
    if bias is not None:
        bias_code = _check_bias(bias, n, device)
        bias = bias.contiguous()
    if not matrix:
        a = a.reshape(shape[:-1].numel(), k)
        a_scales = a_scales.reshape(a.shape[0], groups)
    if not a.is_cuda:
        out = _host_product(a, a_scales, b, b_scales, b_rows, bias, out_dtype)
        return out if matrix else out.view(*shape[:-1], n)
    a_row, a_step = a.stride()
    if a_step != 1 and k > 1 or a_row < k:  # a column by column, or rows that overlap
        a = a.contiguous()
        a_row = k
    b_row, b_step = b.stride()
    if b_step != 1 and k > 1 or b_row < k:
        b = b.contiguous()
        b_row = k
    out = _product(a, a_row, a_scales, b, b_row, b_scales, b_rows, bias, bias_code, out_dtype, oc, bool(power_of_two))
    return out if matrix else out.view(*shape[:-1], n)


def _host_product(a, a_scales, b, b_scales, b_rows, bias, out_dtype) -> Tensor:
    with torch.no_grad(), torch.autocast("cpu", enabled=False):  # the sums are fp32 in any mode
        out = _host.block_values(a, a_scales, 1) @ _host.block_values(b, b_scales, b_rows).t()
        return (out if bias is None else out + bias.float()).to(out_dtype)


def _product(a, a_row, a_scales, b, b_row, b_scales, b_rows, bias, bias_code, out_dtype, oc, power_of_two) -> Tensor:
    """The product of checked matrices on CUDA with rows a_row and b_row apart."""
    m, k = a.shape
    n, device = b.shape[0], a.device
    out = torch.empty(m, n, dtype=out_dtype, device=device)
    a_ptr, b_ptr = a.data_ptr(), b.data_ptr()
    args = _MM.pack(
        m, n, k, a_ptr, a_row, b_ptr, b_row, a_scales.data_ptr(), *a_scales.stride(), b_scales.data_ptr(),
        *b_scales.stride(), 0 if bias is None else bias.data_ptr(), out.data_ptr(), b_rows, bias_code, oc, power_of_two)
    nbytes, ws = 0, None
    if (a_ptr | b_ptr | a_row | b_row) & 15:
        name = "rmsnorm_b200_block_mm_workspace_size"
        nbytes = _lib.workspace_bytes(_lib.packed_entry(name, _BYTES, _OUT), name, device.index, args)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    name = "rmsnorm_b200_block_mm"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _STREAM, _SIZE, _STREAM), name, device.index, args,
                 None if ws is None else ws.data_ptr(), nbytes)
    return out


class BlockLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad):
        x2 = _rows_of(x)
        need = ctx.needs_input_grad if grad else (False, False)  # they are what the inputs want, whatever the mode
        ctx.x_shape, ctx.dtypes = x.shape, (x.dtype, weight.dtype, None if bias is None else bias.dtype)
        if x.is_cuda:
            code = 0
            if bias is not None:
                bias, code = bias.contiguous(), _CODE[bias.dtype]
            y, kept = _linear_forward(x2, _rows_of(weight), bias, code, need[0], need[1])
        else:
            q, s, x_t, x_ts, _ = _quantize(x2, 1, True, need[1])
            w, ws, w_t, w_ts, _ = _quantize(_rows_of(weight), _BLOCK, True, need[0])
            kept = x_t, x_ts, w_t, w_ts
            y = _host_product(q, s, w, ws, _BLOCK, bias, x.dtype)
        ctx.save_for_backward(*kept)
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        x_dtype, w_dtype, b_dtype = ctx.dtypes
        if not need_b:
            b_dtype = None
        if dy.is_cuda:
            dx, dw, db = _linear_backward(_rows_of(dy), *ctx.saved_tensors, ctx.x_shape[-1], x_dtype if need_x else None,
                                          w_dtype if need_w else None, b_dtype)
        else:
            x_t, x_ts, w_t, w_ts = ctx.saved_tensors
            dx = dw = None
            q, s, d_t, d_ts, db = _quantize(_rows_of(dy), 1, need_x, need_w, b_dtype)
            if need_x:
                dx = _host_product(q, s, w_t, w_ts, _BLOCK, None, x_dtype)
            if need_w:
                dw = _host_product(d_t, d_ts, x_t, x_ts, 1, None, w_dtype)
        if need_x:
            dx = dx.view(ctx.x_shape)
        return (*first_order("block_linear", (dx, dw, db)), None)


# On CUDA a matrix and its scales share a buffer of bytes, values first: a training step of few tokens
# is the host's time, of which 17 allocations and the views of odd widths took a quarter: 333 tokens,
# 1001 to 520 with bias, 159 us a step with 10 allocations, 210 with a tensor for each.
def _room(rows: int, k: int, scales: int, device: torch.device) -> Tuple[Tensor, int, int]:
    """A buffer for `rows` x k values and so many scales; the addresses of both."""
    size = rows * (-(-k // 16) * 16)
    buf = torch.empty(size + 4 * scales, dtype=torch.uint8, device=device)
    at = buf.data_ptr()
    return buf, at, at + size


def _enqueue_product(m, n, k, a, a_scales, sa_row, sa_group, b, b_scales, sb_row, sb_group, b_rows, bias, bias_code,
                     out) -> None:
    """Of what lies at these addresses, rows at multiples of 16 bytes, with powers of two as scales."""
    pitch = -(-k // 16) * 16
    args = _MM.pack(m, n, k, a, pitch, b, pitch, a_scales, sa_row, sa_group, b_scales, sb_row, sb_group,
                    0 if bias is None else bias.data_ptr(), out.data_ptr(), b_rows, bias_code, _CODE[out.dtype], 1)
    name = "rmsnorm_b200_block_mm"
    _lib.enqueue(_lib.packed_entry(name, _BYTES, _STREAM, _SIZE, _STREAM), name, out.device.index, args, None, 0)


def _linear_forward(x: Tensor, weight: Tensor, bias, bias_code: int, keep_w: bool, keep_x: bool):
    """(y, (x transposed, weight transposed)) of matrices, those that are kept."""
    (m, k), n, device = x.shape, weight.shape[0], x.device
    gm, gn, gk = -(-m // _BLOCK), -(-n // _BLOCK), -(-k // _BLOCK)
    x_buf, q, s = _room(m, k, m * gk, device)
    w_buf, w, ws = _room(n, k, gn * gk, device)
    x_t, x_q, x_s = _room(k, m, k * gm, device) if keep_x else (None, 0, 0)
    w_t, w_q, w_s = _room(k, n, gk * gn, device) if keep_w else (None, 0, 0)
    y = torch.empty(m, n, dtype=x.dtype, device=device)
    _enqueue_quantize(x, 1, q, s, 1, m, x_q, x_s, None)
    _enqueue_quantize(weight, _BLOCK, w, ws, gk, 1, w_q, w_s, None)
    _enqueue_product(m, n, k, q, s, 1, m, w, ws, gk, 1, _BLOCK, bias, bias_code, y)
    return y, (x_t, w_t)


def _linear_backward(dy: Tensor, x_t, w_t, k: int, x_dtype, w_dtype, b_dtype):
    """The gradients for which a dtype is given."""
    (m, n), device = dy.shape, dy.device
    gm, gn, gk = -(-m // _BLOCK), -(-n // _BLOCK), -(-k // _BLOCK)
    d_buf, q, s = _room(m, n, m * gn, device) if x_dtype else (None, 0, 0)
    t_buf, d_q, d_s = _room(n, m, n * gm, device) if w_dtype else (None, 0, 0)
    dx = dw = db = None
    if b_dtype:
        db = torch.empty(n, dtype=b_dtype, device=device)
    _enqueue_quantize(dy, 1, q, s, 1, m, d_q, d_s, db)
    if x_dtype:
        dx = torch.empty(m, k, dtype=x_dtype, device=device)
        at = w_t.data_ptr()
        _enqueue_product(m, k, n, q, s, 1, m, at, at + k * (-(-n // 16) * 16), 1, gk, _BLOCK, None, 0, dx)
    if w_dtype and m:
        dw = torch.empty(n, k, dtype=w_dtype, device=device)
        at = x_t.data_ptr()
        _enqueue_product(n, k, m, d_q, d_s, 1, n, at, at + k * (-(-m // 16) * 16), 1, k, 1, None, 0, dw)
    elif w_dtype:
        dw = torch.zeros(n, k, dtype=w_dtype, device=device)
    return dx, dw, db


def block_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None) -> Tensor:
    """x weight^T + bias in x's dtype by 8-bit products, with autograd: x (..., K) is quantised
    per 128 columns of a row, weight (N, K) per 128 x 128 block (`block_quantize`), and in the
    backward the gradient per 128 columns for x's and, like x, per 128 rows for weight's. Every
    sum is held in fp32, those of large products with 16-bit results in the tensor cores (`block_mm`
    with `power_of_two`: weight's gradient adds up as many products as x has rows). What the
    backward needs of x and weight is kept in 8 bits. The gradients are those of the product at the
    quantised values (rounding counts as the identity); they cannot be differentiated again: that is
    an error."""
    if _is_compiling():
        return _linear_untraced(x, weight, bias)
    for name, t in (("X", x), ("Weight", weight)):
        if t.dtype not in _CODE:
            _check_tensor_dtype(name, t)
    if not x.shape or not x.shape[-1]:
        _check_x_shape(x.shape)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or not weight.shape[0]:
        raise ValueError(f"weight must be (N, K) with K={x.shape[-1]} and at least one row, got {tuple(weight.shape)}")
    if weight.device != x.device:
        _check_same_device("weight", weight, x.device)
    _check_bias(bias, weight.shape[0], x.device)
    return BlockLinearFunction.apply(x, weight, bias, torch.is_grad_enabled())


_quantize_untraced = torch.compiler.disable(block_quantize)
_mm_untraced = torch.compiler.disable(block_mm)
_linear_untraced = torch.compiler.disable(block_linear)
