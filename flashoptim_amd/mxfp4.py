"""Microscaled 4-bit floating point (MXFP4): quantiser, products, and a linear layer that trains and serves in it.

32 values share one power of two and are E2M1 codes each: 17/32 bytes a value, and the matrix cores multiply them at four times
the bfloat16 rate.  The reference package has nothing of the kind; the format is that of the OCP microscaling specification.
"""

from __future__ import annotations

from typing import Optional, Union

import torch
from torch.autograd import forward_ad

from . import _native, kernels
from ._native import DTYPE_CODE

GROUP_SIZE = 32
BLOCK = 128  # rows are filled up to multiples of it
_MOST_TOKENS = 64  # FO_MXFP4_MOST_TOKENS
_RAW_BLOCKS = 256  # blocks of the input that the product for few rows quantises itself (fo_mxfp4_tokens_workspace)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


class MXFP4Tensor:
    """A ``rows x cols`` matrix in MXFP4, its rows cut into groups of 32.

    Args:
        codes: uint8 ``(rows, 64 * ceil(cols / 128))``, contiguous: two E2M1 codes a byte (sign, two exponent bits, one
            mantissa bit), the first in the low half; zero beyond `cols`.
        scales: uint8 ``(rows, 4 * ceil(cols / 128))``, contiguous: the power of two of 32 values, plus 127; 255 for a group
            that held an infinity or a NaN.
        shape: ``(rows, cols)``.
    """

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        rows, cols = shape
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"codes and scales must be uint8, got {codes.dtype} and {scales.dtype}.")
        if rows < 0 or cols < 0 or tuple(codes.shape) != (rows, 64 * _blocks(cols)) or tuple(scales.shape) != (rows, 4 * _blocks(cols)):
            raise ValueError(
                f"a {rows} x {cols} matrix has codes of shape {(rows, 64 * _blocks(cols))} and scales of shape "
                f"{(rows, 4 * _blocks(cols))}, got {tuple(codes.shape)} and {tuple(scales.shape)}.")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        kernels._require_same_device(codes, scales, "scales")
        self.codes, self.scales, self.shape = codes, scales, (int(rows), int(cols))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, device) -> "MXFP4Tensor":
        return MXFP4Tensor(self.codes.to(device), self.scales.to(device), self.shape)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return mxfp4_dequantize(self, dtype)

    def __repr__(self) -> str:
        return f"MXFP4Tensor(shape={self.shape}, device={self.device})"


def _check_matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    kernels._require_device(x, what)
    if x.dtype not in DTYPE_CODE:
        raise ValueError(f"{what} expects fp32, bf16 or fp16 input, got {x.dtype}.")
    if x.dim() != 2:
        raise ValueError(f"{what} expects a matrix, got shape {tuple(x.shape)}.")
    if x.requires_grad:
        x = x.detach()
    return x.resolve_neg() if x.is_neg() else x


def _empty(rows: int, cols: int, device: torch.device) -> MXFP4Tensor:
    q = MXFP4Tensor.__new__(MXFP4Tensor)  # what is made here needs no check
    q.codes = torch.empty((rows, 64 * _blocks(cols)), dtype=torch.uint8, device=device)
    q.scales = torch.empty((rows, 4 * _blocks(cols)), dtype=torch.uint8, device=device)
    q.shape = (rows, cols)
    return q


def _quantize(x: torch.Tensor, rows: bool, columns: bool) -> tuple[Optional[MXFP4Tensor], Optional[MXFP4Tensor]]:
    """The row forms of `x` and of its transpose, as asked for, from one read."""
    r, c = x.shape
    if x.stride(1) != 1 and c > 1:
        if x.stride(0) == 1 or r == 1:  # the transpose's rows are what is contiguous
            columns_out, rows_out = _quantize(x.t(), columns, rows)
            return rows_out, columns_out
        x = x.contiguous()
    by_row = _empty(r, c, x.device) if rows else None
    by_column = _empty(c, r, x.device) if columns else None
    if x.numel() > 0:
        ptr = [None if t is None else p for t in (by_row, by_column)
               for p in ((None, None) if t is None else (t.codes.data_ptr(), t.scales.data_ptr()))]
        with _native.device_guard(x.device):
            rc = _native.lib().fo_mxfp4_quantize(x.data_ptr(), DTYPE_CODE[x.dtype], r, c, x.stride(0), *ptr,
                                                 _native.current_stream_ptr(x.device))
        _native.check(rc, "fo_mxfp4_quantize")
    return by_row, by_column


def mxfp4_quantize(x: torch.Tensor, transpose: bool = False) -> MXFP4Tensor:
    """The matrix `x` (fp32, bf16 or fp16, any strides), or its transpose, in MXFP4.

    The scale of a group is the power of two of its largest magnitude, over 4; values are rounded to the nearest code,
    ties to the even one, and cut off at 6 times the scale.  A group with an infinity or a NaN comes back as NaNs.  No gradient flows
    through.
    """
    rows, columns = _quantize(_check_matrix(x, "mxfp4_quantize"), not transpose, transpose)
    return columns if transpose else rows


def mxfp4_quantize_both(x: torch.Tensor) -> tuple[MXFP4Tensor, MXFP4Tensor]:
    """``(mxfp4_quantize(x), mxfp4_quantize(x, transpose=True))`` from one read of `x`."""
    return _quantize(_check_matrix(x, "mxfp4_quantize_both"), True, True)


def mxfp4_dequantize(q: MXFP4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that `q` stands for, as a matrix of `dtype` (fp32, bf16 or fp16).  bf16 and fp32 hold them exactly."""
    if not isinstance(q, MXFP4Tensor):
        raise ValueError(f"mxfp4_dequantize expects an MXFP4Tensor, got {type(q)}.")
    if dtype not in DTYPE_CODE:
        raise ValueError(f"Unsupported dtype {dtype}.")
    kernels._require_device(q.codes, "mxfp4_dequantize")
    rows, cols = q.shape
    out = torch.empty((rows, cols), dtype=dtype, device=q.device)
    if out.numel() > 0:
        with _native.device_guard(q.device):
            rc = _native.lib().fo_mxfp4_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), rows, cols, out.data_ptr(),
                                                   DTYPE_CODE[dtype], _native.current_stream_ptr(q.device))
        _native.check(rc, "fo_mxfp4_dequantize")
    return out


def _tokens(x: torch.Tensor, weight: MXFP4Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The product for a few rows of plain values; every argument is checked, x's columns are adjacent."""
    m, (n, k) = x.shape[0], weight.shape
    out = torch.empty((m, n), dtype=dtype, device=x.device)
    blocks = m * _blocks(k)
    size, workspace = 0, None
    if blocks > _RAW_BLOCKS:
        size = blocks * 68
        workspace = torch.empty(size, dtype=torch.uint8, device=x.device)  # held until the launches are in the stream
    with _native.device_guard(x.device):
        rc = _native.lib().fo_mxfp4_tokens(x.data_ptr(), DTYPE_CODE[x.dtype], m, x.stride(0), weight.codes.data_ptr(), weight.scales.data_ptr(),
                                           n, k, out.data_ptr(), DTYPE_CODE[dtype], _native.ptr(workspace), size, _native.current_stream_ptr(x.device))
    if rc:
        _native.check(rc, "fo_mxfp4_tokens")
    return out


def mxfp4_matmul(a: Union[MXFP4Tensor, torch.Tensor], b: MXFP4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T`` of an ``m x k`` and an ``n x k`` matrix in MXFP4, summed in fp32, as an ``m x n`` matrix of `dtype`.

    `a` may be a plain matrix: it is quantised on the way, in the product's own kernel where it is a few short rows.  No gradient flows
    through; :func:`mxfp4_linear` has them.
    """
    if not isinstance(b, MXFP4Tensor):
        raise ValueError(f"mxfp4_matmul expects its second operand as an MXFP4Tensor, got {type(b)}.")
    if dtype not in DTYPE_CODE:
        raise ValueError(f"Unsupported dtype {dtype}.")
    plain = not isinstance(a, MXFP4Tensor)
    if plain:
        a = _check_matrix(a, "mxfp4_matmul")
    kernels._require_device(b.codes, "mxfp4_matmul")
    if a.device != b.device:
        raise ValueError(f"b is on {b.device}, expected {a.device}.")
    (m, k), n = a.shape, b.shape[0]
    if b.shape[1] != k:
        raise ValueError(f"operands of shapes {tuple(a.shape)} and {tuple(b.shape)} do not contract over one length")
    if k == 0:
        return torch.zeros((m, n), dtype=dtype, device=b.device)
    if m == 0 or n == 0:
        return torch.empty((m, n), dtype=dtype, device=b.device)
    if plain and m <= _MOST_TOKENS:
        return _tokens(a if a.stride(1) == 1 or k == 1 else a.contiguous(), b, dtype)
    if plain:
        a = _quantize(a, True, False)[0]
    out = torch.empty((m, n), dtype=dtype, device=b.device)
    with _native.device_guard(b.device):
        rc = _native.lib().fo_mxfp4_product(a.codes.data_ptr(), a.scales.data_ptr(), m, b.codes.data_ptr(), b.scales.data_ptr(),
                                            n, k, out.data_ptr(), DTYPE_CODE[dtype], _native.current_stream_ptr(b.device))
    _native.check(rc, "fo_mxfp4_product")
    return out


def _form_bytes(rows: int, cols: int) -> int:
    return (rows * _blocks(cols) * 68 + 255) // 256 * 256  # fo_mxfp4_form_bytes


def _adjacent(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _linear(x: torch.Tensor, weight: torch.Tensor, need_dx: bool, need_dw: bool) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The layer's output, and the column forms that its gradients need: of x for dw, then of the weight for dx."""
    x, weight = _check_matrix(x, "mxfp4_linear"), _check_matrix(weight, "mxfp4_linear")
    (tokens, inner), outer = x.shape, weight.shape[0]
    if not (tokens and inner and outer):
        return torch.zeros((tokens, outer), dtype=x.dtype, device=x.device), None
    x, weight = _adjacent(x), _adjacent(weight)
    device = x.device
    x_bytes, w_bytes = _form_bytes(inner, tokens) if need_dw else 0, _form_bytes(inner, outer) if need_dx else 0
    kept, at = None, 0
    if need_dx or need_dw:
        kept = torch.empty(x_bytes + w_bytes, dtype=torch.uint8, device=device)
        at = kept.data_ptr()
    used = _form_bytes(tokens, inner) + _form_bytes(outer, inner)  # the row forms
    workspace = torch.empty(used, dtype=torch.uint8, device=device)
    y = torch.empty((tokens, outer), dtype=x.dtype, device=device)
    with _native.device_guard(device):
        rc = _native.lib().fo_mxfp4_linear_forward(
            x.data_ptr(), DTYPE_CODE[x.dtype], tokens, x.stride(0), weight.data_ptr(), DTYPE_CODE[weight.dtype], outer, weight.stride(0),
            inner, at if need_dw else None, at + x_bytes if need_dx else None, y.data_ptr(), workspace.data_ptr(), used,
            _native.current_stream_ptr(device))
    if rc:
        _native.check(rc, "fo_mxfp4_linear_forward")
    return y, kept


class _Linear(torch.autograd.Function):
    """x (tokens, in) and weight (out, in) to x weight', every product on MXFP4 forms of its operands along the contracted axis.

    What the backward pass needs of x and of the weight is their column forms, 17/32 bytes a value, made in the same read
    as the row forms; x itself is not kept.
    """

    @staticmethod
    def forward(ctx, x, weight):
        ctx.dtypes, ctx.shapes = (x.dtype, weight.dtype), (x.shape, weight.shape)
        y, kept = _linear(x, weight, *ctx.needs_input_grad)
        ctx.save_for_backward(kept)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_dx, need_dw = ctx.needs_input_grad
        (tokens, inner), (outer, _) = ctx.shapes
        device = dy.device
        empty = not (tokens and inner and outer)
        make = torch.zeros if empty else torch.empty
        dx = make((tokens, inner), dtype=ctx.dtypes[0], device=device) if need_dx else None
        dw = make((outer, inner), dtype=ctx.dtypes[1], device=device) if need_dw else None
        if empty:
            return dx, dw
        (kept,) = ctx.saved_tensors
        dy = _adjacent(_check_matrix(dy, "mxfp4_linear backward"))
        at = kept.data_ptr()
        x_bytes = _form_bytes(inner, tokens) if need_dw else 0
        used = (_form_bytes(tokens, outer) if need_dx else 0) + (_form_bytes(outer, tokens) if need_dw else 0)
        workspace = torch.empty(used, dtype=torch.uint8, device=device)
        with _native.device_guard(device):
            rc = _native.lib().fo_mxfp4_linear_backward(
                dy.data_ptr(), DTYPE_CODE[dy.dtype], tokens, dy.stride(0), outer, inner, at if need_dw else None, at + x_bytes if need_dx else None,
                _native.ptr(dx), DTYPE_CODE[ctx.dtypes[0]], _native.ptr(dw), DTYPE_CODE[ctx.dtypes[1]], workspace.data_ptr(), used,
                _native.current_stream_ptr(device))
        if rc:
            _native.check(rc, "fo_mxfp4_linear_backward")
        return dx, dw


class _FrozenLinear(torch.autograd.Function):
    """The same with a weight that is held in MXFP4 and not trained."""

    @staticmethod
    def forward(ctx, x, codes, scales, shape):
        ctx.dtype, ctx.shape = x.dtype, shape
        ctx.save_for_backward(codes, scales)
        return mxfp4_matmul(x, MXFP4Tensor(codes, scales, shape), x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        weight = MXFP4Tensor(*ctx.saved_tensors, ctx.shape)
        # the scales have to run along the other axis now; bf16 holds the weight's values
        columns = mxfp4_quantize(mxfp4_dequantize(weight), transpose=True)
        return mxfp4_matmul(dy, columns, ctx.dtype), None, None, None


def _has_tangent(x: torch.Tensor) -> bool:
    return forward_ad.unpack_dual(x).tangent is not None


def mxfp4_linear(x: torch.Tensor, weight: Union[torch.Tensor, MXFP4Tensor]) -> torch.Tensor:
    """``x @ weight.T`` in MXFP4, with gradients.

    Args:
        x: ``(..., in)`` in fp32, bf16 or fp16.
        weight: ``(out, in)``; a tensor is quantised in the call and receives a gradient, an :class:`MXFP4Tensor` is frozen.

    Returns:
        ``(..., out)`` in the type of `x`.

    Each of the three products of a training step contracts over another axis, so each operand is quantised along two:

        y = Q(x) Q(w)',    dx = Q(dy) Q(w')',    dw = Q(dy') Q(x')'

    with Q along rows; the quantisation itself counts as the identity in the backward pass.

    Raises:
        NotImplementedError: no ROCm device, or an operand with a forward-mode tangent (there is no such derivative here).
    """
    inner = weight.shape[-1]
    if (type(weight) is MXFP4Tensor and type(x) is torch.Tensor and x.dim() == 2 and x.shape[1] == inner and x.is_cuda
            and 0 < x.shape[0] <= _MOST_TOKENS and x.stride(1) == 1 and inner and weight.shape[0] and x.dtype in DTYPE_CODE
            and x.device == weight.codes.device and not x.is_neg() and not (x.requires_grad and torch.is_grad_enabled()) and not _has_tangent(x)):
        return _tokens(x, weight, x.dtype)  # the call of a decoding step, without the ways round
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] != inner:
        raise ValueError(f"mxfp4_linear: input of shape {tuple(x.shape)} does not fit a weight of shape {tuple(weight.shape)}")
    if weight.device != x.device:
        raise ValueError(f"weight is on {weight.device}, expected {x.device}.")
    if _has_tangent(x) or (isinstance(weight, torch.Tensor) and _has_tangent(weight)):
        raise NotImplementedError("mxfp4_linear has no forward-mode derivative")
    tokens = x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), inner)
    if isinstance(weight, MXFP4Tensor):
        if torch.is_grad_enabled() and x.requires_grad:
            y = _FrozenLinear.apply(tokens, weight.codes, weight.scales, weight.shape)
        else:
            y = mxfp4_matmul(tokens, weight, x.dtype)
    else:
        if weight.dim() != 2:
            raise ValueError(f"mxfp4_linear expects a matrix as weight, got shape {tuple(weight.shape)}.")
        if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
            y = _Linear.apply(tokens, weight)
        else:
            y, _ = _linear(tokens, weight, False, False)
        if x.dim() == 2:
            return y
    return y.reshape(*x.shape[:-1], weight.shape[0])


class MXFP4Linear(torch.nn.Linear):
    """``torch.nn.Linear`` whose three products run in MXFP4 (:func:`mxfp4_linear`); the weight keeps its type, so the optimizers of
    this package hold masters and correction bits for it as for any other; every call quantises it, so a weight that is only served is better
    held by :func:`mxfp4_quantize`.  A bias is added by torch's rules: one in fp32 makes an fp32 output of a 16-bit input."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        y = mxfp4_linear(input, self.weight)
        return y if self.bias is None else y + self.bias
