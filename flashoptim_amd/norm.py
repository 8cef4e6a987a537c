"""Root-mean-square norm with the residual's addition in front of it, with gradients, and with its output in MXFP4.

The reference package has nothing of the kind.  ``torch.nn.functional.rms_norm``'s meaning over the last axis.
"""

from __future__ import annotations

import math
import operator
from typing import Optional, Union

import torch

from . import _autograd, _native
from ._native import DTYPE_CODE
from .embed import _check_values, _differentiable_once, _plain, _save, _saved, _sizes, _traced
from .mxfp4 import MXFP4Tensor, _empty


def _rows(x: torch.Tensor, width: int) -> torch.Tensor:
    x = _plain(x)
    return x if x.dim() == 2 else x.reshape(math.prod(_sizes(x)[:-1]), width)


def _forward(x, weight, residual, eps, keep):
    """x and residual as matrices of adjacent values.  y, the stream, and the number a row that the backward pass takes."""
    rows, width = _sizes(x)
    device = x.device
    y = torch.empty((rows, width), dtype=x.dtype, device=device)
    stream = None if residual is None else torch.empty((rows, width), dtype=residual.dtype, device=device)
    inverse = torch.empty(rows, dtype=torch.float32, device=device) if keep else None
    with _native.device_guard(device):
        rc = _native.lib().fo_rms_norm(
            x.data_ptr(), DTYPE_CODE[x.dtype], rows, width, x.stride(0), _native.ptr(residual), 0 if residual is None else DTYPE_CODE[residual.dtype],
            0 if residual is None else residual.stride(0), _native.ptr(weight), 0 if weight is None else DTYPE_CODE[weight.dtype], eps, _native.ptr(stream),
            y.data_ptr(), _native.ptr(inverse), _native.current_stream_ptr(device))
    if rc:
        _native.check(rc, "fo_rms_norm")
    return y, stream, inverse


class _RMSNorm(torch.autograd.Function):
    """Keeps the stream (without a residual x itself) and one number a row."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        ctx.x_dtype = x.dtype
        plain = None if weight is None else _plain(weight)
        x_rows = _rows(x, x.shape[-1])
        y, stream, inverse = _forward(x_rows, plain, None if residual is None else _rows(residual, x.shape[-1]), eps, True)
        _save(ctx, x_rows if residual is None else stream, plain, inverse)
        ctx.shape = _sizes(x)
        y = y.view(x.shape)
        return y if residual is None else (y, stream.view(x.shape))

    @staticmethod
    @_differentiable_once
    def backward(ctx, dy, dstream=None):
        need_dx, need_dw, need_dresidual, _ = ctx.needs_input_grad
        if dy is None:    # nothing comes from the norm, whatever stands in its rows
            if dstream is None:
                return None, None, None, None
            dw = None
            if need_dw:
                shape, dtype, device = ctx.saved_as[1]
                dw = torch.zeros(shape, dtype=dtype, device=device)
            return dstream.to(ctx.x_dtype) if need_dx else None, dw, dstream if need_dresidual else None, None
        s, weight, inverse = _saved(ctx, "rms_norm")
        rows, width = s.shape
        device, lib = s.device, _native.lib()
        dy = _rows(dy, width)
        dstream = None if dstream is None else _rows(dstream, width)
        same = s.dtype == ctx.x_dtype
        dx = torch.empty((rows, width), dtype=ctx.x_dtype, device=device) if need_dx or (need_dresidual and same) else None
        dresidual = torch.empty((rows, width), dtype=s.dtype, device=device) if need_dresidual and not same else None
        dw, workspace, size = None, None, 0
        with _native.device_guard(device):
            if need_dw:
                dw = torch.empty(weight.shape, dtype=weight.dtype, device=device) if rows else torch.zeros(weight.shape, dtype=weight.dtype, device=device)
                size = lib.fo_rms_norm_backward_workspace(rows, width)
                if size < 0:
                    _native.check(size, "fo_rms_norm_backward")
                workspace = torch.empty(size, dtype=torch.uint8, device=device)
            rc = lib.fo_rms_norm_backward(
                s.data_ptr(), DTYPE_CODE[s.dtype], s.stride(0), _native.ptr(weight), 0 if weight is None else DTYPE_CODE[weight.dtype], inverse.data_ptr(),
                dy.data_ptr(), DTYPE_CODE[dy.dtype], dy.stride(0), _native.ptr(dstream), 0 if dstream is None else dstream.stride(0), rows, width,
                _native.ptr(dx), _native.ptr(dresidual), _native.ptr(dw), _native.ptr(workspace), size, _native.current_stream_ptr(device))
        if rc:
            _native.check(rc, "fo_rms_norm_backward")
        dx = None if dx is None else dx.view(ctx.shape)
        if same and need_dresidual:
            dresidual = dx
        elif dresidual is not None:
            dresidual = dresidual.view(ctx.shape)
        return dx if need_dx else None, dw, dresidual, None


def _check(x, weight, residual, eps, what) -> float:
    _check_values(x, what, "x")
    if x.dim() < 1:
        raise ValueError(f"{what} expects rows, got a single value.")
    if weight is not None:
        _check_values(weight, what, "weight")
        if tuple(weight.shape) != (x.shape[-1],):
            raise ValueError(f"{what}: a weight of shape {tuple(weight.shape)} does not fit rows of {x.shape[-1]} values")
        if weight.device != x.device:
            raise ValueError(f"weight is on {weight.device}, expected {x.device}.")
    if residual is not None:
        _check_values(residual, what, "residual")
        if residual.shape != x.shape:
            raise ValueError(f"{what}: a residual of shape {tuple(residual.shape)} does not fit x of shape {tuple(x.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{what}: the residual is of x's type or fp32, got {residual.dtype} beside {x.dtype}.")
        if residual.device != x.device:
            raise ValueError(f"residual is on {residual.device}, expected {x.device}.")
    eps = float(eps)
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError(f"eps must be finite and not negative, got {eps}.")
    return eps


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6) -> Union[torch.Tensor, tuple[torch.Tensor, torch.Tensor]]:
    """``s / sqrt(mean(s * s) + eps) * weight`` over the last axis of ``s = x + residual``, with gradients.

    Args:
        x: ``(..., width)`` in fp32, bf16 or fp16.
        weight: ``(width,)`` of any of these types; ones where it is left out.
        residual: the stream so far, of the shape of `x` and of its type or fp32.

    Returns:
        The norm's output in the type of `x`; with a residual ``(output, s)``, `s` being the stream that goes on, rounded to the residual's
        type.  The norm is taken of the rounded `s`.

    The mean of the squares is summed in fp64, the gradients' sums in fp32; outputs and gradients are rounded once and repeat to the bit.  Where only `s` has a
    gradient, that is handed on as it is, whatever the norm of its rows.

    Raises:
        NotImplementedError: no ROCm device, or an operand with a forward-mode tangent (there is no such derivative here).
    """
    if _autograd.rms_norm is not None:
        got = _autograd.rms_norm(x, weight, residual, eps)
        if got is not None:
            return got
    _autograd.bind()
    eps = _check(x, weight, residual, eps, "rms_norm")
    needed = x.requires_grad or (weight is not None and weight.requires_grad) or (residual is not None and residual.requires_grad)
    if _traced("rms_norm") or (torch.is_grad_enabled() and needed):
        return _RMSNorm.apply(x, weight, residual, eps)
    width = x.shape[-1]
    y, stream, _ = _forward(_rows(x, width), None if weight is None else _plain(weight), None if residual is None else _rows(residual, width), eps, False)
    y = y.view(x.shape)
    return y if residual is None else (y, stream.view(x.shape))


def rms_norm_mxfp4(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                   eps: float = 1e-6) -> Union[MXFP4Tensor, tuple[MXFP4Tensor, torch.Tensor]]:
    """:func:`rms_norm` of a matrix's rows with the output in MXFP4, as :func:`mxfp4_matmul` reads it: one launch in place of the norm and
    the quantiser, the output quantised from fp32.  No gradient flows through.
    """
    if _autograd.rms_norm_mxfp4 is not None:
        got = _autograd.rms_norm_mxfp4(x, weight, residual, eps)
        if got is not None:
            y = MXFP4Tensor.__new__(MXFP4Tensor)  # what is made here needs no check
            y.codes, y.scales, y.shape = got[0], got[1], tuple(x.shape)
            return y if residual is None else (y, got[2])
    _autograd.bind()
    eps = _check(x, weight, residual, eps, "rms_norm_mxfp4")
    if _traced("rms_norm_mxfp4"):
        raise NotImplementedError("rms_norm_mxfp4 cannot be traced: what it makes is not a tensor")
    if x.dim() != 2:
        raise ValueError(f"rms_norm_mxfp4 expects a matrix, got shape {tuple(x.shape)}.")
    x, weight, residual = _plain(x), None if weight is None else _plain(weight), None if residual is None else _plain(residual)
    rows, width = x.shape
    device = x.device
    y = _empty(rows, width, device)
    stream = None if residual is None else torch.empty((rows, width), dtype=residual.dtype, device=device)
    with _native.device_guard(device):
        rc = _native.lib().fo_rms_norm_mxfp4(
            x.data_ptr(), DTYPE_CODE[x.dtype], rows, width, x.stride(0), _native.ptr(residual), 0 if residual is None else DTYPE_CODE[residual.dtype],
            0 if residual is None else residual.stride(0), _native.ptr(weight), 0 if weight is None else DTYPE_CODE[weight.dtype], eps, _native.ptr(stream),
            y.codes.data_ptr(), y.scales.data_ptr(), _native.current_stream_ptr(device))
    if rc:
        _native.check(rc, "fo_rms_norm_mxfp4")
    return y if residual is None else (y, stream)


class FlashRMSNorm(torch.nn.RMSNorm):
    """``torch.nn.RMSNorm`` over the last axis through :func:`rms_norm`: ``norm(x)``, or ``y, stream = norm(x, stream)``."""

    def __init__(self, width: int, eps: float = 1e-6, elementwise_affine: bool = True, device=None, dtype=None):
        super().__init__(operator.index(width), eps=eps, elementwise_affine=elementwise_affine, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if self.weight is None and x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"FlashRMSNorm: x of shape {tuple(x.shape)} does not have rows of {self.normalized_shape[0]} values")
        return rms_norm(x, self.weight, residual, self.eps)
