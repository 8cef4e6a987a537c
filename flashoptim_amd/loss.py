"""Cross entropy over a vocabulary from hidden states and the output matrix, without the logits in memory, with gradients.

The reference package has nothing of the kind.  ``torch.nn.functional.cross_entropy``'s meaning and arguments, of the logits that
``torch.nn.functional.linear`` would make.
"""

from __future__ import annotations

import torch

from . import _autograd, _native
from ._native import DTYPE_CODE
from .embed import _INDEX_BYTES, _check_tokens, _check_values, _differentiable_once, _plain, _save, _saved, _sizes, _traced

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}  # fo_reduction


def _forward(x, weight, target, how):
    """The loss, and what the backward pass takes beside the operands."""
    (tokens, width), (vocabulary, _) = _sizes(x), _sizes(weight)
    device, lib = x.device, _native.lib()
    ignore, reduction, smoothing = how
    loss = torch.empty(tokens if reduction == 0 else (), dtype=torch.float32, device=device)
    # fp32 numbers and int32 labels.  Hooks on saved tensors may convert what is floating-point; these are bits.
    kept = torch.empty(_native.LOSS_NUMBERS_A_TOKEN * tokens + 1, dtype=torch.int32, device=device)
    with _native.device_guard(device):
        size = lib.fo_linear_cross_entropy_workspace(x.data_ptr(), DTYPE_CODE[x.dtype], tokens, x.stride(0), weight.data_ptr(), weight.stride(0), vocabulary, width,
                                                     smoothing)
        if size < 0:
            _native.check(size, "fo_linear_cross_entropy")
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        rc = lib.fo_linear_cross_entropy(
            x.data_ptr(), DTYPE_CODE[x.dtype], tokens, x.stride(0), weight.data_ptr(), weight.stride(0), vocabulary, width, target.data_ptr(),
            _INDEX_BYTES[target.dtype], ignore, reduction, smoothing, loss.data_ptr(), kept.data_ptr(), workspace.data_ptr(), size,
            _native.current_stream_ptr(device))
    if rc:
        _native.check(rc, "fo_linear_cross_entropy")
    return loss, kept


class _LinearCrossEntropy(torch.autograd.Function):
    """Keeps its operands and three numbers a row."""

    @staticmethod
    def forward(ctx, x, weight, target, how):
        x, weight = _plain(x), _plain(weight)
        loss, kept = _forward(x, weight, target, how)
        _save(ctx, x, weight, kept)
        _, ctx.reduction, ctx.smoothing = how
        return loss

    @staticmethod
    @_differentiable_once
    def backward(ctx, upstream):
        x, weight, kept = _saved(ctx, "linear_cross_entropy")
        need_dx, need_dw = ctx.needs_input_grad[:2]
        (tokens, width), vocabulary = x.shape, weight.shape[0]
        device, lib = x.device, _native.lib()
        upstream = upstream.resolve_neg() if upstream.is_neg() else upstream
        dx = torch.empty((tokens, width), dtype=x.dtype, device=device) if need_dx else None
        dw = torch.empty((vocabulary, width), dtype=x.dtype, device=device) if need_dw else None
        with _native.device_guard(device):
            size = lib.fo_linear_cross_entropy_backward_workspace(x.data_ptr(), DTYPE_CODE[x.dtype], tokens, x.stride(0), weight.data_ptr(), weight.stride(0),
                                                                  vocabulary, width, need_dx, need_dw)
            if size < 0:
                _native.check(size, "fo_linear_cross_entropy_backward")
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
            rc = lib.fo_linear_cross_entropy_backward(
                x.data_ptr(), DTYPE_CODE[x.dtype], tokens, x.stride(0), weight.data_ptr(), weight.stride(0), vocabulary, width, ctx.reduction,
                ctx.smoothing, kept.data_ptr(), upstream.data_ptr(), upstream.stride(0) if upstream.dim() else 0, _native.ptr(dx), _native.ptr(dw), workspace.data_ptr(), size, _native.current_stream_ptr(device))
        if rc:
            _native.check(rc, "fo_linear_cross_entropy_backward")
        return dx, dw, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100, reduction: str = "mean",
                         label_smoothing: float = 0.0) -> torch.Tensor:
    """``cross_entropy(x @ weight.T, target, ...)`` in fp32, with gradients; the logits never exist in memory.

    Args:
        x: ``(..., width)`` in fp32, bf16 or fp16.
        weight: ``(vocabulary, width)`` of the type of `x`.
        target: int64 or int32, of the shape of `x` without its last axis.
        ignore_index: targets of this value have no loss and no gradient, whatever stands in their rows of `x`.
        reduction: "mean" over the targets that are not ignored (NaN where all are, as in torch), "sum" or "none".
        label_smoothing: the share of each target that is spread over the vocabulary.

    Returns:
        The loss in fp32: a number, or of the shape of `target`.

    Logits are summed in fp32 and not rounded.  Their gradient is rounded once to the type of `x`, between the products; what the target's entry, by far the largest of most rows, loses in
    that goes into the gradient of `x` all the same, not into that of `weight`.  The backward pass computes them again, a piece of the vocabulary at a time, so that of size tokens
    x vocabulary there is only a piece of their gradient; the sums have a fixed order, so results repeat to the bit.  Between the passes
    `x`, `weight` and three numbers a row are kept.  A target outside the vocabulary makes a NaN (the call does not wait for
    the GPU to look at the targets).

    Raises:
        NotImplementedError: no ROCm device, or an operand with a forward-mode tangent (there is no such derivative here).
    """
    if _autograd.linear_cross_entropy is not None and reduction in _REDUCTIONS:
        loss = _autograd.linear_cross_entropy(x, weight, target, ignore_index, _REDUCTIONS[reduction], label_smoothing)
        if loss is not None:
            return loss
    _autograd.bind()
    _check_values(x, "linear_cross_entropy", "x")
    _check_values(weight, "linear_cross_entropy", "weight")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: x of shape {tuple(x.shape)} does not fit a weight of shape {tuple(weight.shape)}")
    if weight.device != x.device:
        raise ValueError(f"weight is on {weight.device}, expected {x.device}.")
    if weight.dtype != x.dtype:
        raise ValueError(f"linear_cross_entropy expects a weight of x's type, got {weight.dtype} beside {x.dtype}.")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction is one of {', '.join(_REDUCTIONS)}, got {reduction!r}.")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be between 0 and 1, got {label_smoothing}.")
    flat = _check_tokens(target, x.device, "linear_cross_entropy")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: targets of shape {tuple(target.shape)} do not fit x of shape {tuple(x.shape)}")
    if not (weight.shape[0] and weight.shape[1]):
        raise ValueError("linear_cross_entropy: a vocabulary or rows of no values")
    if flat.numel() == 0:
        raise ValueError("linear_cross_entropy: no rows")
    how = (int(ignore_index), _REDUCTIONS[reduction], float(label_smoothing))
    rows = x if x.dim() == 2 else x.reshape(flat.numel(), x.shape[-1])
    if _traced("linear_cross_entropy") or (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)):
        loss = _LinearCrossEntropy.apply(rows, weight, flat, how)
    else:
        loss, _ = _forward(_plain(rows), _plain(weight), flat, how)
    return loss.view(target.shape) if reduction == "none" else loss
