"""Rows of an embedding matrix by token, scaled, with a gradient that is summed in a fixed order.

The reference package has nothing of the kind.  ``torch.nn.Embedding``'s meaning and arguments, as far as they are taken here.
"""

from __future__ import annotations

import functools
import math
import sys
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _autograd, _native, kernels
from ._native import DTYPE_CODE

_INDEX_BYTES = {torch.int64: 8, torch.int32: 4}


def _check_tokens(tokens: torch.Tensor, device: torch.device, what: str) -> torch.Tensor:
    """`tokens` as the kernels read them: flat and contiguous."""
    if not isinstance(tokens, torch.Tensor) or tokens.dtype not in _INDEX_BYTES:
        raise ValueError(f"{what} expects int64 or int32 tokens, got {getattr(tokens, 'dtype', type(tokens))}.")
    if tokens.device != device:
        raise ValueError(f"tokens are on {tokens.device}, expected {device}.")
    return tokens.reshape(-1).contiguous()


def _check_values(x: torch.Tensor, what: str, name: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{what} expects {name} as a tensor, got {type(x)}.")
    kernels._require_device(x, what)
    if x.dtype not in DTYPE_CODE:
        raise ValueError(f"{what} expects fp32, bf16 or fp16 as {name}, got {x.dtype}.")
    if x.numel() and not x.data_ptr():    # to the C entry points an operand without an address is one that was left out
        raise NotImplementedError(f"{what} expects {name} in memory, got a {type(x).__name__} that has none of its own.")
    if forward_ad.unpack_dual(x).tangent is not None:
        raise NotImplementedError(f"{what} has no forward-mode derivative")
    return x


def _plain(x: torch.Tensor) -> torch.Tensor:
    """`x` for the kernels: a tensor whose last axis is adjacent in memory and whose negation, if torch put one off, is done."""
    if x.requires_grad:
        x = x.detach()
    if x.is_neg():
        x = x.resolve_neg()
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


def _traced(what: str) -> bool:
    """Whether torch.jit.trace records.  It sees torch's operations, of which a launch is none: a call goes into the trace as one operation, a Function's.  A tracer into
    an fx graph has no such thing, and is refused."""
    fx = sys.modules.get("torch.fx.experimental.proxy_tensor")
    if fx is not None and fx.get_proxy_mode() is not None:
        raise NotImplementedError(f"{what} cannot be traced into an fx graph: it is not made of torch's operations")
    return torch.jit.is_tracing()


def _sizes(x: torch.Tensor) -> tuple:
    """The shape of `x` in numbers; under torch.jit.trace it is made of tensors."""
    return tuple(map(int, x.shape))


def _save(ctx, *tensors: Optional[torch.Tensor]) -> None:
    ctx.save_for_backward(*tensors)
    ctx.saved_as = [None if t is None else (_sizes(t), t.dtype, t.device) for t in tensors]


def _saved(ctx, what: str) -> list:
    """What _save was given, as the kernels read it.  Hooks on saved tensors may lay them out anew, but not give back other ones."""
    out = []
    for t, was in zip(ctx.saved_tensors, ctx.saved_as):
        if (None if t is None else (tuple(t.shape), t.dtype, t.device)) != was:
            raise RuntimeError(f"{what}: a hook on saved tensors gave back {(tuple(t.shape), t.dtype, t.device)} in place of {was}.")
        out.append(None if t is None else _plain(t))
    return out


def _differentiable_once(backward):
    """A backward pass without a derivative of its own: in a graph that records it, its results lead to an error."""

    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        error = torch._C._functions.DelayedError(b"trying to differentiate twice a function that has one derivative only", 1)
        return tuple(o if o is None else error(o.detach().requires_grad_()) for o in out)

    return wrapper


def _lookup(tokens: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    """tokens: flat.  Every argument is checked."""
    weight = _plain(weight)
    (vocabulary, width), n = _sizes(weight), int(tokens.numel())
    y = torch.empty((n, width), dtype=weight.dtype, device=weight.device)
    with _native.device_guard(weight.device):
        rc = _native.lib().fo_embedding(tokens.data_ptr(), _INDEX_BYTES[tokens.dtype], n, weight.data_ptr(), DTYPE_CODE[weight.dtype], vocabulary,
                                        width, weight.stride(0), scale, y.data_ptr(), _native.current_stream_ptr(weight.device))
    if rc:
        _native.check(rc, "fo_embedding")
    return y


class _Embedding(torch.autograd.Function):
    """Keeps the tokens alone."""

    @staticmethod
    def forward(ctx, weight, tokens, scale, padding):
        ctx.shape, ctx.scale, ctx.padding = _sizes(weight), scale, padding
        _save(ctx, tokens)
        return _lookup(tokens, weight, scale)

    @staticmethod
    @_differentiable_once
    def backward(ctx, dy):
        (tokens,) = _saved(ctx, "embedding")
        vocabulary, width = ctx.shape
        dy = _plain(dy)
        device, lib = dy.device, _native.lib()
        dw = torch.empty((vocabulary, width), dtype=dy.dtype, device=device)
        size = lib.fo_embedding_backward_workspace(tokens.numel(), vocabulary, width)
        if size < 0:
            _native.check(size, "fo_embedding_backward")
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        with _native.device_guard(device):
            rc = lib.fo_embedding_backward(tokens.data_ptr(), _INDEX_BYTES[tokens.dtype], tokens.numel(), dy.data_ptr(), DTYPE_CODE[dy.dtype], dy.stride(0),
                                           vocabulary, width, ctx.scale, ctx.padding, dw.data_ptr(), workspace.data_ptr(), size,
                                           _native.current_stream_ptr(device))
        if rc:
            _native.check(rc, "fo_embedding_backward")
        return dw, None, None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[tokens]``, rounded once, with the gradient of `weight`.

    Args:
        tokens: int64 or int32, any shape.
        weight: ``(vocabulary, width)`` in fp32, bf16 or fp16, any strides.
        scale: what every row is multiplied by (the root of the width in models that scale their embeddings).
        padding_idx: a token that gives `weight` no gradient; negative ones count from the end.

    Returns:
        ``(*tokens.shape, width)`` in the type of `weight`.

    The gradient is dense, summed in fp32 in a fixed order and rounded once, so it repeats to the bit.  A token outside the
    vocabulary makes a row of NaNs and gives no gradient (the call does not wait for the GPU to look at the tokens).

    Raises:
        NotImplementedError: no ROCm device, or a weight with a forward-mode tangent (there is no such derivative here).
    """
    if _autograd.embedding is not None and (padding_idx is None or (isinstance(weight, torch.Tensor) and weight.dim() == 2 and 0 <= padding_idx < weight.shape[0])):
        y = _autograd.embedding(tokens, weight, scale, -1 if padding_idx is None else padding_idx)
        if y is not None:
            return y
    _autograd.bind()
    _check_values(weight, "embedding", "weight")
    if weight.dim() != 2:
        raise ValueError(f"embedding expects a matrix as weight, got shape {tuple(weight.shape)}.")
    vocabulary, width = weight.shape
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}.")
    padding = -1
    if padding_idx is not None:
        if not -vocabulary <= padding_idx < vocabulary:
            raise ValueError(f"padding_idx must be within the vocabulary of {vocabulary}, got {padding_idx}.")
        padding = int(padding_idx % vocabulary)
    flat = _check_tokens(tokens, weight.device, "embedding")
    if _traced("embedding") or (torch.is_grad_enabled() and weight.requires_grad):
        y = _Embedding.apply(weight, flat, scale, padding)
    else:
        y = _lookup(flat, weight, scale)
    return y.view(*tokens.shape, width)


class FlashEmbedding(torch.nn.Embedding):
    """``torch.nn.Embedding`` through :func:`embedding`, with its `scale`.  Of torch's options `padding_idx` is taken; the gradient is
    dense."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, scale: float = 1.0, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale = scale

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx: Optional[int] = None, scale: float = 1.0) -> "FlashEmbedding":
        """A module whose weight is `embeddings`, without a gradient where `freeze` says so."""
        if embeddings.dim() != 2:
            raise ValueError(f"FlashEmbedding expects a matrix, got shape {tuple(embeddings.shape)}.")
        made = cls(*embeddings.shape, padding_idx=padding_idx, scale=scale, device="meta", dtype=embeddings.dtype)
        made.weight = torch.nn.Parameter(embeddings, requires_grad=not freeze)
        return made

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return embedding(input, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return super().extra_repr() + f", scale={self.scale}"
