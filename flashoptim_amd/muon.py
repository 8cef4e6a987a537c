"""Orthogonalised updates: the Newton-Schulz iteration on stacks of matrices, and FlashMuon, the optimizer that steps hidden
matrices along the orthogonalised momentum.

The reference package has neither; names and defaults of the optimizer are those of ``torch.optim.Muon``, everything
around the update (8-bit momentum, correction bits, state dicts, gradient release) is :class:`FlashOptimizer`'s.
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Iterable
from typing import Any, Literal, Optional, Sequence

import torch

from . import _native, kernels
from ._native import DTYPE_CODE, MATRIX_MOST_LINES, FoMatrixShape, FoTensorDesc
from .base import FlashOptimizer, LaunchKey
from .launcher import BucketPlan, StepTensors
from .state import QuantizedTensorSpec

DEFAULT_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
DEFAULT_STEPS = 5
DEFAULT_EPS = 1e-7

# Device memory that the matrices of one launch may take (10 bytes an element and 6 per entry of a square of the shorter side), unless
# a single one needs more: a stack or list beyond it goes through in parts, to the same result.  It is held for the call only.  One
# layer of an 8B-parameter transformer needs 2.7 GB.  Four of them take 58.5 ms within 8 GiB and 59.0 to 60.0 within 1 to 4;
# 32 layers of a model 1000 wide 11.9 ms within 8, 12.2 within 3, 13.6 within 1.
WORKSPACE_BYTES = 8 << 30


def _check_iteration(steps: int, coefficients: Sequence[float], eps: float) -> None:
    if int(steps) != steps or not 1 <= steps < 100:
        raise ValueError(f"Newton-Schulz steps must be a whole number from 1 to 99, got {steps}")
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f"Newton-Schulz coefficients must be three finite numbers, got {coefficients}")
    if not eps >= 0.0:
        raise ValueError(f"Invalid epsilon value: {eps}")


def _check_lines(shape: Sequence[int]) -> None:
    if max(shape[-2:]) > MATRIX_MOST_LINES:
        raise ValueError(f"a matrix of {tuple(shape[-2:])} has more than {MATRIX_MOST_LINES} rows or columns")


def _workspace_bytes(shapes, n: int) -> int:
    size = _native.lib().fo_newton_schulz_workspace(shapes, n)
    if size < 0:
        _native.check(int(size), "fo_newton_schulz_workspace")
    return int(size)


def _three(coefficients: Sequence[float]):
    return (ctypes.c_float * 3)(*coefficients)


def newton_schulz(
    x: torch.Tensor,
    steps: int = DEFAULT_STEPS,
    coefficients: Sequence[float] = DEFAULT_COEFFICIENTS,
    eps: float = DEFAULT_EPS,
) -> torch.Tensor:
    """Orthogonalise a matrix, or every matrix of a stack, by Newton-Schulz products.

    With X the matrix or, where it has more rows than columns, its transpose: ``X <- X / (|X|_F + eps)``, then `steps` times
    ``X <- a X + (b S + c S S) X`` with ``S = X X'`` and (a, b, c) the `coefficients`.  The singular vectors stay, the
    singular values come near one.

    Args:
        x: ``(..., rows, cols)`` in fp32, bf16 or fp16 on a ROCm GPU, any strides.
        steps: how often the polynomial is applied (1 to 99).
        coefficients: (a, b, c) of the polynomial.  One that takes singular values far beyond one, so that an entry on the way passes fp16's
            range, comes back with infinities or NaNs.
        eps: added to the norm; a matrix of zeros stays one.

    Returns:
        bfloat16, whatever the type of `x` (the products run on fp16 parts: their error is 1e-4 to 1.3e-3 of the
        result's norm, less than this rounding's), in the shape of
        `x`; contiguous, or laid out like `x` where its columns and not its rows are contiguous.  A matrix with an infinity or
        a NaN comes back as NaNs.  No gradient flows through.
    """
    kernels._require_device(x, "newton_schulz")
    if x.dtype not in DTYPE_CODE:
        raise ValueError(f"newton_schulz expects fp32, bf16 or fp16 input, got {x.dtype}.")
    if x.dim() < 2:
        raise ValueError(f"newton_schulz expects matrices, got shape {tuple(x.shape)}.")
    _check_iteration(steps, coefficients, eps)
    _check_lines(x.shape)
    x = x.detach()
    shape = x.shape
    if x.is_neg():
        x = x.resolve_neg()
    if x.numel() == 0:
        return torch.empty(shape, dtype=torch.bfloat16, device=x.device)
    # orthogonalising a transpose is transposing the orthogonalised
    turned = x.stride(-1) != 1 and x.stride(-2) == 1 and x.shape[-1] > 1
    if turned:
        x = x.transpose(-1, -2)
    elif x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    x = x.reshape(-1, x.shape[-2], x.shape[-1]) if x.dim() != 3 else x
    if x.stride(-1) != 1 and x.shape[-1] > 1:  # reshape made a copy of its own layout
        x = x.contiguous()
    count, rows, cols = x.shape
    out = torch.empty((count, rows, cols), dtype=torch.bfloat16, device=x.device)
    each = _workspace_bytes((FoMatrixShape * 1)(FoMatrixShape(rows, cols, 1, 0.0)), 1)
    part = max(1, min(count, WORKSPACE_BYTES // each))
    with _native.device_guard(x.device):
        workspace = torch.empty(each * part, dtype=torch.uint8, device=x.device)
        for first in range(0, count, part):
            rc = _native.lib().fo_newton_schulz(
                x[first].data_ptr(), DTYPE_CODE[x.dtype], min(part, count - first), rows, cols, x.stride(0), x.stride(1),
                out[first].data_ptr(), int(steps), _three(coefficients), float(eps), workspace.data_ptr(),
                workspace.numel(), _native.current_stream_ptr(x.device))
            _native.check(rc, "fo_newton_schulz")
    if turned:
        out = out.transpose(-1, -2)
    return out.reshape(shape) if out.dim() != len(shape) else out


def _update_factor(adjust: Optional[str], rows: int, cols: int) -> float:
    """What multiplies the learning rate for a matrix of this shape."""
    if adjust == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    return math.sqrt(max(1.0, rows / cols))


class MuonPlan(BucketPlan):
    """Launch tables of the matrices that share a Muon step: equal shapes lie next to each other in the descriptor table."""

    _kinds = ("muon",)

    def _divide(self, tensors: Sequence[StepTensors], numels: Sequence[int], tiles_per_chunk: int) -> None:
        runs: list = []  # rows, cols, count
        for t in tensors:
            rows, cols = t.param.shape
            if runs and runs[-1][:2] == [rows, cols]:
                runs[-1][2] += 1
            else:
                runs.append([rows, cols, 1])
        # parts whose workspace keeps within the bound: (index of the first matrix, shapes)
        self._parts: list = []
        first, used, shapes = 0, 0, []
        self.workspace_bytes = 0
        for rows, cols, count in runs:
            each = _workspace_bytes((FoMatrixShape * 1)(FoMatrixShape(rows, cols, 1, 0.0)), 1)
            while count > 0:
                fit = count if each == 0 else max(0, (WORKSPACE_BYTES - used) // each)
                take = min(count, fit if fit or used else 1)
                if take == 0:
                    first = self._close(first, shapes)
                    used, shapes = 0, []
                    continue
                shapes.append((rows, cols, take))
                used += take * each
                count -= take
        self._close(first, shapes)
        self.n_chunks = sum(numels)  # an empty list launches nothing

    def _close(self, first: int, shapes: list) -> int:
        if not shapes:
            return first
        table = (FoMatrixShape * len(shapes))(*[FoMatrixShape(r, c, n, 0.0) for r, c, n in shapes])
        self.workspace_bytes = max(self.workspace_bytes, _workspace_bytes(table, len(shapes)))
        self._parts.append((first, table))
        return first + sum(n for _, _, n in shapes)

    def _launch_head(self) -> tuple:
        return (DTYPE_CODE[self.dtype], self.ecc_bytes, int(self.quantized))

    def launch(self, **scalars) -> None:
        """Enqueue the step on the current stream with the given scalars."""
        if self.n_chunks == 0:
            return
        with _native.device_guard(self.device):
            if self._dirty:
                self._upload()
            workspace = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=self.device)
            coefficients, adjust, lr = _three(scalars["coefficients"]), scalars["adjust_lr_fn"], scalars["lr"]
            for first, shapes in self._parts:
                for s in shapes:
                    if s.rows and s.cols:
                        s.lr = lr * _update_factor(adjust, s.rows, s.cols)
                rc = _native.lib().fo_muon_step(
                    self.descs_dev.data_ptr() + first * ctypes.sizeof(FoTensorDesc), shapes, len(shapes), *self._head, scalars["keep"],
                    scalars["momentum"], int(scalars["nesterov"]), scalars["steps"], coefficients, scalars["eps"],
                    workspace.data_ptr(), workspace.numel(), _native.current_stream_ptr(self.device))
                _native.check(rc, "fo_muon_step")


class FlashMuon(FlashOptimizer):
    """Muon for the hidden matrices of a network: momentum, orthogonalised by :func:`newton_schulz`, with decoupled weight decay.

    ``m <- momentum m + (1 - momentum) g``; ``u = (1 - momentum) g + momentum m`` with `nesterov`, else ``m``;
    ``p <- p (1 - lr weight_decay) - lr factor orthogonalised(u)``.  The orthogonalised update goes from the last
    product straight into the weights, it is never stored.

    Embeddings, output layers, norms and biases belong to another optimizer (:class:`FlashAdamW`).

    Args:
        params: parameters or param-group dicts; every parameter a matrix.
        lr: learning rate (default 1e-3).
        weight_decay: decoupled decay (default 0.1).
        momentum: momentum factor (default 0.95).
        nesterov: Nesterov momentum (default).
        ns_coefficients, eps, ns_steps: of the iteration.
        adjust_lr_fn: how the learning rate follows a matrix's shape: "original" (default) sqrt(max(1, rows / cols)),
            "match_rms_adamw" 0.2 sqrt(max(rows, cols)).
        quantize, compress_state_dict, master_weight_bits, check_numerics, fused: see :class:`FlashOptimizer`.

    Raises:
        ValueError: a hyper-parameter out of range, or a parameter that is no matrix.
        NotImplementedError: a sharded parameter (a shard's orthogonalisation is not the matrix's).
    """

    def __init__(
        self,
        params: Iterable[torch.Tensor],
        lr: float = 1e-3,
        weight_decay: float = 0.1,
        momentum: float = 0.95,
        nesterov: bool = True,
        ns_coefficients: Sequence[float] = DEFAULT_COEFFICIENTS,
        eps: float = DEFAULT_EPS,
        ns_steps: int = DEFAULT_STEPS,
        adjust_lr_fn: Optional[str] = None,
        quantize: bool = True,
        compress_state_dict: bool = False,
        master_weight_bits: Optional[Literal[24, 32]] = 24,
        check_numerics: bool = False,
        fused: bool = True,
    ):
        defaults = {"momentum": momentum, "weight_decay": weight_decay, "nesterov": bool(nesterov), "ns_coefficients": ns_coefficients, "eps": eps,
                    "ns_steps": ns_steps, "adjust_lr_fn": adjust_lr_fn}
        self._check_hyperparameters(defaults)
        super().__init__(
            params, lr=lr, defaults={**defaults, "ns_coefficients": tuple(ns_coefficients), "ns_steps": int(ns_steps)},
            quantize=quantize, compress_state_dict=compress_state_dict, master_weight_bits=master_weight_bits,
            check_numerics=check_numerics, fused=fused,
        )

    @staticmethod
    def _check_hyperparameters(hparams: dict[str, Any]) -> None:
        if not 0.0 <= hparams["momentum"] < 1.0:
            raise ValueError(f"Invalid momentum value: {hparams['momentum']}")
        if not 0.0 <= hparams["weight_decay"]:
            raise ValueError(f"Invalid weight_decay value: {hparams['weight_decay']}")
        if hparams["adjust_lr_fn"] not in (None, "original", "match_rms_adamw"):
            raise ValueError(f'adjust_lr_fn must be "original" or "match_rms_adamw", got {hparams["adjust_lr_fn"]!r}')
        _check_iteration(hparams["ns_steps"], hparams["ns_coefficients"], hparams["eps"])

    def add_param_group(self, param_group: dict[str, Any]) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_hyperparameters(group)
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"FlashMuon steps matrices only, got a parameter of shape {tuple(p.shape)}.")
                if max(p.shape) > MATRIX_MOST_LINES:
                    raise ValueError(f"FlashMuon steps matrices of at most {MATRIX_MOST_LINES} rows and columns, got {tuple(p.shape)}.")
        except ValueError:
            self.param_groups.pop()
            raise
        group.update(ns_coefficients=tuple(group["ns_coefficients"]), ns_steps=int(group["ns_steps"]))

    def _quantized_state_spec(self) -> dict[str, QuantizedTensorSpec]:
        return {"momentum_buffer": QuantizedTensorSpec(signed=True)}

    def _kernel_kind(self, hparams: dict[str, Any]) -> str:
        return "muon"

    def _moment_names(self, kind: str) -> tuple[Optional[str], Optional[str]]:
        return "momentum_buffer", None

    def _kernel_scalars(self, hparams: dict[str, Any], step: Optional[int]) -> dict[str, Any]:
        lr = float(hparams["lr"])
        return dict(lr=lr, keep=1.0 - lr * hparams["weight_decay"], momentum=hparams["momentum"], nesterov=hparams["nesterov"],
                    steps=hparams["ns_steps"], coefficients=tuple(hparams["ns_coefficients"]), eps=hparams["eps"],
                    adjust_lr_fn=hparams["adjust_lr_fn"])

    def _min_step_of(self, p: torch.Tensor, group: dict[str, Any]) -> float:
        # an orthogonalised rows x cols matrix has entries of about 1 / sqrt(the longer side); as with Adam's ratio, updates
        # routinely shrink to a tenth of that
        return 0.1 * _update_factor(group["adjust_lr_fn"], *p.shape) / math.sqrt(max(p.shape))

    def _plan_signature(self, hparams: dict[str, Any]) -> Any:
        return super()._plan_signature(hparams), hparams["adjust_lr_fn"]

    def _prepare_param(self, p: torch.Tensor, group: dict[str, Any]):
        if hasattr(p, "to_local"):
            raise NotImplementedError("FlashMuon does not step sharded parameters: a shard's orthogonalisation is not the matrix's.")
        return super()._prepare_param(p, group)

    def _order_bucket(self, items: list) -> list:
        return sorted(items, key=lambda item: tuple(item[0].shape))

    def _make_plan(self, key: LaunchKey, tensors: list) -> Optional[BucketPlan]:
        return MuonPlan(key.kind, key.dtype, key.ecc_bytes, key.quantized, tensors)

    def _launch_single(self, kind: str, quantized: bool, scalars: dict[str, Any], t: StepTensors) -> None:
        # one matrix on its own (gradient release): the gradient was made just now, and its table with it
        plan = MuonPlan(kind, t.param.dtype, kernels._ecc_bytes(t.ecc), quantized, [t])
        plan.launch(**scalars)
