"""Single import point mirroring ``flashoptim.optimizers`` of the reference: everything its users and tests
import from there is importable from here under the same name."""

from .adam import FlashAdam, FlashAdamW
from .base import (
    _BITS_TO_BYTES,
    _DTYPE_WIDTHS,
    FlashOptimizer,
    NumericsError,
    _log2_min_expressible_step_size,
)
from .cast import cast_model
from .embed import FlashEmbedding, embedding
from .kernels import (
    _fused_adam_step,
    _fused_momentum_step,
    compute_ecc_bits,
    dequantize,
    quantize,
    reconstruct_fp32_param,
)
from .lion import FlashLion
from .loss import linear_cross_entropy
from .muon import FlashMuon, newton_schulz
from .mxfp4 import (
    MXFP4Linear,
    MXFP4Tensor,
    mxfp4_dequantize,
    mxfp4_linear,
    mxfp4_matmul,
    mxfp4_quantize,
    mxfp4_quantize_both,
)
from .norm import FlashRMSNorm, rms_norm, rms_norm_mxfp4
from .release import GradientReleaseHandle, enable_gradient_release
from .sgd import FlashSGD, FlashSGDW
from .state import QuantizedTensorSpec, _MaybeQuantizedTensor

__all__ = [
    "NumericsError",
    "FlashOptimizer",
    "FlashLion",
    "FlashMuon",
    "FlashSGD",
    "FlashSGDW",
    "FlashAdam",
    "FlashAdamW",
    "GradientReleaseHandle",
    "MXFP4Linear",
    "MXFP4Tensor",
    "cast_model",
    "compute_ecc_bits",
    "enable_gradient_release",
    "mxfp4_dequantize",
    "mxfp4_linear",
    "mxfp4_matmul",
    "mxfp4_quantize",
    "mxfp4_quantize_both",
    "newton_schulz",
    "reconstruct_fp32_param",
    "FlashEmbedding",
    "FlashRMSNorm",
    "embedding",
    "linear_cross_entropy",
    "rms_norm",
    "rms_norm_mxfp4",
]
