"""flashoptim_amd: MI355X (gfx950) implementation of FlashOptim's fused optimizer-step path.

Drop-in for the reference package's public names (``/root/reference/flashoptim/__init__.py:3-33``).  The
numerical work runs in hand-written HIP kernels (``flashoptim_amd/csrc``) reached through the C ABI of
``flashoptim_amd/lib/libflashoptim_hip.so``; this package is the host-side mirror of the optimizer interface.
"""

from .optimizers import (
    FlashAdam,
    FlashAdamW,
    FlashEmbedding,
    FlashLion,
    FlashMuon,
    FlashOptimizer,
    FlashRMSNorm,
    FlashSGD,
    FlashSGDW,
    GradientReleaseHandle,
    MXFP4Linear,
    MXFP4Tensor,
    NumericsError,
    cast_model,
    compute_ecc_bits,
    embedding,
    enable_gradient_release,
    linear_cross_entropy,
    mxfp4_dequantize,
    mxfp4_linear,
    mxfp4_matmul,
    mxfp4_quantize,
    mxfp4_quantize_both,
    newton_schulz,
    reconstruct_fp32_param,
    rms_norm,
    rms_norm_mxfp4,
)

__version__ = "0.1.0"

__all__ = [
    "FlashAdam",
    "FlashAdamW",
    "FlashEmbedding",
    "FlashLion",
    "FlashMuon",
    "FlashOptimizer",
    "FlashRMSNorm",
    "FlashSGD",
    "FlashSGDW",
    "GradientReleaseHandle",
    "MXFP4Linear",
    "MXFP4Tensor",
    "NumericsError",
    "cast_model",
    "compute_ecc_bits",
    "embedding",
    "enable_gradient_release",
    "linear_cross_entropy",
    "mxfp4_dequantize",
    "mxfp4_linear",
    "mxfp4_matmul",
    "mxfp4_quantize",
    "mxfp4_quantize_both",
    "newton_schulz",
    "reconstruct_fp32_param",
    "rms_norm",
    "rms_norm_mxfp4",
]
