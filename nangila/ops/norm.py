"""RMS norm of the last dimension, alone, with the residual's addition before it, or with an output in 8 bits
(``csrc/kernels/rms_norm.cu``).

float32, float16 and bfloat16 rows of up to 32768 values; the weight may have another of the three types. Sums are float32: the squares of a
row have to fit.
CUDA tensors take one kernel forward and two backward; CPU tensors take the formula in torch operations.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._native import glue


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in the type of ``x``. Differentiable once in ``x`` and ``weight``."""
    return glue().rms_norm(x, weight, eps)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(y, h)`` with ``h = x + residual``, rounded to their type, and ``y = rms_norm(h)``: a block's norm in one pass. The gradients of both
    outputs meet in one kernel; ``x`` and ``residual`` get the same one."""
    return glue().add_rms_norm(x, residual, weight, eps)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: Optional[torch.Tensor] = None,
                 group: Optional[int] = None) -> Tuple[torch.Tensor, ...]:
    """``(q, scale)``, or ``(q, scale, h)`` with a residual: the norm in float8_e4m3fn, ``q * scale`` being its values. ``scale`` (float32) is
    ``max(|y|, 1e-12) / 448`` over the row, or over each ``group`` of 128 columns; it has the shape of ``x`` with one value for the row, or for
    each group, in the last dimension. A row or group that is not all finite is not a number throughout. No gradient: inputs that require
    one are refused unless gradients are off."""
    q, scale, h = glue().rms_norm_fp8(x, weight, eps, residual, 0 if group is None else group)
    return (q, scale) if h is None else (q, scale, h)
