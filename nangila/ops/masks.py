"""Dropout whose mask follows from a seed and is never stored (``csrc/kernels/dropout.cu``): the gradient makes it again.

Element ``i`` (in the order of a packed tensor) is kept where its 32-bit number reaches ``round(p 2^32)``. The numbers come from Philox4x32 with ten rounds
(J. Salmon and others, 2011), its key the seed: the upper halves of elements ``8 b .. 8 b + 7`` are the 128 bits of the counter ``(b, draw, 0)``, the lower halves
those of ``(b, draw, 1)``. Tensors on the CPU get the same masks.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from ._native import glue


def dropout(x: torch.Tensor, p: float = 0.5, seed: Union[int, torch.Tensor, None] = None, residual: Optional[torch.Tensor] = None, draw: int = 0) -> torch.Tensor:
    """``x`` with each element set to zero with probability ``p`` and the others divided by ``1 - p``, plus ``residual`` where one is given (of the
    shape and type of ``x``): a new packed tensor, computed in float32 and rounded once. float32, float16 and bfloat16.

    ``seed``: a number below 2^64, or one int64 on the device of ``x``, which is read when the kernel runs, forward and backward: a captured graph draws other masks
    when it is changed between replays. None: taken from PyTorch's default CPU generator (``torch.manual_seed``), not while a graph is captured.
    ``draw``, below 2^32, tells apart masks of one seed. Data-parallel ranks need seeds of their own, or they drop the same elements. ``p`` is held
    in 2^-32, and the factor goes by what is held. What is dropped may be infinite or not a number. Differentiable once in ``x`` and ``residual``."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"nangila: p must be 0 to 1, got {p}")
    if not 0 <= draw < 2 ** 32:
        raise ValueError(f"nangila: draw must be 0 to 2^32 - 1, got {draw}")
    number = None
    if seed is not None and not isinstance(seed, torch.Tensor):
        if not 0 <= seed < 2 ** 64:
            raise ValueError(f"nangila: seed must be 0 to 2^64 - 1, got {seed}")
        number, seed = (seed if seed < 2 ** 63 else seed - 2 ** 64), None
    return glue().dropout(x, residual, round(p * 2 ** 32), draw, number, seed)
