"""The two ends of a language model: rows of a table by token, with a gradient by sorted tokens (``csrc/kernels/embedding.cu``), and the loss of a
head whose logits are not kept (``csrc/kernels/linear_ce.cu``)."""
from __future__ import annotations

from typing import Optional

import torch

from ._native import glue

REDUCTIONS = ("none", "mean", "sum")


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids]``: a packed tensor of shape ``[*ids.shape, width]`` in the type of ``weight`` (float32, float16 or bfloat16). Differentiable
    once in ``weight``, without gradient for row ``padding_idx``.

    ``ids``: int64 or int32 of any shape; an id outside the table makes its row not a number and adds nothing to the gradient. The gradient's sums are taken in float32 in an order
    that the ids alone decide, and rounded once: the same call gives the same bits."""
    return glue().embedding(ids, weight, scale, padding_idx)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, bias: Optional[torch.Tensor] = None, num_classes: Optional[int] = None, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """``F.cross_entropy(F.linear(x, weight, bias)[..., :num_classes], targets)`` in float32, without the logits: they are formed tile by tile and never kept.
    Differentiable once in ``x``, ``weight`` and ``bias``; the gradients' products take exponentials that are rounded to the type of ``x``.

    ``x``: ``[..., width]``, ``weight``: ``[classes, width]``, both float16 or both bfloat16 on a CUDA device (under ``torch.autocast`` they are cast to its type); ``bias``: ``[classes]``,
    of any of the three types; ``targets``: int64 or int32, ``x.shape[:-1]``. Rows of ``weight`` from ``num_classes`` on are padding: no classes, and a gradient of zero.
    ``reduction``: ``"mean"`` over the targets that are not ``ignore_index`` (not a number if all are), ``"sum"``, or ``"none"``, losses of the shape of ``targets``. A row whose
    target is ``ignore_index`` has loss 0 and adds nothing to any gradient, whatever it holds and whether or not ``ignore_index`` is a class; one whose target is no class
    has a loss that is not a number, and adds nothing either.

    With gradients, a group of tokens at a time has its exponentials in 16 bits in a workspace of up to a gigabyte (256 tokens at least); where there are several groups, the weight's
    gradient lies beside them in float32. In bfloat16 the gradients of a mean or a sum are formed along with the loss and kept until the backward pass: evaluate under ``torch.no_grad()``.
    Those of ``x`` and ``weight`` are rounded once more when the upstream gradient is not a power of two. float16 and ``"none"`` form the logits again in the backward pass. With
    float16 and ``"none"``, what is below 2^-38 of the largest ``|upstream * x|`` is lost to the weight's gradient."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"nangila: reduction must be one of {REDUCTIONS}, got {reduction!r}")
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        x, weight = x.to(dtype), weight.to(dtype)
    return glue().linear_cross_entropy(x, weight, targets, bias, num_classes, ignore_index, REDUCTIONS.index(reduction))
