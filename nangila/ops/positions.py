"""Rotary positions (``csrc/kernels/rotary.cu``): pairs of columns of q and k turned by the angles of their positions (J. Su and others, 2021).

The scalings for long contexts are published ones: positions divided (S. Chen and others, 2023), theta raised, and a blend of both by the pair's speed (B. Peng and
others, 2023), with their constants as defaults.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from ._native import glue

LAYOUTS = ("interleaved", "half")
SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_table(seq: int, rot: int, theta: float = 10000.0, device: Union[torch.device, str, None] = None, scaling: Optional[str] = None,
                 factor: float = 1.0, original_seq: Optional[int] = None, beta_fast: float = 32.0, beta_slow: float = 1.0) -> torch.Tensor:
    """float32 ``[seq, rot / 2, 2]``: cosine and sine of ``position * theta^(-2i / rot)``, the angles formed in 64 bits.

    For contexts ``factor`` times as long as the model was trained on:

    * ``"linear"``: positions divided by ``factor``;
    * ``"ntk"``: ``theta`` times ``factor^(rot / (rot - 2))``, which leaves the fastest pair alone and slows the slowest by ``factor``;
    * ``"yarn"``: pairs that make more than ``beta_fast`` turns over ``original_seq`` positions are left alone, those that make fewer than
      ``beta_slow`` are slowed by ``factor``, linearly in between by the pair's index; cosine and sine are multiplied by ``0.1 ln(factor) + 1``.
    """
    if seq < 1:
        raise ValueError(f"nangila: seq must be positive, got {seq}")
    if rot < 2 or rot % 2:
        raise ValueError(f"nangila: rot must be even and positive, got {rot}")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError(f"nangila: theta must be positive, got {theta}")
    if scaling not in SCALINGS:
        raise ValueError(f"nangila: scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (math.isfinite(factor) and factor >= 1) or (scaling is None and factor != 1):
        raise ValueError(f"nangila: factor must be at least 1, and is given with a scaling, got {factor}")
    half = rot // 2
    index = torch.arange(half, device=device, dtype=torch.float64)
    magnitude = 1.0
    if scaling == "ntk":
        if rot == 2 and factor != 1:
            raise ValueError("nangila: ntk scaling needs rot of 4 or more")
        theta = theta * factor ** (rot / (rot - 2)) if rot > 2 else theta
    inv = theta ** (-2.0 * index / rot)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if original_seq is None or original_seq < 1:
            raise ValueError("nangila: yarn scaling needs original_seq, the length that the model was trained on")
        if theta == 1.0 or not beta_fast > beta_slow > 0:
            raise ValueError("nangila: yarn scaling needs theta other than 1 and beta_fast > beta_slow > 0")

        def pair_with(turns: float) -> float:  # index of the pair that makes so many turns over original_seq
            return rot * math.log(original_seq / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = max(math.floor(pair_with(beta_fast)), 0), min(math.ceil(pair_with(beta_slow)), rot - 1)
        slowed = ((index - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        inv = inv * (1 - slowed) + inv / factor * slowed
        magnitude = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(seq, device=device, dtype=torch.float64)[:, None] * inv
    return (torch.stack((angle.cos(), angle.sin()), dim=-1) * magnitude).float()


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], table: torch.Tensor, positions: Optional[torch.Tensor] = None,
           layout: str = "interleaved") -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``q`` and ``k`` (``[batch, seq, heads, head_dim]``, each with its own number of heads, any strides) with their first
    ``2 * table.size(1)`` columns turned and the others as they are: new packed tensors, ``(q, k)``, or ``q`` alone where ``k`` is None.

    ``layout``: ``"interleaved"`` turns columns ``(2i, 2i + 1)`` together, ``"half"`` columns ``(i, i + rot / 2)``. ``positions``: int64 or int32,
    ``[seq]`` or ``[batch, seq]``, rows of ``table``; None: ``0 .. seq - 1``. A position outside the table makes the turned columns of its
    token not a number. Differentiable once in ``q`` and ``k``; computed in float32 and rounded once."""
    if layout not in LAYOUTS:
        raise ValueError(f"nangila: layout must be one of {LAYOUTS}, got {layout!r}")
    out = glue().rotary(q, k, table, positions, layout == "half")
    return out[0] if k is None else out
