"""Updates made orthogonal by Newton-Schulz steps, and the Muon step on them (``csrc/kernels/orthogonalize.cu``).

With ``X = U / max(|U|, eps)`` (Frobenius norm), each step takes ``A = X X^T`` on the shorter side and ``X <- a X + (b A + c A^2) X``, which moves
every singular value towards one. The products' operands are float16, accumulated in float32, and X is kept to 22 bits between the steps (in float32 where a matrix
has a side of at most 128 and the other of at most 24 * 128): with the default coefficients that is within 0.5e-3 to 1.7e-3 (relative, 2-norm) of the formula in exact
arithmetic, noise being the worst, and the result's rounding to bfloat16 adds 1.7e-3: about 2e-3 in all. CPU tensors take the formula in float32.

Larger matrices take a workspace for the call: 6 bytes an element of the matrices that go together and 4 an element of a square of their shorter side. As many go together
as that leaves below a gigabyte, one at least. It comes from PyTorch's allocator and goes back to it.

The update is Muon's (K. Jordan and others, 2024), with their coefficients; the ``"rms"`` scale is that of J. Liu and others (2025).
"""
from __future__ import annotations

import math
from typing import List, Sequence, Tuple, Union

import torch

from ._native import glue

#: Moves singular values from 1.6e-3 to 1 into 0.68 to 1.21 within five steps (1e-3 to 0.47).
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_STEPS = 32
SCALES = ("spectral", "rms", None)
_Coefficients = Union[Tuple[float, float, float], Sequence[Tuple[float, float, float]]]


def _schedule(steps: int, coefficients: _Coefficients) -> List[float]:
    if not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"nangila: steps must be 1 to {MAX_STEPS}, got {steps}")
    rows = list(coefficients)
    if len(rows) == 3 and all(isinstance(v, (int, float)) for v in rows):
        rows = [tuple(rows)] * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError(f"nangila: coefficients must be three numbers, or three for each of the {steps} steps")
    flat = [float(v) for r in rows for v in r]
    if not all(math.isfinite(v) for v in flat):
        raise ValueError("nangila: coefficients must be finite")
    return flat


#: An update of zeros is divided by eps and multiplied by up to 256, in float32.
MIN_EPS = 1e-36


def _check_eps(eps: float) -> None:
    if not (math.isfinite(eps) and eps >= MIN_EPS):
        raise ValueError(f"nangila: eps must be finite and at least {MIN_EPS}, got {eps}")


def _plain(u: torch.Tensor, flat: List[float], eps: float) -> torch.Tensor:
    """The formula in float32."""
    x = u.float()
    # times a power of two that brings the largest value near one: squares of any update then fit into float32
    by = torch.ldexp(torch.ones((), device=x.device), -torch.frexp(x.abs().amax()).exponent.clamp(-126, 126))
    x = x * by
    x = x / torch.maximum(torch.linalg.vector_norm(x), eps * by)
    tall = x.size(0) > x.size(1)
    x = x.mT if tall else x
    for i in range(0, len(flat), 3):
        gram = x @ x.mT
        x = flat[i] * x + (flat[i + 1] * gram + flat[i + 2] * (gram @ gram)) @ x
    return x.mT if tall else x


@torch.no_grad()
def orthogonalize(update: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5, coefficients: _Coefficients = COEFFICIENTS,
                  eps: float = 1e-7) -> Union[torch.Tensor, List[torch.Tensor]]:
    """``update`` with its singular values moved towards one, in bfloat16 (the accuracy of the steps warrants no more). A matrix, a stack
    ``[count, rows, cols]``, or a list of matrices of any shapes, types and devices: those that agree go through the kernels together, and
    their results share one allocation. ``coefficients``: ``(a, b, c)``, or one such triple for each step; they have to keep the singular values
    below about two. No gradient flows through it."""
    flat = _schedule(steps, coefficients)
    _check_eps(eps)
    if isinstance(update, torch.Tensor) and update.dim() != 3:
        many = [update]
    elif isinstance(update, torch.Tensor) and update.size(0) == 0:
        glue().orthogonalize([update.new_empty(update.shape[1:], device="cpu")], flat, eps)  # its checks
        return update.new_empty(update.shape, dtype=torch.bfloat16)
    else:
        many = list(update)
    if not all(isinstance(t, torch.Tensor) for t in many):
        raise TypeError("nangila: updates must be tensors")
    results = glue().orthogonalize(many, flat, eps)
    results = [_plain(t, flat, eps).to(torch.bfloat16) if r is None else r for t, r in zip(many, results)]
    if not isinstance(update, torch.Tensor):
        return results
    if update.dim() != 3:
        return results[0]
    # (the results of a stack on a GPU lie one behind the other)
    return torch.stack(results) if not update.is_cuda else results[0].as_strided(update.shape, (update.size(1) * update.size(2), update.size(2), 1))


def update_scale(rows: int, cols: int, scale: Union[str, None]) -> float:
    """What a ``rows x cols`` update is multiplied by: ``"spectral"``: ``sqrt(max(1, rows / cols))``; ``"rms"``: ``0.2 sqrt(max(rows, cols))``, the size of
    an AdamW update, so that its learning rate and weight decay carry over; None: 1."""
    if scale == "spectral":
        return math.sqrt(max(1.0, rows / cols))
    if scale == "rms":
        return 0.2 * math.sqrt(max(rows, cols))
    if scale is None:
        return 1.0
    raise ValueError(f"nangila: scale must be one of {SCALES}, got {scale!r}")


@torch.no_grad()
def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], lr: float, momentum: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5, coefficients: _Coefficients = COEFFICIENTS, eps: float = 1e-7,
              scale: Union[str, None] = "rms") -> None:
    """One Muon step in place, for matrices of any shapes::

        momenta <- momentum * momenta + grads
        update   = orthogonalize(grads + momentum * momenta)      (momenta alone without nesterov)
        params  <- params * (1 - lr * weight_decay) - lr * update_scale * update

    ``momenta`` are float32 (zeros before the first step). Everything is packed; no two of ``params`` and ``momenta`` share memory, with one another
    or with ``grads``. Matrices of one shape and type go through the kernels together; the parameters are updated in the last product's epilogue.
    ``lr`` and the others are plain numbers: a captured CUDA graph keeps the ones that it was captured with."""
    flat = _schedule(steps, coefficients)
    _check_eps(eps)
    for name, v in (("lr", lr), ("momentum", momentum), ("weight_decay", weight_decay)):
        if not (math.isfinite(v) and v >= 0):
            raise ValueError(f"nangila: {name} must be finite and not negative, got {v}")
    update_scale(1, 1, scale)
    params, grads, momenta = list(params), list(grads), list(momenta)
    for i in glue().muon_step(params, grads, momenta, flat, eps, momentum, nesterov, lr, weight_decay, SCALES.index(scale)):
        p, g, m = params[i], grads[i], momenta[i]
        m.mul_(momentum).add_(g)
        u = m * momentum + g if nesterov else m
        p.copy_(p.float() * (1.0 - lr * weight_decay) - lr * update_scale(p.size(0), p.size(1), scale) * _plain(u, flat, eps))
