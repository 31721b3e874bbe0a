"""How far the gradients of the head's loss may be off, for any number of tokens, classes and columns."""
import torch

from tests._model_ops import half_step, rounding
from tests.test_linear_ce_kernel_gpu import U, exp_error


def check_grads_anywhere(grads, want, x, w, d, dtype, also=0.0, results=1):
    """Each element of E is rounded once, by half a step. The target's rounding is divided out of the row's factor, which moves all other elements of the row by as much as that: a second half
    step. Where a class, a column or a row has many terms both average out; where it has one or two they do not, so each term has them here. dw has a third one for x times the factor.
    (With h half a step: (1 + h)(1 + h)(1 + h) - 1 <= 3 h (1 + 2 h) for h <= 2^-8.) ``also``: a further absolute error of dw; ``results``: how often a result is rounded."""
    rows, n = w.size(0), x.numel() // d
    hs, exp = half_step(dtype), exp_error(want, d, rows)
    tiny = 2.0 ** -39 if dtype == torch.float16 else 2.0 ** -100  # fp16's subnormal steps under 2^15
    last = lambda name, t: results * 1.01 * rounding(want[name], t)  # noqa: E731
    allowed = {
        "dx": want["dx_size"] * (2 * hs * (1 + 2 * hs) + exp + (rows / 16 + 17) * 2.0 ** -22 + 8 * U) + tiny * want["u_size"] * w.double().abs().sum(0) + last("dx", dtype),
        "dw": want["dw_size"] * (3 * hs * (1 + 2 * hs) + exp + (n / 8 + 25) * 2.0 ** -22 + 8 * U) + tiny * want["x_size"] + last("dw", dtype) + also,
    }
    if len(grads) > 2:
        allowed["db"] = want["db_size"] * (2 * hs * (1 + 2 * hs) + exp + (n + 8) * U) + tiny * want["u_size"] + last("db", grads[2].dtype)
    for got, (name, tol) in zip(grads, allowed.items()):
        over = (got.double().reshape(want[name].shape) - want[name]).abs() - tol
        assert bool((over <= 0).all()), (name, over.max())
