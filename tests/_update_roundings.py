"""The Newton-Schulz steps with the roundings that the kernels state, in 64 bits otherwise: what they have to come close to, whatever the formula gives.

A product's operands X, A and B are float16. X itself is kept in two halves (``lo``: 22 bits) or, where a matrix stays on the SMs, in float32. In the last step
the polynomial is taken around one.
"""
import torch


def scale_of(m, n):
    s = 1.0
    while s * s < max(m, n):
        s *= 2.0
    return s


def stays_on_the_sms(m, n):
    return min(m, n) <= 128 and max(m, n) <= 24 * 128


def rounded(u, coefficients, eps, low=True, shifted=True, operand=torch.float16, product=torch.float64):
    """The result before its own rounding. ``low``: X has its low half; ``shifted``: the last step's form; ``operand``: what the products take; ``product``: in
    what they are summed up."""
    m, n = u.shape
    s, keep = scale_of(m, n), stays_on_the_sms(m, n)
    x = u.double()
    x = x / torch.linalg.matrix_norm(x).clamp(min=eps) * s
    tall = m > n
    x = x.T.contiguous() if tall else x

    def as_operand(v):
        return v.to(operand).to(product)

    def kept(v):
        hi = v.to(torch.float16).double()
        if not low:
            return hi
        return v.float().double() if keep else hi + ((v - hi) * 2048.0).to(torch.float16).double() / 2048.0

    for i, (a, b, c) in enumerate(coefficients):
        shift = -(b + c) if shifted and i == len(coefficients) - 1 else 0.0
        x = kept(x)
        h = as_operand(x)
        gram = as_operand((h @ h.T).double() / (s * s))
        poly = b * gram.double() + c * (gram @ gram).double()
        poly.diagonal().add_(shift)
        x = (a - shift) * x + (as_operand(poly) @ h).double()
    x = x / s
    return x.T.contiguous() if tall else x
