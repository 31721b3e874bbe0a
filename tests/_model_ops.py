"""Plain 64-bit forms of the model and update operators, for their tests."""
import torch


def norm(h, w, eps):
    h, w = h.double(), w.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w


def norm_grads(h, w, eps, dy=None, dh=None):
    """(dx, dw, what bounds dx's terms, what bounds dw's) from the formula."""
    h, w = h.double().reshape(-1, h.size(-1)), w.double()
    dy = torch.zeros_like(h) if dy is None else dy.double().reshape(h.shape)
    dh = torch.zeros_like(h) if dh is None else dh.double().reshape(h.shape)
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit = h * rstd
    g = dy * w
    dx = dh + rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
    size = dh.abs() + rstd * (g.abs() + unit.abs() * (g * unit).abs().mean(-1, keepdim=True))
    return dx, (dy * unit).sum(0), size, (dy * unit).abs().sum(0)


def turned(x, table, positions, layout, inverse=False):
    """(result, what bounds its terms): positions [batch or 1, seq]."""
    n = table.size(1)
    ang = table.double()[positions]  # [b, t, n, 2]
    c, s = ang[..., 0].unsqueeze(2), ang[..., 1].unsqueeze(2) * (-1.0 if inverse else 1.0)
    f = x.double()
    out, size = f.clone(), f.abs()
    ia = torch.arange(n, device=x.device) * (2 if layout == "interleaved" else 1)
    ib = ia + (1 if layout == "interleaved" else n)
    a, b = f[..., ia], f[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia], size[..., ib] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return out, size


def orthogonal(u, steps, coefficients, eps):
    x = u.double()
    x = x / torch.linalg.matrix_norm(x).clamp(min=eps)
    rows = [coefficients] * steps if isinstance(coefficients[0], (int, float)) else coefficients
    flip = x.size(0) > x.size(1)
    x = x.T if flip else x
    for a, b, c in rows:
        s = x @ x.T
        x = a * x + b * (s @ x) + c * (s @ (s @ x))
    return x.T if flip else x


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(want, dtype):
    """Half a step of `dtype` at each value: of the value, or fixed among the subnormals (fp16 reaches them)."""
    return want.abs() * half_step(dtype) + torch.finfo(dtype).tiny * half_step(dtype)
