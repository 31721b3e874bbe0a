"""Plain 64-bit forms of the operators at a language model's ends, for their tests."""
import numpy as np
import torch

M32 = 0xFFFFFFFF


def philox_block(counter, key):
    """Philox4x32, ten rounds, in whole numbers: four words of the counter, the key's two."""
    c, (k0, k1) = list(counter), key
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k0, b & M32, (a >> 32) ^ c[3] ^ k1, a & M32]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return c


def numbers(n, seed, draw=0):
    """The 32-bit numbers of n elements, as numpy uint64."""
    out = np.empty((2, -(-n // 8) * 8), dtype=np.uint64)
    low, half = np.uint64(M32), np.uint64(32)
    for which in (0, 1):
        block = np.arange(-(-n // 8), dtype=np.uint64)
        c = [block & low, block >> half, np.full_like(block, draw), np.full_like(block, which)]
        k0, k1 = seed & M32, seed >> 32 & M32
        for _ in range(10):
            a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
            c = [(b >> half) ^ c[1] ^ np.uint64(k0), b & low, (a >> half) ^ c[3] ^ np.uint64(k1), a & low]
            k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
        words = np.stack(c, axis=1)
        out[which] = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), axis=2).reshape(-1)
    return (out[0] * np.uint64(65536) + out[1])[:n]


def kept(shape, p, seed, draw=0):
    n = int(np.prod(shape)) if len(shape) else 1
    return torch.from_numpy(numbers(n, seed, draw) >= np.uint64(round(p * 2 ** 32))).reshape(shape)


def share(p):
    """What the elements that are kept are divided by."""
    return (2 ** 32 - round(p * 2 ** 32)) / 2 ** 32


def embedding_grad(ids, dy, rows, scale, padding=None):
    """(dw, sum of the terms' sizes, how many terms a row has)"""
    ids, dy = ids.reshape(-1).long(), dy.double().reshape(ids.numel(), -1)
    use = (ids >= 0) & (ids < rows)
    if padding is not None:
        use &= ids != padding
    ids, dy = ids[use], dy[use]
    dw = torch.zeros(rows, dy.size(1), dtype=torch.float64, device=dy.device).index_add_(0, ids, dy) * scale
    size = torch.zeros_like(dw).index_add_(0, ids, dy.abs()) * abs(scale)
    return dw, size, torch.bincount(ids, minlength=rows)


def head(x, w, targets, bias=None, classes=None, ignore=-100, reduction="mean", upstream=None):
    """Losses, loss and gradients in 64 bits with what bounds their terms: a dict. Rows whose target is ignored or no class are left out of all but
    the mean's count. upstream: a number, or one for each row with reduction none."""
    x, w, targets = x.double().reshape(-1, x.size(-1)), w.double(), targets.reshape(-1).long()
    classes = w.size(0) if classes is None else classes
    ignored = targets == ignore
    outside = ((targets < 0) | (targets >= classes)) & ~ignored
    live = ~ignored & ~outside
    x = torch.where(live[:, None], x, 0.0)
    b = torch.zeros(w.size(0), dtype=torch.float64, device=w.device) if bias is None else bias.double()
    wc, t = w[:classes], targets.clamp(0, classes - 1)[:, None]
    z = x @ wc.T + b[:classes]
    zt = z.gather(1, t)
    others = z.scatter(1, t, -float("inf")) - zt
    top = others.amax(1, keepdim=True).clamp(min=0)
    # log(1 + sum over the others of exp(z - zt))
    rest = (others - top).exp().sum(1, keepdim=True)
    losses = torch.where(top == 0, torch.log1p(rest), top + torch.log(rest + (-top).exp())).squeeze(1)
    losses = torch.where(ignored, 0.0, torch.where(outside, float("nan"), losses))
    lse = torch.logsumexp(z, 1, keepdim=True)
    g = (z - lse).exp()
    p_others = g.scatter(1, t, 0.0).sum(1, keepdim=True)
    g = g.scatter(1, t, -p_others)
    u = torch.as_tensor(1.0 if upstream is None else upstream, dtype=torch.float64, device=x.device).reshape(-1, 1)
    if reduction == "mean":
        u = u / (~ignored).sum() if bool((~ignored).any()) else torch.zeros_like(u)
    g = torch.where(live[:, None], g * u, 0.0)
    pad = lambda v: torch.cat((v, torch.zeros(w.size(0) - classes, *v.shape[1:], dtype=v.dtype, device=v.device)))  # noqa: E731
    out = {"losses": losses, "loss": losses.sum() / (~ignored).sum() if reduction == "mean" else losses.sum()}
    out["dx"], out["dw"], out["db"] = g @ wc, pad(g.T @ x), pad(g.sum(0))
    # (exp(-z) of the target's element has its own error: the sum of all others)
    out["dx_size"], out["dw_size"], out["db_size"] = g.abs() @ wc.abs(), pad(g.abs().T @ x.abs()), pad(g.abs().sum(0))
    out["x_size"] = (x.abs() * u.abs()).sum(0)
    out["u_size"] = float(torch.where(live[:, None], u.abs().expand(len(x), 1), 0.0).sum())
    out["z_size"] = x.abs() @ wc.abs().T + b[:classes].abs()
    out["z_most"] = float(z.abs().amax()) if z.numel() else 0.0
    return out
