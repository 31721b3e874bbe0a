"""What the model and update operators are timed on: norms, rotary positions, and updates made orthogonal.

Kinds
  norm     ``rms_norm`` / ``add_rms_norm``, forward alone or with the gradients
  norm8    ``rms_norm_fp8``: the norm with an output in 8 bits and its scales
  rotary   ``rotary``, forward alone or with the gradients
  orth     ``orthogonalize`` of a list of matrices of one shape
  muon     ``muon_step``: momentum, orthogonalisation and the parameters' update

The plain forms compute in 32 bits and round once at the end.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NORM_FLOOR = 1e-7
LR, MOMENTUM, WEIGHT_DECAY = 0.02, 0.95, 0.1


def listed():
    return [
        # one token of a decoder of width 2048 going through a block's second norm: latency
        {"name": "norm_token", "kind": "norm", "rows": 1, "d": 2048, "dtype": "bf16", "residual": True, "backward": False},
        # the decoder's training step, 4 x 2048 tokens: a block's second norm with the residual's addition and all gradients
        {"name": "norm_train_bf16", "kind": "norm", "rows": 8192, "d": 2048, "dtype": "bf16", "residual": True, "backward": True},
        # a width that no vector divides, without a residual, in single precision
        {"name": "norm_odd_fp32", "kind": "norm", "rows": 4099, "d": 1001, "dtype": "fp32", "residual": False, "backward": True},
        # a wide layer's input in 8 bits with one scale for each 128 columns, ragged number of rows
        {"name": "norm_8bit_groups", "kind": "norm8", "rows": 8191, "d": 5632, "dtype": "bf16", "residual": True, "group": 128},
        # one new token of each of 32 sequences at far positions, half layout, shared key heads
        {"name": "rotary_tokens", "kind": "rotary", "batch": 32, "seq": 1, "heads": 16, "kv": 4, "d": 128, "rot": 128, "layout": "half", "given": True,
         "dtype": "bf16", "backward": False},
        # the decoder's training step: 16 heads of 128, neighbours turned together, with the gradients
        {"name": "rotary_train_bf16", "kind": "rotary", "batch": 4, "seq": 2048, "heads": 16, "kv": 16, "d": 128, "rot": 128, "layout": "interleaved",
         "given": False, "dtype": "bf16", "backward": True},
        # a long prompt: part of the head is turned, key heads shared, positions given
        {"name": "rotary_long_part", "kind": "rotary", "batch": 1, "seq": 32749, "heads": 32, "kv": 8, "d": 128, "rot": 64, "layout": "half", "given": True,
         "dtype": "fp16", "backward": False},
        # GPT-2 small's output projection on its own
        {"name": "orth_768", "kind": "orth", "m": 768, "n": 768, "count": 1, "dtype": "fp32"},
        # odd sizes, taller than wide
        {"name": "orth_odd_tall", "kind": "orth", "m": 2051, "n": 517, "count": 3, "dtype": "fp32"},
        # a wide layer of a large model
        {"name": "orth_4096x16384", "kind": "orth", "m": 4096, "n": 16384, "count": 1, "dtype": "bf16"},
        # the MLPs of a small model's blocks: many small matrices in one step
        {"name": "muon_small", "kind": "muon", "m": 352, "n": 128, "count": 24, "dtype": "bf16"},
        # the attention projections of four blocks of the decoder
        {"name": "muon_2048", "kind": "muon", "m": 2048, "n": 2048, "count": 16, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm8", "rotary", "orth", "muon"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if kind in ("norm", "norm8"):
        d = _log(rng, 32, 16384)
        rows = _log(rng, 1, max(1, 100_000_000 // (SIZE[dtype] * d)))
        if kind == "norm":
            return {"kind": kind, "rows": rows, "d": d, "dtype": dtype, "residual": rng.random() < 0.6, "backward": rng.random() < 0.6}
        group = rng.choice([0, 128])
        if group:
            d = max(128, d // 128 * 128)
        return {"kind": kind, "rows": rows, "d": d, "dtype": dtype, "residual": rng.random() < 0.6, "group": group}
    if kind == "rotary":
        d = rng.choice([32, 64, 80, 96, 128, 128, 256])
        rot = rng.choice([d, d, d // 2, d // 4 // 2 * 2])
        heads = rng.choice([4, 8, 12, 16, 32])
        kv = rng.choice([heads, heads // 2, heads // 4])
        batch = _log(rng, 1, 64)
        seq = _log(rng, 1, max(1, 200_000_000 // (SIZE[dtype] * batch * (heads + kv) * d)))
        return {"kind": kind, "batch": batch, "seq": seq, "heads": heads, "kv": kv, "d": d, "rot": rot, "layout": rng.choice(["half", "interleaved"]),
                "given": rng.random() < 0.5, "dtype": dtype, "backward": rng.random() < 0.5}
    m, n = _log(rng, 32, 4096), _log(rng, 32, 4096)
    count = _log(rng, 1, max(1, min(32, 16 * 2048 ** 2 // (m * n))))
    if kind == "orth":
        return {"kind": kind, "m": m, "n": n, "count": count, "dtype": dtype}
    return {"kind": kind, "m": m, "n": n, "count": count, "dtype": rng.choice(["bf16", "bf16", "fp16"])}


# ---- inputs ----------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _activations(g, dtype, *shape):
    """Values of a residual stream: columns of different spread."""
    spread = torch.exp(0.5 * torch.randn(shape[-1], device="cuda", generator=g))
    return (torch.randn(*shape, device="cuda", generator=g) * spread).to(dtype)


def _gradients(g, dtype, m, n, count):
    """Gradients of linear layers: singular values that fall off by a power law, and the noise of a batch."""
    k = min(m, n)
    fall = (1.0 + torch.arange(k, device="cuda")).pow(-0.5)
    left = torch.randn(count, m, k, device="cuda", generator=g) * fall
    grads = left @ torch.randn(count, k, n, device="cuda", generator=g)
    grads += torch.randn(count, m, n, device="cuda", generator=g)
    return [v.clone() for v in (grads * 1e-4).to(dtype).unbind(0)]


def _table(seq, rot, theta=10000.0):
    """Cosine and sine of every position's angles: [seq, rot / 2, 2]."""
    inv = theta ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(seq, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack((angle.cos(), angle.sin()), dim=-1).float()


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = dict(case)
    if kind in ("norm", "norm8"):
        rows, d = case["rows"], case["d"]
        wants = bool(case.get("backward"))
        state["x"] = _activations(g, dtype, rows, d).requires_grad_(wants)
        state["r"] = _activations(g, dtype, rows, d).requires_grad_(wants) if case["residual"] else None
        state["w"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=g)).to(dtype).requires_grad_(wants)
        if wants:
            state["dy"] = _activations(g, dtype, rows, d)
            state["dh"] = _activations(g, dtype, rows, d) if case["residual"] else None
    elif kind == "rotary":
        b, t, d = case["batch"], case["seq"], case["d"]
        wants = case["backward"]
        state["q"] = torch.randn(b, t, case["heads"], d, device="cuda", generator=g).to(dtype).requires_grad_(wants)
        state["k"] = torch.randn(b, t, case["kv"], d, device="cuda", generator=g).to(dtype).requires_grad_(wants)
        reach = t + 4096 if case["given"] else t  # the table reaches further than this prompt
        state["table"] = _table(reach, case["rot"])
        state["positions"] = None
        if case["given"]:
            start = torch.randint(0, reach - t + 1, (b, 1), device="cuda", generator=g)
            state["positions"] = start + torch.arange(t, device="cuda")
        if wants:
            state["dq"] = torch.randn(b, t, case["heads"], d, device="cuda", generator=g).to(dtype)
            state["dk"] = torch.randn(b, t, case["kv"], d, device="cuda", generator=g).to(dtype)
    else:
        m, n, count = case["m"], case["n"], case["count"]
        state["grads"] = _gradients(g, dtype, m, n, count)
        if kind == "muon":
            state["momenta"] = [v.float() for v in _gradients(g, torch.float32, m, n, count)]
            state["params"] = [(0.02 * torch.randn(m, n, device="cuda", generator=g)).to(dtype) for _ in range(count)]
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from nangila import ops

    kind = s["kind"]
    if kind == "norm":
        if s["residual"]:
            y, h = ops.add_rms_norm(s["x"], s["r"], s["w"], eps=EPS)
            if not s["backward"]:
                return {"y": y, "h": h}
            dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["r"], s["w"]), (s["dy"], s["dh"]))
            return {"y": y, "h": h, "dx": dx, "dr": dr, "dw": dw}
        y = ops.rms_norm(s["x"], s["w"], eps=EPS)
        if not s["backward"]:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if kind == "norm8":
        group = s["group"] or None
        if s["residual"]:
            q, scale, h = ops.rms_norm_fp8(s["x"], s["w"], eps=EPS, residual=s["r"], group=group)
            return {"q": q, "scale": scale, "h": h}
        q, scale = ops.rms_norm_fp8(s["x"], s["w"], eps=EPS, group=group)
        return {"q": q, "scale": scale}
    if kind == "rotary":
        q, k = ops.rotary(s["q"], s["k"], s["table"], positions=s["positions"], layout=s["layout"])
        if not s["backward"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if kind == "orth":
        return ops.orthogonalize(s["grads"], steps=STEPS, coefficients=COEFFICIENTS, eps=NORM_FLOOR)
    ops.muon_step(s["params"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM, weight_decay=WEIGHT_DECAY, nesterov=True, steps=STEPS,
                  coefficients=COEFFICIENTS, eps=NORM_FLOOR, scale="spectral")
    return {"params": s["params"], "momenta": s["momenta"]}


@torch.no_grad()
def _plain(s):
    kind = s["kind"]
    if kind == "norm":
        return _plain_norm(s)
    if kind == "norm8":
        return _plain_norm8(s)
    if kind == "rotary":
        return _plain_rotary(s)
    if kind == "orth":
        return list(_plain_orth(torch.stack(s["grads"]).float()).to(torch.bfloat16).unbind(0))
    momenta = MOMENTUM * torch.stack(s["momenta"]) + torch.stack(s["grads"]).float()
    updates = _plain_orth(torch.stack(s["grads"]).float() + MOMENTUM * momenta)
    rate = LR * math.sqrt(max(1.0, s["m"] / s["n"]))
    params = torch.stack(s["params"]).float() * (1 - LR * WEIGHT_DECAY) - rate * updates
    torch._foreach_copy_(s["momenta"], list(momenta.unbind(0)))
    torch._foreach_copy_(s["params"], list(params.unbind(0)))
    return {"params": s["params"], "momenta": s["momenta"]}


def _plain_norm(s):
    x, w = s["x"], s["w"].float()
    dtype = x.dtype
    h = x if s["r"] is None else (x.float() + s["r"].float()).to(dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.square().mean(-1, keepdim=True) + EPS)
    unit = hf * rstd
    out = {"y": (unit * w).to(dtype)}
    if s["r"] is not None:
        out["h"] = h
    if s["backward"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(dtype)
        if s["r"] is not None:
            out["dr"] = out["dx"]
        out["dw"] = (dy * unit).sum(0).to(dtype)
    return out


def _plain_norm8(s):
    x = s["x"]
    h = x if s["r"] is None else (x.float() + s["r"].float()).to(x.dtype)
    hf = h.float()
    f = hf * torch.rsqrt(hf.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
    f = f.view(s["rows"], -1, s["group"] or s["d"])
    scale = f.abs().amax(-1).clamp(min=1e-12) / 448.0
    q = (f / scale[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(s["rows"], s["d"])
    out = {"q": q, "scale": scale}
    if s["r"] is not None:
        out["h"] = h
    return out


def _turn(x, table, layout, sign):
    """Each pair of the first columns turned by its position's angle; the columns after them as they are."""
    half = table.size(-2)
    c, sn = table[..., 0].unsqueeze(-2), sign * table[..., 1].unsqueeze(-2)
    xf = x.float()
    if layout == "half":
        a, b = xf[..., :half], xf[..., half:2 * half]
        turned = torch.cat((a * c - b * sn, a * sn + b * c), dim=-1)
    else:
        a, b = xf[..., 0:2 * half:2], xf[..., 1:2 * half:2]
        turned = torch.stack((a * c - b * sn, a * sn + b * c), dim=-1).flatten(-2)
    return torch.cat((turned, xf[..., 2 * half:]), dim=-1).to(x.dtype)


def _plain_rotary(s):
    table = s["table"][:s["seq"]] if s["positions"] is None else s["table"][s["positions"]]
    out = {"q": _turn(s["q"], table, s["layout"], 1.0), "k": _turn(s["k"], table, s["layout"], 1.0)}
    if s["backward"]:
        out["dq"] = _turn(s["dq"], table, s["layout"], -1.0)
        out["dk"] = _turn(s["dk"], table, s["layout"], -1.0)
    return out


def _plain_orth(u):
    """[count, m, n] in 32 bits: the Newton-Schulz steps on the shorter side."""
    a, b, c = COEFFICIENTS
    x = u / u.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=NORM_FLOOR)
    if u.size(-2) > u.size(-1):
        x = x.mT.contiguous()
    for _ in range(STEPS):
        gram = x @ x.mT
        x = torch.baddbmm(x, b * gram + c * (gram @ gram), x, beta=a)
    return x.mT if u.size(-2) > u.size(-1) else x


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("norm", "norm8"):
        w = s["w"].double()
        total = s["x"].double() + (s["r"].double() if case["residual"] else 0.0)
        h = total.to(s["x"].dtype).double()  # what is normalised is the sum as it is kept
        root = torch.sqrt(torch.linalg.vecdot(h, h) / case["d"] + EPS)[:, None]
        y = h / root * w
        if kind == "norm8":
            parts = y.reshape(case["rows"], -1, case["group"] or case["d"])
            scale = torch.maximum(parts.max(-1).values, -parts.min(-1).values) / 448
            out = {"q": (parts / scale[..., None]).reshape(case["rows"], case["d"]), "scale": scale}
        else:
            out = {"y": y}
        if case["residual"]:
            out["h"] = total
        if case.get("backward"):
            dy = s["dy"].double()
            # y = h w / root, and d root / dh = h / (d root)
            dx = dy * w / root - h * (torch.linalg.vecdot(dy * w, h)[:, None] / (case["d"] * root ** 3))
            if case["residual"]:
                dx = dx + s["dh"].double()
                out["dr"] = dx
            out["dx"] = dx
            out["dw"] = torch.einsum("rd,rd->d", dy, h / root)
        return out
    if kind == "rotary":
        half = case["rot"] // 2
        turns = torch.view_as_complex(s["table"].double().contiguous())
        turns = (turns[:case["seq"]] if s["positions"] is None else turns[s["positions"]]).unsqueeze(-2)

        def turned(x, by):
            x = x.double()
            head, rest = x[..., :2 * half], x[..., 2 * half:]
            if case["layout"] == "half":
                z = torch.complex(head[..., :half], head[..., half:]) * by
                return torch.cat((z.real, z.imag, rest), dim=-1)
            z = torch.view_as_complex(head.reshape(*head.shape[:-1], half, 2).contiguous()) * by
            return torch.cat((torch.view_as_real(z).flatten(-2), rest), dim=-1)

        out = {"q": turned(s["q"], turns), "k": turned(s["k"], turns)}
        if case["backward"]:
            out["dq"], out["dk"] = turned(s["dq"], turns.conj()), turned(s["dk"], turns.conj())
        return out

    def orthogonal(u):
        # the shorter side to the right: X <- X (a + b S + c S^2) with S = X^T X
        x = u.T if u.size(0) < u.size(1) else u
        x = x / max(float(torch.linalg.matrix_norm(x)), NORM_FLOOR)
        for _ in range(STEPS):
            sym = x.T @ x
            poly = COEFFICIENTS[2] * sym + COEFFICIENTS[1] * torch.eye(len(sym), device="cuda", dtype=torch.float64)
            poly = poly @ sym
            poly.diagonal().add_(COEFFICIENTS[0])
            x = x @ poly
        return x.T if u.size(0) < u.size(1) else x

    if kind == "orth":
        return [orthogonal(v.double()) for v in s["grads"]]
    momenta = [MOMENTUM * v.double() + w.double() for v, w in zip(s["momenta"], s["grads"])]
    rate = LR * max(1.0, case["m"] / case["n"]) ** 0.5
    params = [p.double() - LR * WEIGHT_DECAY * p.double() - rate * orthogonal(w.double() + MOMENTUM * v)
              for p, v, w in zip(s["params"], momenta, s["grads"])]
    return {"params": params, "momenta": momenta}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "norm":
        n, d = case["rows"] * case["d"], case["d"]
        tensors = 4 if case["residual"] else 2            # x, r -> y, h
        nbytes, flops = tensors * n * size + d * size, 5 * n
        if case["backward"]:                              # dy, dh -> dx (which is dr too), dw
            nbytes += (3 if case["residual"] else 2) * n * size + d * size
            flops += 10 * n
        return {"bytes": nbytes, "flops": flops}
    if kind == "norm8":
        n, d = case["rows"] * case["d"], case["d"]
        scales = case["rows"] * (d // case["group"] if case["group"] else 1) * 4
        return {"bytes": (3 if case["residual"] else 1) * n * size + n + scales + d * size, "flops": 8 * n}
    if kind == "rotary":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv"]) * case["d"]
        passes = 2 if case["backward"] else 1
        rows = tokens if case["given"] else case["seq"]
        table = min(rows, case["seq"] + 4096) * case["rot"] * 4 + (tokens * 8 if case["given"] else 0)
        return {"bytes": passes * 2 * n * size + table, "flops": passes * 3 * tokens * (case["heads"] + case["kv"]) * case["rot"]}
    m, n, count = min(case["m"], case["n"]), max(case["m"], case["n"]), case["count"]
    # X X^T and A A are symmetric: half of each
    flops = count * STEPS * (m * m * n + m * m * m + 2 * m * m * n)
    if kind == "orth":
        return {"bytes": count * m * n * (size + 2), "flops": flops}
    return {"bytes": count * m * n * (3 * size + 8), "flops": flops}
