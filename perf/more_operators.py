"""What the vocabulary's operators are timed on: token embeddings, dropout, and the loss of a head whose logits are not kept.

Kinds
  embed    ``embedding``: rows of a table by token, scaled; forward alone or with the table's gradient
  drop     ``dropout`` with a mask that follows from a seed, with or without a residual; forward alone or with the gradients
  loss     ``linear_cross_entropy``: a projection onto the vocabulary and its softmax cross entropy; forward alone or with the gradients

The plain forms compute in 32 bits and round once at the end.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORED = -100


def listed():
    return [
        # the prompt of one short sequence looked up in the decoder's table: latency
        {"name": "embed_sequence", "kind": "embed", "tokens": 128, "rows": 32000, "d": 2048, "dtype": "bf16", "scale": 1.0, "common": 0.0, "padding": False, "backward": False},
        # the decoder's training step, 4 x 2048 tokens, with the table's gradient
        {"name": "embed_decoder", "kind": "embed", "tokens": 8192, "rows": 32000, "d": 2048, "dtype": "bf16", "scale": 1.0, "common": 0.0, "padding": False, "backward": True},
        # the encoder's, 16 x 512 tokens of which 15 % are the same mask token; parameters in single precision, scaled by the root of the width
        {"name": "embed_encoder_fp32", "kind": "embed", "tokens": 8192, "rows": 30592, "d": 1024, "dtype": "fp32", "scale": 32.0, "common": 0.15, "padding": False, "backward": True},
        # a ragged batch, half of it padding that gets no gradient, a width that no vector divides
        {"name": "embed_odd_fp16", "kind": "embed", "tokens": 16381, "rows": 50257, "d": 769, "dtype": "fp16", "scale": 27.5, "common": 0.5, "padding": True, "backward": True},
        # a short sequence of GPT-2 small in evaluation of a stochastic ensemble: latency
        {"name": "drop_sequence", "kind": "drop", "rows": 128, "d": 768, "dtype": "bf16", "p": 0.1, "residual": False, "backward": False},
        # the decoder's training step: a projection's output dropped and added to the residual stream, with the gradients
        {"name": "drop_residual_bf16", "kind": "drop", "rows": 8192, "d": 2048, "dtype": "bf16", "p": 0.1, "residual": True, "backward": True},
        # odd sizes in single precision, a third dropped
        {"name": "drop_odd_fp32", "kind": "drop", "rows": 4099, "d": 1001, "dtype": "fp32", "p": 0.3, "residual": False, "backward": True},
        # the losses of a few tokens one by one, no gradients (scoring of a continuation)
        {"name": "loss_few_tokens", "kind": "loss", "tokens": 16, "d": 2048, "rows": 32000, "classes": 32000, "dtype": "bf16", "bias": False, "ignored": 0.0,
         "reduction": "none", "backward": False},
        # the encoder's masked tokens, 15 % of 16 x 512, with a bias and padded classes
        {"name": "loss_encoder", "kind": "loss", "tokens": 1229, "d": 1024, "rows": 30592, "classes": 30522, "dtype": "bf16", "bias": True, "ignored": 0.0,
         "reduction": "mean", "backward": True},
        # GPT-2 small's training step, 8 x 1024 tokens, padded classes
        {"name": "loss_gpt2", "kind": "loss", "tokens": 8192, "d": 768, "rows": 50304, "classes": 50257, "dtype": "bf16", "bias": False, "ignored": 0.0,
         "reduction": "mean", "backward": True},
        # the decoder's training step, 4 x 2048 tokens
        {"name": "loss_decoder", "kind": "loss", "tokens": 8192, "d": 2048, "rows": 32000, "classes": 32000, "dtype": "bf16", "bias": False, "ignored": 0.0,
         "reduction": "mean", "backward": True},
        # ragged sizes in half precision, weights for the tokens' losses, a fifth of them ignored
        {"name": "loss_odd_fp16", "kind": "loss", "tokens": 1023, "d": 1000, "rows": 10007, "classes": 10007, "dtype": "fp16", "bias": True, "ignored": 0.2,
         "reduction": "none", "backward": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "drop", "loss", "loss"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    backward = rng.random() < 0.6
    if kind == "embed":
        d = _log(rng, 32, 4096)
        d = d if rng.random() < 0.3 else max(32, d // 64 * 64)
        rows = _log(rng, 500, max(501, min(130000, 250_000_000 // (SIZE[dtype] * d))))
        tokens = _log(rng, 1, min(131072, 250_000_000 // (SIZE[dtype] * d)))
        return {"kind": kind, "tokens": tokens, "rows": rows, "d": d, "dtype": dtype, "scale": rng.choice([1.0, round(math.sqrt(d), 2)]),
                "common": rng.choice([0.0, 0.15, 0.5]), "padding": rng.random() < 0.3, "backward": backward}
    if kind == "drop":
        d = _log(rng, 32, 8192)
        rows = _log(rng, 1, max(1, 100_000_000 // (SIZE[dtype] * d)))
        return {"kind": kind, "rows": rows, "d": d, "dtype": dtype, "p": rng.choice([0.05, 0.1, 0.2, 0.5, 0.75]), "residual": rng.random() < 0.5, "backward": backward}
    d = _log(rng, 32, 4096)
    d = d if rng.random() < 0.2 else max(64, d // 64 * 64)
    rows = _log(rng, 500, 100000)
    tokens = _log(rng, 1, max(1, min(16384, 8192 * 2048 * 32000 // (d * rows))))
    return {"kind": kind, "tokens": tokens, "d": d, "rows": rows, "classes": rows - rng.choice([0, 0, 1, 47, 70]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "bias": rng.random() < 0.4, "ignored": rng.choice([0.0, 0.0, 0.2, 0.85]), "reduction": rng.choice(["mean", "mean", "sum", "none"]), "backward": backward}


# ---- inputs ----------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _tokens(g, count, rows):
    """Token ids as texts have them: the r-th most frequent one in proportion to 1 / r."""
    rank = torch.exp(torch.rand(count, device="cuda", generator=g, dtype=torch.float64) * math.log(rows)).long() - 1
    return torch.randperm(rows, device="cuda", generator=g)[rank.clamp(0, rows - 1)]


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    wants = case["backward"]
    state = dict(case)
    if kind == "embed":
        n, rows, d = case["tokens"], case["rows"], case["d"]
        ids = _tokens(g, n, rows)
        if case["common"]:
            ids = torch.where(torch.rand(n, device="cuda", generator=g) < case["common"], torch.full_like(ids, 3), ids)
        state["ids"] = ids
        state["padding_idx"] = 3 if case["padding"] else None
        state["w"] = (0.02 * _normal(g, torch.float32, rows, d)).to(dtype).requires_grad_(wants)
        if wants:
            state["dy"] = _normal(g, dtype, n, d)
    elif kind == "drop":
        rows, d = case["rows"], case["d"]
        state["seed"] = int(torch.randint(0, 2 ** 62, (1,), generator=torch.Generator().manual_seed(int(seed))))
        state["x"] = _normal(g, dtype, rows, d).requires_grad_(wants)
        state["r"] = _normal(g, dtype, rows, d).requires_grad_(wants) if case["residual"] else None
        if wants:
            state["dy"] = _normal(g, dtype, rows, d)
    else:
        n, rows, d, classes = case["tokens"], case["rows"], case["d"], case["classes"]
        w = (_normal(g, torch.float32, rows, d) / math.sqrt(d)).to(dtype)
        targets = _tokens(g, n, classes)
        # tokens from those that the model knows nothing of to those that it is sure about
        sure = 12 * torch.rand(n, 1, device="cuda", generator=g)
        known = w[targets].float()
        x = _normal(g, torch.float32, n, d) + sure * known / known.square().sum(-1, keepdim=True)
        if case["ignored"]:
            skip = torch.rand(n, device="cuda", generator=g) < case["ignored"]
            skip[0] = False
            targets = torch.where(skip, torch.full_like(targets, IGNORED), targets)
        state["x"], state["w"], state["targets"] = x.to(dtype).requires_grad_(wants), w.requires_grad_(wants), targets
        state["b"] = (0.1 * _normal(g, torch.float32, rows)).to(dtype).requires_grad_(wants) if case["bias"] else None
        if wants:
            if case["reduction"] == "none":
                state["dloss"] = 0.5 + torch.rand(n, device="cuda", generator=g)
            else:  # (the scale of the loss that half precision is trained with)
                state["dloss"] = torch.tensor(4096.0 if case["dtype"] == "fp16" else 1.0, device="cuda")
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from nangila import ops

    kind = s["kind"]
    if kind == "embed":
        y = ops.embedding(s["ids"], s["w"], scale=s["scale"], padding_idx=s["padding_idx"])
        if not s["backward"]:
            return {"y": y}
        return {"y": y, "dw": torch.autograd.grad(y, s["w"], s["dy"])[0]}
    if kind == "drop":
        y = ops.dropout(s["x"], s["p"], seed=s["seed"], residual=s["r"])
        if not s["backward"]:
            return {"y": y}
        if s["r"] is None:
            return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
        dx, dr = torch.autograd.grad(y, (s["x"], s["r"]), s["dy"])
        return {"y": y, "dx": dx, "dr": dr}
    loss = ops.linear_cross_entropy(s["x"], s["w"], s["targets"], bias=s["b"], num_classes=s["classes"], ignore_index=IGNORED, reduction=s["reduction"])
    if not s["backward"]:
        return {"loss": loss}
    grads = torch.autograd.grad(loss, (s["x"], s["w"]) if s["b"] is None else (s["x"], s["w"], s["b"]), s["dloss"])
    return {"loss": loss, **dict(zip(("dx", "dw", "db"), grads))}


@torch.no_grad()
def _plain(s):
    if s["kind"] == "embed":
        return _plain_embed(s)
    if s["kind"] == "drop":
        return _plain_drop(s)
    return _plain_loss(s)


def _plain_embed(s):
    w, ids = s["w"], s["ids"]
    out = {"y": (w[ids].float() * s["scale"]).to(w.dtype)}
    if s["backward"]:
        wide = torch.float64 if s["dtype"] == "fp32" else torch.float32  # (the common token's sum is a long one)
        dw = torch.zeros(w.shape, dtype=wide, device="cuda").index_add_(0, ids, s["dy"].to(wide))
        if s["padding_idx"] is not None:
            dw[s["padding_idx"]] = 0
        out["dw"] = (dw * s["scale"]).to(w.dtype)
    return out


LOW = 0xFFFFFFFF


def _product(a, b):
    """Both halves of a 32 x 32 bit product: (high, low). ``a`` a number, ``b`` a tensor of numbers below 2^32."""
    high = (a * (b >> 16) + ((a * (b & 0xFFFF)) >> 16)) >> 16
    return high, (a * b) & LOW


def _philox(block, draw, which, key):
    """Four 32-bit numbers for each block: Philox4x32 with ten rounds (J. Salmon and others, 2011)."""
    c = [block & LOW, block >> 32, torch.full_like(block, draw), torch.full_like(block, which)]
    k = [key & LOW, key >> 32 & LOW]
    for _ in range(10):
        (h0, l0), (h1, l1) = _product(0xD2511F53, c[0]), _product(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k[0], l1, h0 ^ c[3] ^ k[1], l0]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return torch.stack(c, dim=-1)


def _plain_kept(s):
    """Of each element, whether its 32-bit number, the upper half from one block of eight elements and the lower from another, reaches p's."""
    n = s["rows"] * s["d"]
    block = torch.arange((n + 7) // 8, device="cuda")
    upper, lower = (_philox(block, 0, which, s["seed"]) for which in (0, 1))
    upper, lower = (torch.stack((v & 0xFFFF, v >> 16), dim=-1).view(-1)[:n] for v in (upper, lower))
    return ((upper << 16 | lower) >= round(s["p"] * 2 ** 32)).view(s["rows"], s["d"])


def _plain_drop(s):
    kept = _plain_kept(s)
    scale = 1 / (1 - round(s["p"] * 2 ** 32) / 2 ** 32)
    dropped = torch.where(kept, s["x"].float() * scale, 0.0)
    out = {"y": (dropped if s["r"] is None else s["r"].float() + dropped).to(s["x"].dtype)}
    if s["backward"]:
        out["dx"] = torch.where(kept, s["dy"].float() * scale, 0.0).to(s["x"].dtype)
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _plain_loss(s):
    x, w, targets, classes = s["x"].float(), s["w"].float(), s["targets"], s["classes"]
    valid = targets != IGNORED
    at = targets.clamp(min=0)[:, None]
    z = x @ w[:classes].T
    if s["b"] is not None:
        z += s["b"][:classes].float()
    top = z.amax(-1, keepdim=True)
    of_target = z.gather(1, at)
    e = (z - top).exp_()
    total = e.sum(-1, keepdim=True)
    losses = torch.where(valid, (top + total.log() - of_target).squeeze(1), 0.0)
    count = valid.sum()
    out = {"loss": losses if s["reduction"] == "none" else losses.sum() if s["reduction"] == "sum" else losses.sum() / count}
    if s["backward"]:
        g = valid.float() * s["dloss"] / (count if s["reduction"] == "mean" else 1)
        e /= total
        e.scatter_add_(1, at, -torch.ones_like(top))
        e *= g[:, None]
        out["dx"] = (e @ w[:classes]).to(s["x"].dtype)
        dw = torch.zeros_like(w)
        torch.mm(e.T, x, out=dw[:classes])
        out["dw"] = dw.to(s["w"].dtype)
        if s["b"] is not None:
            db = torch.zeros_like(s["b"])
            db[:classes] = e.sum(0).to(db.dtype)
            out["db"] = db
    return out


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _numbers(n, key):
    """The 32-bit numbers of n elements, with numpy's 64-bit integers."""
    blocks = np.arange(-(-n // 8), dtype=np.uint64)
    low, sixteen, thirty_two = np.uint64(LOW), np.uint64(0xFFFF), np.uint64(32)

    def halves(which):
        a, b = blocks & low, blocks >> thirty_two
        c, d = np.zeros_like(blocks), np.full_like(blocks, which)
        for r in range(10):
            p, q = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
            ka, kb = np.uint64(((key & LOW) + r * 0x9E3779B9) & LOW), np.uint64(((key >> 32 & LOW) + r * 0xBB67AE85) & LOW)
            a, b, c, d = (q >> thirty_two) ^ b ^ ka, q & low, (p >> thirty_two) ^ d ^ kb, p & low
        words = np.stack((a, b, c, d), axis=1)
        return np.stack((words & sixteen, words >> np.uint64(16)), axis=2).reshape(-1)[:n]

    return halves(0) * np.uint64(65536) + halves(1)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        out = {"y": torch.nn.functional.embedding(s["ids"], s["w"].double()) * case["scale"]}
        if case["backward"]:
            order = torch.argsort(s["ids"], stable=True)
            ids, lengths = torch.unique_consecutive(s["ids"][order], return_counts=True)
            sums = torch.segment_reduce(s["dy"].double()[order], "sum", lengths=lengths, axis=0) * case["scale"]
            dw = torch.zeros(case["rows"], case["d"], dtype=torch.float64, device="cuda")
            dw[ids] = sums if s["padding_idx"] is None else torch.where((ids == s["padding_idx"])[:, None], 0.0, sums)
            out["dw"] = dw
        return out
    if case["kind"] == "drop":
        least = round(case["p"] * 2 ** 32)
        kept = torch.from_numpy((_numbers(case["rows"] * case["d"], s["seed"]) >= np.uint64(least)).reshape(case["rows"], case["d"])).cuda()
        share = (2 ** 32 - least) / 2 ** 32
        y = s["x"].double() / share * kept
        out = {"y": y if s["r"] is None else y + s["r"].double()}
        if case["backward"]:
            out["dx"] = s["dy"].double() / share * kept
            if s["r"] is not None:
                out["dr"] = s["dy"].double()
        return out
    x, w, b = (None if s[k] is None else s[k].double().requires_grad_(case["backward"]) for k in ("x", "w", "b"))
    with torch.set_grad_enabled(case["backward"]):
        z = torch.nn.functional.linear(x, w, b)[:, :case["classes"]]
        loss = torch.nn.functional.cross_entropy(z, s["targets"], ignore_index=IGNORED, reduction=case["reduction"])
    if not case["backward"]:
        return {"loss": loss}
    grads = torch.autograd.grad(loss, (x, w) if b is None else (x, w, b), s["dloss"].double())
    return {"loss": loss.detach(), **dict(zip(("dx", "dw", "db"), grads))}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "embed":
        n, d = case["tokens"], case["d"]
        nbytes, flops = n * 8 + 2 * n * d * size, n * d
        if case["backward"]:
            nbytes += n * d * size + case["rows"] * d * size
            flops += n * d
        return {"bytes": nbytes, "flops": flops}
    if kind == "drop":
        n = case["rows"] * case["d"]
        nbytes, flops = (3 if case["residual"] else 2) * n * size, 2 * n
        if case["backward"]:
            nbytes, flops = nbytes + 2 * n * size, flops + n
        return {"bytes": nbytes, "flops": flops}
    n, d, rows, classes = case["tokens"], case["d"], case["rows"], case["classes"]
    nbytes, flops = (n * d + classes * d + (classes if case["bias"] else 0)) * size + 8 * n + (4 * n if case["reduction"] == "none" else 4), 2 * n * d * classes
    if case["backward"]:
        nbytes += (n * d + rows * d + (rows if case["bias"] else 0)) * size
        flops *= 3
    return {"bytes": nbytes, "flops": flops}
