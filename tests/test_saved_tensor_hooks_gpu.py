"""Hooks on saved tensors: what they give back has to be what they were given, in any layout; anything else is refused before a kernel reads it."""
import pytest
import torch

from nangila import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
NAMES = ["dropout", "embedding", "loss", "losses", "half", "odd", "norm", "added", "rotary", "positions"]


def calls():
    g = torch.Generator(device=DEV).manual_seed(0)

    def make(*shape, dtype=BF16):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype)

    x, w, b, norm = make(6, 64), make(50, 64), make(50), make(64)
    ids, seed = torch.tensor([1, 4, 4, 0, 2, 7], device=DEV), torch.tensor([5], device=DEV)
    q, k, table = make(2, 3, 4, 16), make(2, 3, 2, 16), ops.rotary_table(8, 16, device=DEV)
    where = torch.tensor([[0, 2, 4], [1, 3, 5]], device=DEV)
    return {
        "dropout": (lambda a: ops.dropout(a, 0.5, seed=seed), (x,)),
        "embedding": (lambda a: ops.embedding(ids, a), (w,)),
        "loss": (lambda a, c, e: ops.linear_cross_entropy(a, c, ids, bias=e), (x, w, b)),
        "losses": (lambda a, c, e: ops.linear_cross_entropy(a, c, ids, bias=e, reduction="none"), (x, w, b)),
        "half": (lambda a, c: ops.linear_cross_entropy(a, c, ids), (x.half(), w.half())),
        "odd": (lambda a, c: ops.linear_cross_entropy(a, c, ids), (x[:, :33], w[:, :33])),
        "norm": (ops.rms_norm, (x, norm)),
        "added": (lambda a, c, e: ops.add_rms_norm(a, c, e)[0], (x, x.flip(0), norm)),
        "rotary": (lambda a, c: torch.cat([v.flatten() for v in ops.rotary(a, c, table)]), (q, k)),
        "positions": (lambda a: ops.rotary(a, None, table, positions=where), (q,)),
    }


def gradients(call, args, unpack=None):
    leaves = [a.detach().clone().requires_grad_() for a in args]
    if unpack is None:
        y = call(*leaves)
    else:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = call(*leaves)
    return torch.autograd.grad(y, leaves, torch.ones_like(y))


def apart(t):
    """The same values, not side by side."""
    return torch.stack((t, t), -1)[..., 0]


@pytest.mark.parametrize("name", NAMES)
def test_the_same_values_in_another_layout(name):
    call, args = calls()[name]
    for got in (gradients(call, args, apart), gradients(call, args, lambda t: t.cpu().to(DEV))):
        assert all(torch.equal(a, c) for a, c in zip(got, gradients(call, args)))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("wrong", ["device", "type", "fewer", "more"])
def test_anything_else_is_refused(name, wrong):
    call, args = calls()[name]
    unpack = {"device": lambda t: t.cpu(), "type": lambda t: t.double(), "fewer": lambda t: t[:-1], "more": lambda t: torch.cat((t, t))}[wrong]
    count = []
    gradients(call, args, lambda t: count.append(t) or t)
    for i in range(len(count)):
        if count[i].dim() == 0:
            continue
        if name in ("rotary", "positions") and wrong in ("fewer", "more") and count[i].dim() == 3:
            continue  # (a longer table has all that is asked for; a shorter one here too)
        if name == "positions" and wrong == "fewer" and count[i].dim() == 2:
            continue  # (one row of positions is for all of the batch)
        seen = []

        def one(t):
            seen.append(t)
            return unpack(t) if len(seen) == i + 1 else t

        with pytest.raises((ValueError, TypeError, RuntimeError), match="nangila"):
            gradients(call, args, one)
