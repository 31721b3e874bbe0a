"""Embeddings, dropout and the head's loss on the CPU: the formulas, and what is refused."""
import pytest
import torch
import torch.nn.functional as F

from nangila import ops
from tests._vocab_ops import embedding_grad, head, kept, numbers, philox_block, share


def test_philox_known_answers():
    # published with the generator: counter and key of zeros, of ones, and of the digits of pi
    assert philox_block((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert philox_block((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox_block((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    v = numbers(16, 0x299F31D0A4093822, 5)
    for b in (0, 1):
        upper, lower = (philox_block((b, 0, 5, which), (0xA4093822, 0x299F31D0)) for which in (0, 1))
        for i in range(8):
            s = 16 * (i & 1)
            assert int(v[8 * b + i]) == (upper[i // 2] >> s & 0xFFFF) << 16 | lower[i // 2] >> s & 0xFFFF


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dropout(dtype):
    x, r = torch.randn(31, 17).to(dtype).requires_grad_(), torch.randn(31, 17).to(dtype).requires_grad_()
    keep = kept((31, 17), 0.3, 99, 4)
    y = ops.dropout(x, 0.3, seed=99, residual=r, draw=4)
    want = r.double() + torch.where(keep, x.double() / share(0.3), 0.0)
    assert y.dtype == dtype and torch.allclose(y.double(), want, rtol=torch.finfo(dtype).eps, atol=1e-6)
    dx, dr = torch.autograd.grad(y.sum(), (x, r))
    assert torch.equal(dx != 0, keep) and bool((dr == 1).all())
    torch.manual_seed(1)
    a = ops.dropout(x)
    torch.manual_seed(1)
    assert torch.equal(a, ops.dropout(x)) and not torch.equal(a, ops.dropout(x))
    assert torch.equal(ops.dropout(x, 0.0), x) and not ops.dropout(x, 1.0).any()
    assert torch.equal(ops.dropout(x, 0.3, seed=torch.tensor(99), draw=4, residual=r), y)


def test_embedding():
    w, ids = torch.randn(20, 6, requires_grad=True), torch.tensor([[1, 2, 2], [19, -1, 20]])
    y = ops.embedding(ids, w, scale=2.0, padding_idx=19)
    inside = (ids >= 0) & (ids < 20)
    assert torch.equal(y[inside], 2 * w[ids[inside]]) and bool(y[~inside].isnan().all())
    dy = torch.randn(2, 3, 6)
    dw, = torch.autograd.grad(y, w, dy)
    assert torch.allclose(dw.double(), embedding_grad(ids, dy, 20, 2.0, 19)[0], atol=1e-6)
    assert ops.embedding(torch.empty(0, 3, dtype=torch.int32), w).shape == (0, 3, 6)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_linear_cross_entropy(reduction):
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(4, 5, 12, generator=g), torch.randn(30, 12, generator=g), torch.randn(30, generator=g)
    t = torch.randint(0, 28, (4, 5), generator=g)
    t[1, 2] = -100
    leaves = [v.requires_grad_() for v in (x, w, b)]
    loss = ops.linear_cross_entropy(x, w, t, bias=b, num_classes=28, reduction=reduction)
    theirs = F.cross_entropy(F.linear(x, w, b)[..., :28].reshape(-1, 28), t.reshape(-1), reduction=reduction)
    assert torch.allclose(loss.reshape(-1), theirs.reshape(-1), atol=1e-5)
    up = torch.rand(loss.shape, generator=g)
    want = head(x.detach(), w.detach(), t, b.detach(), 28, reduction=reduction, upstream=up)
    for got, name in zip(torch.autograd.grad(loss, leaves, up), ("dx", "dw", "db")):
        assert torch.allclose(got.double().reshape(want[name].shape), want[name], atol=1e-5), name
    assert bool(ops.linear_cross_entropy(x, w, torch.full_like(t, 30), reduction="none").isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_that_add_nothing_hold_anything(reduction, dtype):
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(9, 8, generator=g).to(dtype), torch.randn(12, 8, generator=g).to(dtype)
    t = torch.randint(0, 10, (9,), generator=g)
    t[::3] = -100
    t[1] = 10  # no class
    results = []
    for row, other, padding in ((0.0, 0.0, 0.0), (float("nan"), float("inf"), float("nan"))):
        x[::3], x[1], w[10:] = row, other, padding
        leaves = [v.clone().requires_grad_() for v in (x, w)]
        loss = ops.linear_cross_entropy(*leaves, t, num_classes=10, reduction=reduction)
        results.append((loss, *torch.autograd.grad(loss, leaves, torch.ones_like(loss))))
    for clean, dirty in zip(*results):
        assert torch.equal(clean.nan_to_num(7.0), dirty.nan_to_num(7.0))
    _, dx, dw = results[1]
    assert bool(dx.isfinite().all() and dw.isfinite().all()) and not dx[::3].any() and not dx[1].any() and not dw[10:].any()


def test_autocast_on_the_cpu_leaves_float32():
    g = torch.Generator().manual_seed(2)
    x, w, t = torch.randn(9, 8, generator=g), torch.randn(12, 8, generator=g), torch.randint(0, 12, (9,), generator=g)
    results = []
    for on in (False, True):
        leaves = [v.clone().requires_grad_() for v in (x, w)]
        with torch.autocast("cpu", dtype=torch.bfloat16, enabled=on):
            losses = ops.linear_cross_entropy(*leaves, t, reduction="none")
            y = ops.embedding(t, leaves[1])
        results.append((losses, y, *torch.autograd.grad(losses.sum() + y.sum(), leaves)))
    for plain, cast in zip(*results):
        assert cast.dtype == torch.float32 and torch.equal(plain, cast)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_results_are_packed(dtype):
    ids, w = torch.tensor([[0, 1, 2], [3, 3, 0]]).T, torch.arange(20.0).to(dtype).view(5, 4).T
    for i in (ids, ids.contiguous()):
        for table in (w, w.contiguous()):
            y = ops.embedding(i, table)
            assert y.is_contiguous() and torch.equal(y, w[ids])
    for x in (w, w[:, :1].expand(4, 5)):
        assert ops.dropout(x, 0.5, seed=3).is_contiguous() and ops.dropout(x, 0.5, seed=3, residual=w).is_contiguous()


def test_refusals():
    x, w, t = torch.randn(3, 8), torch.randn(5, 8), torch.tensor([0, 1, 2])
    ids = torch.tensor([1, 2])
    for bad, error, match in [
        (lambda: ops.dropout(x, 1.5), ValueError, "p must be"),
        (lambda: ops.dropout(x, -0.1), ValueError, "p must be"),
        (lambda: ops.dropout(x, float("nan")), ValueError, "p must be"),
        (lambda: ops.dropout(x, 0.5, seed=-1), ValueError, "seed must be"),
        (lambda: ops.dropout(x, 0.5, seed=2 ** 64), ValueError, "seed must be"),
        (lambda: ops.dropout(x, 0.5, seed=1, draw=2 ** 32), ValueError, "draw must be"),
        (lambda: ops.dropout(x, 0.5, seed=torch.tensor([1, 2])), ValueError, "one number"),
        (lambda: ops.dropout(x, 0.5, seed=torch.tensor(1.0)), TypeError, "int64"),
        (lambda: ops.dropout(x.double(), 0.5), TypeError, "float32, float16 or bfloat16"),
        (lambda: ops.dropout(x, 0.5, residual=x[:2]), ValueError, "residual has shape"),
        (lambda: ops.dropout(x, 0.5, residual=x.half()), TypeError, "residual is"),
        (lambda: ops.embedding(ids.float(), w), TypeError, "int64 or int32"),
        (lambda: ops.embedding(ids, w[0]), ValueError, "shape"),
        (lambda: ops.embedding(ids, w.double()), TypeError, "float32, float16 or bfloat16"),
        (lambda: ops.embedding(ids, w, padding_idx=5), ValueError, "padding_idx"),
        (lambda: ops.embedding(ids, w, padding_idx=-6), ValueError, "padding_idx"),
        (lambda: ops.embedding(ids, w, scale=float("inf")), ValueError, "scale"),
        (lambda: ops.embedding(ids, w.to_sparse()), TypeError, "dense"),
        (lambda: ops.linear_cross_entropy(x, w, t, reduction="max"), ValueError, "reduction"),
        (lambda: ops.linear_cross_entropy(x, w[:, :7], t), ValueError, "weight must have shape"),
        (lambda: ops.linear_cross_entropy(x, w.half(), t), TypeError, "weight is"),
        (lambda: ops.linear_cross_entropy(x, w, t[:2]), ValueError, "targets have shape"),
        (lambda: ops.linear_cross_entropy(x, w, t.float()), TypeError, "int64 or int32"),
        (lambda: ops.linear_cross_entropy(x, w, t, num_classes=6), ValueError, "num_classes"),
        (lambda: ops.linear_cross_entropy(x, w, t, num_classes=0), ValueError, "num_classes"),
        (lambda: ops.linear_cross_entropy(x, w, t, bias=w[:, 0][:4]), ValueError, "bias must have shape"),
        (lambda: ops.linear_cross_entropy(x.double(), w.double(), t), TypeError, "float32, float16 or bfloat16"),
    ]:
        with pytest.raises(error, match=match):
            bad()
