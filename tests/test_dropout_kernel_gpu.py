"""Dropout's kernel against its definition: masks exactly, values in 64 bits."""
import pytest
import torch

from nangila import ops
from tests._model_ops import rounding
from tests._vocab_ops import kept, share

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of float32


def make(shape, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def check(y, x, keep, p, dtype, residual=None):
    # the factor is rounded to float32, the product and the sum each once, the result once more
    term = torch.where(keep, x.double() / share(p), 0.0) if p < 1 else torch.zeros_like(x, dtype=torch.float64)
    want = term if residual is None else term + residual.double()
    tol = 2.1 * U * term.abs() + (0 if residual is None else U * want.abs()) + rounding(want, dtype) * (1 + 4 * U)
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
    assert bool(((y.double() - want).abs() <= tol).all()), ((y.double() - want).abs() - tol).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5, 17), (129, 768), (1, 65536 * 3 + 5), (4099, 1001)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_values_masks_and_gradients(dtype, shape, p):
    x, r, dy = (make(shape, dtype, i) for i in range(3))
    keep = kept(shape, p, 1234567890123456789).to(DEV)
    for residual in (None, r):
        xs = x.clone().requires_grad_()
        rs = None if residual is None else residual.clone().requires_grad_()
        y = ops.dropout(xs, p, seed=1234567890123456789, residual=rs)
        check(y, x, keep, p, dtype, residual)
        if residual is None:
            dx, = torch.autograd.grad(y, xs, dy)
        else:
            dx, dr = torch.autograd.grad(y, (xs, rs), dy)
            assert torch.equal(dr, dy)
        check(dx, dy, keep, p, dtype)


@pytest.mark.parametrize("p", [0.0, 1e-9, 1 / 65536, 0.25, 0.3, 1 - 2.0 ** -20, 1.0])
def test_probabilities_at_the_borders(p):
    x = make((1 << 20,), torch.float32)
    keep = kept((1 << 20,), p, 3, 9).to(DEV)
    check(ops.dropout(x, p, seed=3, draw=9), x, keep, p, torch.float32)
    if p == 0.0:
        assert torch.equal(ops.dropout(x, p, seed=3), x)
    if p == 1.0:
        assert not keep.any() and not ops.dropout(x, p, seed=3).any()


def test_ties_in_the_upper_half_go_by_the_lower():
    # among 2^21 numbers some 32 have the upper half of p's: those are told apart by the lower one
    n, p = 1 << 21, 0.1
    from tests._vocab_ops import numbers

    v = numbers(n, 77)
    least = round(p * 2 ** 32)
    tied = torch.from_numpy((v >> 16) == (least >> 16)).to(DEV)
    assert 5 <= int(tied.sum()) <= 100 and 0 < int((tied & (torch.from_numpy(v >= least).to(DEV))).sum()) < int(tied.sum())
    y = ops.dropout(torch.ones(n, device=DEV), p, seed=77)
    assert torch.equal(y != 0, torch.from_numpy(v >= least).to(DEV))


def test_what_is_dropped_is_not_looked_at():
    x = make((64, 64), torch.bfloat16)
    keep = kept((64, 64), 0.4, 5).to(DEV)
    y = ops.dropout(torch.where(keep, x, float("nan")), 0.4, seed=5, residual=x)
    assert torch.equal(y, ops.dropout(torch.where(keep, x, float("inf")), 0.4, seed=5, residual=x)) and bool(y.isfinite().all())


def test_seeds_draws_and_the_cpu_agree():
    x = make((300, 41), torch.bfloat16)
    seeds = [0, 1, 2 ** 32, 2 ** 63, 2 ** 64 - 1]
    masks = [ops.dropout(torch.ones_like(x), 0.5, seed=s, draw=d) != 0 for s in seeds for d in (0, 1, 2 ** 32 - 1)]
    for i, a in enumerate(masks):
        for b in masks[:i]:
            assert 0.4 < float((a == b).float().mean()) < 0.6
    for s in seeds:
        assert torch.equal(ops.dropout(x, 0.3, seed=s, draw=3, residual=x).cpu(), ops.dropout(x.cpu(), 0.3, seed=s, draw=3, residual=x.cpu()))
    tensor = torch.tensor(seeds[2], device=DEV)
    assert torch.equal(ops.dropout(x, 0.3, seed=tensor), ops.dropout(x, 0.3, seed=seeds[2]))


def test_strides_and_starts():
    wide = make((64, 40), torch.bfloat16)
    for x in (wide[:, 3:36], wide.T, wide[::2], wide[:, 1:], make((1, 40), torch.bfloat16).expand(64, 40), wide.flatten()[1:]):
        y = ops.dropout(x, 0.2, seed=8, residual=x)
        assert torch.equal(y, ops.dropout(x.contiguous(), 0.2, seed=8, residual=x.clone()))
    # (a packed tensor that does not start on 16 bytes)
    out = ops.dropout(wide.flatten()[1:], 0.2, seed=8)
    check(out, wide.flatten()[1:], kept((64 * 40 - 1,), 0.2, 8).to(DEV), 0.2, torch.bfloat16)


def test_default_seed_follows_pytorchs_generator():
    x = make((4096,), torch.float32)
    torch.manual_seed(3)
    a, b = ops.dropout(x), ops.dropout(x)
    torch.manual_seed(3)
    assert torch.equal(ops.dropout(x), a) and not torch.equal(a, b)


def test_captured_graph_reads_the_seed_when_it_runs():
    x, dy = make((257, 33), torch.bfloat16).requires_grad_(), make((257, 33), torch.bfloat16, 1)
    seed = torch.tensor(1, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(ops.dropout(x, 0.25, seed=seed), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout(x, 0.25, seed=seed)
        dx, = torch.autograd.grad(y, x, dy)
        with pytest.raises(RuntimeError, match="captured"):
            ops.dropout(x, 0.25)
    for s in (1, 2, 12345678901):
        seed.fill_(s)
        graph.replay()
        keep = kept((257, 33), 0.25, s).to(DEV)
        check(y, x.detach(), keep, 0.25, torch.bfloat16)
        check(dx, dy, keep, 0.25, torch.bfloat16)


def test_a_seed_that_changed_before_the_backward_pass_is_noticed():
    x, seed = make((64,), torch.float32).requires_grad_(), torch.tensor(1, device=DEV)
    y = ops.dropout(x, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_other_streams():
    x = make((1 << 22,), torch.bfloat16)
    want = ops.dropout(x, 0.1, seed=4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.dropout(x, 0.1, seed=4)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
