"""Token embeddings against their formulas in 64 bits."""
import pytest
import torch

from nangila import ops
from tests._model_ops import rounding
from tests._vocab_ops import embedding_grad

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def make(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def random_ids(n, rows, seed=0, common=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ids = (rows * torch.rand(n, device=DEV, generator=g) ** 3).long().clamp(max=rows - 1)
    return torch.where(torch.rand(n, device=DEV, generator=g) < common, rows // 2, ids)


def check_grad(dw, ids, dy, rows, scale, padding=None):
    # sums of `count` terms in float32 in whatever order, then the factor, then one rounding
    want, size, count = embedding_grad(ids, dy, rows, scale, padding)
    tol = (count[:, None] + 2) * U * size + rounding(want, dw.dtype) * (1 + 4 * U)
    assert dw.shape == want.shape and bool(((dw.double() - want).abs() <= tol).all()), ((dw.double() - want).abs() - tol).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (5, 8), (1000, 33), (333, 64), (2000, 769), (700, 2056)])
@pytest.mark.parametrize("n", [1, 2, 31, 257, 4099])
def test_lookup_and_gradient(dtype, rows, d, n):
    w, dy, ids = make(rows, d, dtype=dtype), make(n, d, dtype=dtype, seed=1), random_ids(n, rows)
    for scale in (1.0, -22.6):
        ws = w.clone().requires_grad_()
        y = ops.embedding(ids, ws, scale=scale)
        want = w.double()[ids] * scale
        assert y.dtype == dtype and bool(((y.double() - want).abs() <= rounding(want, dtype) * (1 + 4 * U) + 2.1 * U * want.abs()).all())
        if scale == 1.0:
            assert torch.equal(y, w[ids])
        check_grad(torch.autograd.grad(y, ws, dy)[0], ids, dy, rows, scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,rows,d,common", [(8192, 32000, 256, 0.0), (8192, 997, 40, 0.5), (65536, 50257, 24, 0.9), (70001, 1 << 21, 8, 0.1), (40000, 3, 16, 0.3), (20000, 1, 130, 0.0),
                                             (262144, 1023, 8, 0.01), (262145, 1024, 9, 0.01)])
def test_many_tokens(dtype, n, rows, d, common):
    # digits of one, two and three passes, runs over many pieces, whole batches of one token
    w, dy, ids = make(rows, d, dtype=dtype).requires_grad_(), make(n, d, dtype=dtype, seed=2), random_ids(n, rows, 3, common)
    dw, = torch.autograd.grad(ops.embedding(ids, w, scale=0.5), w, dy)
    check_grad(dw, ids, dy, rows, 0.5)
    again, = torch.autograd.grad(ops.embedding(ids, w, scale=0.5), w, dy)
    assert torch.equal(dw, again)


@pytest.mark.parametrize("piece_edge", [7, 8, 9, 15, 16, 17, 63, 64, 65])
def test_runs_that_end_at_pieces(piece_edge):
    # each id as often as a piece is long, give or take one
    ids = torch.arange(40, device=DEV).repeat_interleave(piece_edge)
    w, dy = make(41, 16).requires_grad_(), make(ids.numel(), 16, seed=4)
    order = torch.randperm(ids.numel(), device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    dw, = torch.autograd.grad(ops.embedding(ids[order], w), w, dy)
    check_grad(dw, ids[order], dy, 41, 1.0)
    assert not dw[40].any()


@pytest.mark.parametrize("d", [33, 64])
def test_ids_outside_and_padding(d):
    ids = torch.tensor([[0, -1, 5, 9], [10, 2 ** 40, 3, -2 ** 62]], device=DEV)
    w, dy = make(10, d, dtype=torch.bfloat16).requires_grad_(), make(2, 4, d, dtype=torch.bfloat16, seed=1)
    y = ops.embedding(ids, w, padding_idx=5)
    inside = (ids >= 0) & (ids < 10)
    assert y.shape == (2, 4, d) and bool(y[~inside].isnan().all()) and torch.equal(y[inside], w[ids[inside]])
    dw, = torch.autograd.grad(y, w, torch.where(inside[..., None], dy, float("nan")))
    check_grad(dw, ids, torch.where(inside[..., None], dy, 0.0), 10, 1.0, padding=5)
    assert not dw[5].any()
    dw, = torch.autograd.grad(ops.embedding(ids, w, padding_idx=-1), w, dy)
    check_grad(dw, ids, dy, 10, 1.0, padding=9)
    # nothing but what is left out
    for only in (torch.full((100,), 5, device=DEV), torch.full((100,), 77, device=DEV)):
        dw, = torch.autograd.grad(ops.embedding(only, w, padding_idx=5), w, make(100, d, dtype=torch.bfloat16))
        assert dw.shape == (10, d) and not dw.any()


def test_no_tokens():
    w = make(10, 16).requires_grad_()
    y = ops.embedding(torch.empty(2, 0, dtype=torch.long, device=DEV), w)
    assert y.shape == (2, 0, 16)
    assert not torch.autograd.grad(y.sum(), w)[0].any()


def test_types_strides_and_orders():
    table = make(50, 80, dtype=torch.float16)
    ids = random_ids(600, 50).view(20, 30)
    dy = make(20, 30, 32, dtype=torch.float16, seed=1)
    want = None
    for w in (table[:, 8:40], table[:, 8:40].contiguous(), table[:, 8:40].T.contiguous().T):
        w = w.detach().requires_grad_()
        for i in (ids, ids.int(), ids.T.contiguous().T, torch.stack((ids, ids), -1)[..., 0]):
            for g in (dy, dy.transpose(0, 1).contiguous().transpose(0, 1), make(20, 30, 40, dtype=torch.float16, seed=9).copy_(torch.nn.functional.pad(dy, (0, 8)))[..., :32]):
                y = ops.embedding(i, w)
                assert torch.equal(y, w[ids])
                dw, = torch.autograd.grad(y, w, g)
                want = dw if want is None else want
                assert torch.equal(dw, want)
    check_grad(want, ids, dy, 50, 1.0)
    # one gradient for all tokens, which has no memory of its own for each
    w = table.detach().requires_grad_()
    dw, = torch.autograd.grad(ops.embedding(ids, w).float().sum(), w)
    check_grad(dw, ids, torch.ones(20, 30, 80, device=DEV), 50, 1.0)


def test_infinities_and_nan_stay_in_their_rows():
    ids = torch.arange(64, device=DEV).repeat(40)
    w, dy = make(64, 24).requires_grad_(), make(64 * 40, 24, seed=1)
    dy[ids == 7], dy[ids == 9] = float("nan"), float("inf")
    dw, = torch.autograd.grad(ops.embedding(ids, w), w, dy)
    assert bool(dw[7].isnan().all()) and bool((dw[9] == float("inf")).all())
    others = [i for i in range(64) if i not in (7, 9)]
    assert bool(dw[others].isfinite().all())


def test_captured_and_replayed_on_other_ids():
    ids, w, dy = random_ids(3000, 700), make(700, 128, dtype=torch.bfloat16).requires_grad_(), make(3000, 128, dtype=torch.bfloat16, seed=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.embedding(ids, w), w, dy)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.embedding(ids, w)
            dw, = torch.autograd.grad(y, w, dy)
        graphs.append((graph, y, dw))
    for seed in (5, 6):
        ids.copy_(random_ids(3000, 700, seed, 0.2))
        for graph, y, dw in graphs:
            graph.replay()
            assert torch.equal(y, w[ids])
            check_grad(dw, ids, dy, 700, 1.0)


def test_differences():
    # the gradient against differences of a weighted sum of the outputs
    ids, w, dy = random_ids(50, 7), make(7, 12).requires_grad_(), make(50, 12, seed=1)
    dw, = torch.autograd.grad(ops.embedding(ids, w, scale=3.0), w, dy)
    step = 2.0 ** -4
    for i, j in ((0, 0), (3, 5), (6, 11)):
        bump = torch.zeros_like(w)
        bump[i, j] = step
        with torch.no_grad():
            high, low = ((ops.embedding(ids, w + s * bump, scale=3.0).double() * dy.double()).sum() for s in (1, -1))
        # linear in w: what is left are roundings of w + step (2^-24 of at most 4) and of the outputs, 50 of them
        assert abs(float((high - low) / (2 * step)) - float(dw[i, j])) <= 50 * 3 * 8 * 2 * U / step * float(dy.abs().max())
