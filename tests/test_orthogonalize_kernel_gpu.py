"""Newton-Schulz orthogonalisation and the Muon step on the GPU against the formulas in 64 bits.

Tolerance of a result, in the 2-norm of all its elements, relative. Each product's operands are rounded to fp16: half a step is u = 2^-11, u / sqrt(3) = 2.8e-4
in the mean. In a step, five such roundings stand behind b A X (X twice and A, B, X once) and seven behind c A^2 X; with singular values near one they come to
2.8e-4 * sqrt(4.775^2 * 5 + 2.0315^2 * 7) = 3.3e-3 of X, independent of one another, and the map's slope is about one in the mean where it has
settled: five steps come to sqrt(5) * 3.3e-3 = 7.5e-3. The bf16 result adds at most 2^-8. (a X is formed from 22 bits, 485 * 2^-22 = 1.2e-4.)
"""
import pytest
import torch

import _model_ops as plain

pytestmark = pytest.mark.gpu
COEF = (3.4445, -4.7750, 2.0315)
TOL = 7.5e-3 + 2.0 ** -8
EPS = 1e-7


def ops():
    from nangila import ops as o

    return o


def rel(got, want):
    return float(torch.linalg.vector_norm(got.double() - want) / torch.linalg.vector_norm(want))


def gradient(m, n, seed=0, dtype=torch.float32, fall=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + m * 31 + n)
    k = min(m, n)
    left = torch.randn(m, k, device="cuda", generator=g) * (1.0 + torch.arange(k, device="cuda")).pow(-fall)
    return ((left @ torch.randn(k, n, device="cuda", generator=g) + 0.1 * torch.randn(m, n, device="cuda", generator=g)) * 1e-4).to(dtype)


SIZES = [(1, 1), (1, 7), (7, 1), (2, 3), (8, 8), (16, 64), (63, 65), (65, 63), (64, 64), (128, 128), (129, 127), (100, 1000), (1000, 100), (255, 257), (257, 255), (384, 256), (130, 515),
         (517, 259), (768, 768), (352, 128), (768, 2304), (1024, 640), (200, 4000), (4001, 136), (129, 2100), (128, 384), (385, 128), (40, 3001),
         (2900, 128), (128, 3073), (17, 769), (1, 65536), (65536, 1), (130, 30000), (30000, 136),
         (65536, 72)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n", SIZES)
def test_one_matrix(m, n, dtype):
    u = gradient(m, n, dtype=dtype) * (1.0 if dtype != torch.float16 else 64.0)
    out = ops().orthogonalize(u)
    assert out.shape == u.shape and out.dtype == torch.bfloat16 and out.is_contiguous()
    assert rel(out, plain.orthogonal(u, 5, COEF, EPS)) < TOL


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
@pytest.mark.parametrize("m,n", [(96, 160), (200, 72)])
def test_numbers_of_steps_and_a_schedule(m, n, steps):
    u = gradient(m, n)
    assert rel(ops().orthogonalize(u, steps=steps), plain.orthogonal(u, steps, COEF, EPS)) < TOL * max(1.0, (steps / 5) ** 0.5)
    rows = [(3.0 - 0.1 * i, -3.2 + 0.1 * i, 1.2) for i in range(steps)]
    assert rel(ops().orthogonalize(u, steps=steps, coefficients=rows), plain.orthogonal(u, steps, rows, EPS)) < TOL * max(1.0, (steps / 5) ** 0.5)


@pytest.mark.parametrize("fall", [0.0, 1.0, 2.0])
def test_spectra(fall):
    """Singular values that fall off fast: the small ones are carried up by a^5 and have to survive the roundings."""
    u = gradient(320, 512, fall=fall)
    out = ops().orthogonalize(u)
    want = plain.orthogonal(u, 5, COEF, EPS)
    assert rel(out, want) < TOL
    s, w = torch.linalg.svdvals(out.double()), torch.linalg.svdvals(want)
    assert float((s - w).abs().max()) < 5 * TOL


def test_a_matrix_of_low_rank_keeps_its_rank():
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.randn(256, 4, device="cuda", generator=g) @ torch.randn(4, 384, device="cuda", generator=g)
    out = ops().orthogonalize(u)
    assert rel(out, plain.orthogonal(u, 5, COEF, EPS)) < TOL
    assert float(torch.linalg.svdvals(out.double())[4]) < 0.05


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1.0, 1e12, 1e30])
def test_sizes_of_the_input(size):
    u = gradient(64, 96) / 1e-4 * size
    assert rel(ops().orthogonalize(u, eps=1e-35), plain.orthogonal(u, 5, COEF, 1e-35)) < TOL


def test_below_eps_and_zero():
    u = gradient(64, 96)
    u = u / u.norm() * 1e-9
    assert rel(ops().orthogonalize(u), plain.orthogonal(u, 5, COEF, EPS)) < TOL
    assert (ops().orthogonalize(torch.zeros(40, 30, device="cuda")) == 0).all()


def test_many_matrices_at_once_are_what_each_is_alone():
    shapes = [(96, 160), (160, 96), (96, 160), (33, 50), (96, 160)] * 30  # more of a shape than go together
    many = [gradient(m, n, seed=i) for i, (m, n) in enumerate(shapes)]
    together = ops().orthogonalize(many)
    for i in (0, 1, 2, 3, 77, 149):
        assert torch.equal(together[i], ops().orthogonalize(many[i]))
    stack = torch.stack([v for v in many if v.shape == (96, 160)])
    out = ops().orthogonalize(stack)
    assert out.shape == stack.shape and torch.equal(out[1], together[2])
    assert ops().orthogonalize([]) == [] and ops().orthogonalize(stack[:0]).shape == (0, 96, 160)
    mixed = ops().orthogonalize([many[0], many[0].bfloat16(), many[0].cpu()])
    assert torch.equal(mixed[0], together[0]) and mixed[2].device.type == "cpu" and rel(mixed[2].cuda(), together[0].double()) < 2 * TOL


@pytest.mark.parametrize("m,n", [(96, 130), (500, 100), (300, 200), (200, 2500)])
def test_a_matrix_that_is_not_finite_spoils_no_other(m, n):
    many = [gradient(m, n, seed=i) for i in range(5)]
    clean = ops().orthogonalize(many)
    many[1][3, 4] = float("nan")
    many[3][0, 0] = float("inf")
    out = ops().orthogonalize(many)
    for i in (0, 2, 4):
        assert torch.equal(out[i], clean[i])
    assert torch.isnan(out[1]).any() and not torch.isfinite(out[3].float()).all()


def test_layouts_and_same_bits():
    u = gradient(300, 200)
    want = ops().orthogonalize(u)
    assert torch.equal(ops().orthogonalize(u.t().contiguous().t()), want)
    wide = torch.zeros(300, 208, device="cuda")
    wide[:, 3:203] = u
    assert torch.equal(ops().orthogonalize(wide[:, 3:203]), want)
    off = torch.empty(60001, device="cuda")[1:].view(300, 200)
    off.copy_(u)
    assert torch.equal(ops().orthogonalize(off), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [ops().orthogonalize(u) for _ in range(10)]
    here = [ops().orthogonalize(u) for _ in range(10)]  # two streams at once
    torch.cuda.synchronize()
    for v in again + here:
        assert torch.equal(v, want)


def test_the_symmetric_halves_agree():
    """A matrix and its transpose take different operand layouts; the results are each other's transposes up to the roundings' order."""
    u = gradient(192, 320)
    assert rel(ops().orthogonalize(u.t().contiguous()).t(), ops().orthogonalize(u).double()) < 2 * TOL


def muon_plain(p, g, m, lr, mu, nesterov, wd, scale):
    m = mu * m.double() + g.double()
    o = plain.orthogonal(g.double() + mu * m if nesterov else m, 5, COEF, EPS)
    r, c = p.shape
    s = {"spectral": max(1.0, r / c) ** 0.5, "rms": 0.2 * max(r, c) ** 0.5, None: 1.0}[scale]
    return p.double() * (1 - lr * wd) - lr * s * o, m, lr * s * float(torch.linalg.vector_norm(o))


@pytest.mark.parametrize("nesterov,scale", [(True, "rms"), (False, "spectral"), (True, None)])
@pytest.mark.parametrize("ptype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n", [(96, 160), (161, 97), (128, 256), (256, 384), (301, 203), (130, 1029), (600, 152)])
def test_muon_step(m, n, ptype, nesterov, scale):
    g = torch.Generator(device="cuda").manual_seed(m)
    ps = [0.1 * torch.randn(m, n, device="cuda", generator=g).to(ptype) for _ in range(3)]
    ms = [torch.zeros(m, n, device="cuda") for _ in range(3)]
    for step in range(3):
        gs = [(gradient(m, n, seed=step * 10 + i) * 100).to(ptype) for i in range(3)]
        want = [muon_plain(p, gr, mo, 0.02, 0.9, nesterov, 0.1, scale) for p, gr, mo in zip(ps, gs, ms)]
        ops().muon_step(ps, gs, ms, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=scale)
        for p, mo, (wp, wm, size) in zip(ps, ms, want):
            # the update's error, and the parameter's rounding (the update is not rounded to bf16 on the way)
            slack = size * 7.5e-3 + float(torch.linalg.vector_norm(wp)) * plain.half_step(ptype)
            assert float(torch.linalg.vector_norm(p.double() - wp)) < slack
            assert rel(mo, wm) < 2.0 ** -22


@pytest.mark.parametrize("rows,cols", [(96, 160), (160, 96), (1000, 104), (264, 200), (200, 2000)])
def test_muon_step_of_unaligned_tensors_and_captured(rows, cols):
    hold = [torch.randn(rows * cols + 1, device="cuda") for _ in range(3)]
    p, g, m = (h[1:].view(rows, cols) for h in hold)
    want, wm, size = muon_plain(p, g, m, 0.02, 0.95, True, 0.0, "rms")
    keep = p.clone(), m.clone()
    ops().muon_step([p], [g], [m], lr=0.02)
    assert float(torch.linalg.vector_norm(p.double() - want)) < size * 7.5e-3 + 1e-4
    once = p.clone(), m.clone()
    p.copy_(keep[0]), m.copy_(keep[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops().muon_step([p], [g], [m], lr=0.02)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p, once[0]) and torch.equal(m, once[1])


def test_two_captured_graphs_and_a_call_between_them():
    """Graphs have workspaces of their own: replays in any order, on streams of their own, give what a call gives."""
    us = [gradient(264, 320, seed=i) for i in range(2)] + [gradient(100, 600, seed=2)]
    want = [ops().orthogonalize(u) for u in us]
    graphs, held = [], []
    for u in us:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(ops().orthogonalize(u))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        between = ops().orthogonalize(us[0])
    torch.cuda.synchronize()
    for h, w in zip(held, want):
        assert torch.equal(h, w)
    assert torch.equal(between, want[0])


def test_orthogonal_update_of_a_step_by_differences():
    """The update does not depend on the gradient's size: its difference quotient along the gradient itself vanishes."""
    u = gradient(160, 200)
    a, b = ops().orthogonalize(u).double(), ops().orthogonalize(u * 1.5).double()
    assert rel(a, b) < 2 * TOL


def test_an_updated_parameter_is_seen_as_changed():
    w = torch.randn(8, 8, device="cuda", requires_grad=True)
    y = (w * w).sum()
    ops().muon_step([w.detach()], [torch.randn(8, 8, device="cuda")], [torch.zeros(8, 8, device="cuda")], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
