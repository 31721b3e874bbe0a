"""Subnormal numbers in norms, rotary positions and updates: kept, as PyTorch's operations keep them.

Tolerances: the results' own rounding (half a step, which is fixed among the subnormals), the relative error of the fp32 arithmetic as in the tests of each operator,
and for each fp32 operation on the way half a step of its own, 2^-150. Flushed values would be off by up to 2^-126.
"""
import pytest
import torch

import _model_ops as plain
from _model_ops import rounding

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -149
WIDE = [torch.float32, torch.bfloat16]  # fp16's subnormals are normal numbers of fp32


def ops():
    from nangila import ops as o

    return o


def small(g, dtype, *shape):
    """Values from 2^-133 to 2^-125: bf16's and fp32's subnormals, and the first normal numbers."""
    v = torch.randn(*shape, device="cuda", generator=g, dtype=torch.float64) * 2.0 ** -127
    return v.to(dtype)


def near(got, want, slack):
    return bool(((got.double() - want).abs() <= slack).all())


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("rows,d", [(5, 64), (4, 1001), (3, 4096), (2, 20000)])
def test_norm(rows, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(d)
    x, r = small(g, dtype, rows, d), small(g, dtype, rows, d)
    w = torch.randn(d, device="cuda", generator=g).to(dtype)
    y, h = ops().add_rms_norm(x, r, w)
    assert torch.equal(h, (x.double() + r.double()).to(dtype)) and (h != 0).any()
    # h / sqrt(1e-5): the sum of its squares is nothing beside eps
    want = plain.norm(h, w, 1e-5)
    assert near(y, want, rounding(want, dtype) + want.abs() * 2.0 ** -17 + 4 * STEP * (1 + w.double().abs()))
    # ordinary rows, results and gradients among the subnormals
    x = torch.randn(rows, d, device="cuda", generator=g).to(dtype).requires_grad_()
    w = small(g, dtype, d).requires_grad_()
    dy = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    y = ops().rms_norm(x, w)
    want = plain.norm(x.detach(), w.detach(), 1e-5)
    assert near(y, want, rounding(want, dtype) + want.abs() * 2.0 ** -17 + STEP)
    wx, _, sx, _ = plain.norm_grads(x.detach(), w.detach(), 1e-5, dy)
    dx, = torch.autograd.grad(y, x, dy)
    # 12 operations behind each result, and behind the mean as many as the row has values, divided by them; |unit| is below 8 here
    assert near(dx, wx, rounding(wx, dtype) + sx * 2.0 ** -17 + 32 * STEP)
    w = torch.randn(d, device="cuda", generator=g).to(dtype).requires_grad_()
    dy = small(g, dtype, rows, d)
    dx, dw = torch.autograd.grad(ops().rms_norm(x, w), (x, w), dy)
    wx, ww, sx, sw = plain.norm_grads(x.detach(), w.detach(), 1e-5, dy)
    assert near(dx, wx, rounding(wx, dtype) + sx * 2.0 ** -17 + 32 * STEP)
    assert near(dw, ww, rounding(ww, dtype) + sw * 2.0 ** -16 + 2 * rows * STEP)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("d,rot", [(64, 64), (20, 8), (7, 6)])
def test_rotary(d, rot, dtype, layout):
    g = torch.Generator(device="cuda").manual_seed(d)
    q, table = small(g, dtype, 2, 9, 3, d), ops().rotary_table(9, rot, device="cuda")
    want, size = plain.turned(q, table, torch.arange(9, device="cuda")[None], layout)
    got = ops().rotary(q, None, table, layout=layout)
    assert near(got, want, rounding(want, dtype) + size * 2.0 ** -21 + 2 * STEP)
    assert torch.equal(got[..., rot:], q[..., rot:])


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("m,n", [(96, 160), (160, 96), (7, 33), (300, 200), (130, 1029)])
def test_parameters_and_momenta(m, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(m)
    p, grad, mom = small(g, dtype, m, n), small(g, dtype, m, n), small(g, torch.float32, m, n)
    keep = p.clone()
    want = grad.double() + 0.5 * mom.double()
    ops().muon_step([p], [grad], [mom], lr=0.0, momentum=0.5)
    assert torch.equal(p, keep) and (p != 0).any()
    assert near(mom, want, want.abs() * 2.0 ** -24 + STEP)


@pytest.mark.parametrize("m,n", [(128, 3000), (3000, 120), (300, 700), (700, 301)])
def test_updates_whose_norm_is_beyond_fp32(m, n):
    """An update's size does not matter, up to the largest numbers: what they are multiplied by is subnormal then."""
    g = torch.Generator(device="cuda").manual_seed(m)
    u = torch.randn(m, n, device="cuda", generator=g)
    u = u / u.abs().max() * 3e38
    want = plain.orthogonal(u / 1e38, 5, (3.4445, -4.7750, 2.0315), 1e-7)
    # as for any other update: the fp16 operands' roundings, and the bf16 result's
    assert float(torch.linalg.vector_norm(ops().orthogonalize(u).double() - want) / torch.linalg.vector_norm(want)) < 7.5e-3 + 2.0 ** -8
