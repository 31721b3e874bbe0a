"""Rotary positions on the GPU against the formula in 64 bits: layouts, part of the head, positions, gradients, strides.

Tolerances: a result is two products and a sum in fp32 (three roundings, 2^-22 of the terms' sizes covers them) and its own rounding, half a
step of its type (fp16's subnormals have a fixed step).
"""
import pytest
import torch

import _model_ops as plain
from _model_ops import rounding

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def ops():
    from nangila import ops as o

    return o


def near(got, x, table, positions, layout, inverse=False):
    want, size = plain.turned(x, table, positions, layout, inverse)
    slack = rounding(want, got.dtype) + size * 2.0 ** -22
    assert ((got.double() - want).abs() <= slack).all()
    rest = 2 * table.size(1)
    assert torch.equal(got[..., rest:], x[..., rest:])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,hq,hk,d,rot", [(1, 1, 1, 1, 2, 2), (2, 5, 4, 2, 128, 128), (3, 17, 12, 12, 64, 64), (1, 33, 3, 1, 80, 80), (2, 7, 8, 2, 128, 64), (2, 3, 5, 5, 96, 24),
                                             (1, 9, 4, 1, 256, 32), (4, 1, 16, 4, 128, 128), (1, 6, 2, 2, 34, 18), (1, 2, 1, 1, 4096, 4096), (2, 300, 4, 4, 32, 8)])
def test_against_the_formula(b, t, hq, hk, d, rot, dtype, layout):
    g = torch.Generator(device="cuda").manual_seed(b * t + d)
    table = ops().rotary_table(t + 50, rot, device="cuda")
    q = torch.randn(b, t, hq, d, device="cuda", generator=g).to(dtype).requires_grad_()
    k = torch.randn(b, t, hk, d, device="cuda", generator=g).to(dtype).requires_grad_()
    pos = torch.randint(0, t + 50, (b, t), device="cuda", generator=g)
    for given, at in ((None, torch.arange(t, device="cuda")[None]), (pos, pos), (pos.int(), pos), (pos[0], pos[:1]), (pos[:1], pos[:1])):
        oq, ok = ops().rotary(q, k, table, positions=given, layout=layout)
        near(oq, q.detach(), table, at, layout)
        near(ok, k.detach(), table, at, layout)
        dq, dk = torch.randn(q.shape, device="cuda", generator=g).to(dtype), torch.randn(k.shape, device="cuda", generator=g).to(dtype)
        gq, gk = torch.autograd.grad((oq, ok), (q, k), (dq, dk))
        near(gq, dq, table, at, layout, True)
        near(gk, dk, table, at, layout, True)
        assert torch.equal(ops().rotary(q, None, table, positions=given, layout=layout), oq)


def test_one_gradient_only_and_shared_heads():
    table = ops().rotary_table(8, 32, device="cuda")
    at = torch.arange(8, device="cuda")[None]
    q = torch.randn(2, 8, 4, 32, device="cuda", requires_grad=True)
    k = torch.randn(2, 8, 1, 32, device="cuda", requires_grad=True)
    oq, ok = ops().rotary(q, k.expand(2, 8, 4, 32), table)  # one head seen by four
    up = torch.randn(2, 8, 4, 32, device="cuda")
    gk, = torch.autograd.grad(ok, k, up, retain_graph=True)
    want, size = plain.turned(up, table, at, "interleaved", True)
    assert ((gk.double() - want.sum(2, keepdim=True)).abs() <= size.sum(2, keepdim=True) * 2.0 ** -20).all()
    gq, none = torch.autograd.grad(oq, (q, k), up, allow_unused=True)
    near(gq, up, table, at, "interleaved", True)
    assert none is None


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_strides_and_alignment(layout):
    """Slices of a joined projection, heads before the sequence, columns that start anywhere."""
    table = ops().rotary_table(20, 64, device="cuda")
    at = torch.arange(20, device="cuda")[None]
    joined = torch.randn(2, 20, 3, 6, 64, device="cuda").bfloat16()
    by_heads = torch.randn(2, 6, 20, 64, device="cuda").bfloat16().transpose(1, 2)
    odd = torch.randn(2, 20, 6, 67, device="cuda").bfloat16()[..., 3:]
    swapped = torch.randn(2, 20, 64, 6, device="cuda").bfloat16().transpose(2, 3)
    for q in (joined[:, :, 0], joined[:, :, 2], by_heads, odd, swapped):
        for k in (joined[:, :, 1], odd):
            oq, ok = ops().rotary(q, k, table, layout=layout)
            assert oq.is_contiguous() and ok.is_contiguous()
            near(oq, q, table, at, layout)
            near(ok, k, table, at, layout)
    wide = torch.arange(40, device="cuda").view(1, 40)[:, ::2]
    near(ops().rotary(joined[:, :, 0], None, ops().rotary_table(40, 64, device="cuda"), positions=wide, layout=layout), joined[:, :, 0],
         ops().rotary_table(40, 64, device="cuda"), wide, layout)


@pytest.mark.parametrize("d", [64, 36])
def test_positions_outside_the_table(d):
    table = ops().rotary_table(10, 32, device="cuda")
    q = torch.randn(1, 5, 2, d, device="cuda")
    pos = torch.tensor([0, 10, -1, 9, 2 ** 40], device="cuda")
    out = ops().rotary(q, None, table, positions=pos)
    good = torch.tensor([0, 3], device="cuda")
    near(out[:, good], q[:, good], table, pos[good][None], "interleaved")
    assert torch.isnan(out[0, [1, 2, 4], :, :32]).all() and torch.equal(out[..., 32:], q[..., 32:])


def test_values_that_are_not_finite_stay_with_their_pair():
    table = ops().rotary_table(4, 16, device="cuda")
    q = torch.randn(1, 4, 1, 16, device="cuda")
    clean = ops().rotary(q, None, table)
    q[0, 2, 0, 6] = float("inf")
    out = ops().rotary(q, None, table)
    keep = [i for i in range(16) if i not in (6, 7)]
    assert torch.equal(out[..., keep], clean[..., keep]) and not torch.isfinite(out[0, 2, 0, 6:8]).any()


def test_nothing_to_do():
    table = ops().rotary_table(4, 16, device="cuda")
    q = torch.empty(0, 4, 2, 16, device="cuda", requires_grad=True)
    k = torch.randn(0, 4, 0, 16, device="cuda")
    oq, ok = ops().rotary(q, k, table)
    oq.sum().backward()
    assert oq.shape == q.shape and ok.shape == k.shape and q.grad.shape == q.shape
    some = torch.randn(1, 4, 2, 16, device="cuda")
    oq, ok = ops().rotary(some, some[:, :, :0], table)
    assert ok.shape == (1, 4, 0, 16) and torch.equal(oq, ops().rotary(some, None, table))
    oq, ok = ops().rotary(some[:, :, :0], some, table)
    assert torch.equal(ok, ops().rotary(some, None, table))


def test_captured_and_replayed_on_new_positions():
    table = ops().rotary_table(100, 64, device="cuda")
    q = torch.randn(2, 3, 4, 64, device="cuda", requires_grad=True)
    k = torch.randn(2, 3, 1, 64, device="cuda")
    pos = torch.zeros(2, 3, dtype=torch.long, device="cuda")

    def run():
        oq, ok = ops().rotary(q, k, table, positions=pos)
        return (oq, ok) + torch.autograd.grad(oq, q, torch.ones_like(oq))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    pos.copy_(torch.randint(0, 100, (2, 3), device="cuda"))
    graph.replay()
    for a, b in zip(held, run()):
        assert torch.equal(a, b)


def test_no_second_derivative():
    q = torch.randn(1, 2, 1, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="again"):
        torch.autograd.grad(ops().rotary(q, None, ops().rotary_table(2, 8, device="cuda")).sum(), q, create_graph=True)
