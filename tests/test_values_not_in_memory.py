"""Views that are negated only when they are read, and zeros without memory, give the same as tensors that hold those values."""
import pytest
import torch

from nangila import ops

neg, zeros = torch._neg_view, torch._efficientzerotensor


def test_a_step_writes_through_such_a_view_on_the_cpu():
    """CPU tensors take PyTorch's operations, which write through the view."""
    p, g, m = torch.randn(4, 6), torch.randn(4, 6), torch.zeros(4, 6)
    a, b = p.clone(), -p
    ops.muon_step([a], [g], [m.clone()], lr=0.1)
    ops.muon_step([neg(b)], [g], [m.clone()], lr=0.1)
    assert torch.equal(-b, a)


@pytest.mark.gpu
def test_negated_views():
    x, r, w = torch.randn(6, 136, device="cuda"), torch.randn(6, 136, device="cuda"), torch.randn(136, device="cuda")
    for got, want in zip(ops.add_rms_norm(neg(x), neg(r), neg(w)), ops.add_rms_norm(-x, -r, -w)):
        assert torch.equal(got, want)
    assert torch.equal(ops.rms_norm_fp8(neg(x), neg(w))[0].view(torch.uint8), ops.rms_norm_fp8(-x, -w)[0].view(torch.uint8))
    leaf, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    for a, b in zip(torch.autograd.grad(ops.rms_norm(neg(leaf), neg(wl)), (leaf, wl), neg(r)), torch.autograd.grad(ops.rms_norm(-leaf, -wl), (leaf, wl), -r)):
        assert torch.equal(a, b)
    q, table = torch.randn(2, 5, 3, 8, device="cuda"), ops.rotary_table(9, 8, device="cuda")
    at = -torch.arange(5, device="cuda")
    for a, b in zip(ops.rotary(neg(q), neg(q[:, :, :1]), neg(table), positions=neg(at)), ops.rotary(-q, -q[:, :, :1], -table, positions=-at)):
        assert torch.equal(a, b)
    assert torch.equal(ops.orthogonalize(neg(x)), ops.orthogonalize(-x))
    ps, ms = [torch.zeros_like(x) for _ in range(2)], [torch.zeros_like(x) for _ in range(2)]
    ops.muon_step(ps[:1], [neg(r)], ms[:1], lr=0.1), ops.muon_step(ps[1:], [-r], ms[1:], lr=0.1)
    assert torch.equal(ps[0], ps[1]) and torch.equal(ms[0], ms[1])
    for p, m in ((neg(x), ms[0]), (x, neg(ms[0]))):
        keep = p.clone(), m.clone()
        with pytest.raises(ValueError, match="nangila"):
            ops.muon_step([p], [r], [m], lr=0.1)
        assert torch.equal(p, keep[0]) and torch.equal(m, keep[1])


@pytest.mark.gpu
def test_zeros_without_memory():
    x, w = torch.randn(6, 136, device="cuda"), torch.randn(136, device="cuda")
    none, full = zeros(6, 136, device="cuda"), torch.zeros(6, 136, device="cuda")
    for got, want in zip(ops.add_rms_norm(none, x, w), ops.add_rms_norm(full, x, w)):
        assert torch.equal(got, want)
    assert torch.equal(ops.rms_norm(none, w), full)
    q = torch.randn(2, 5, 3, 8, device="cuda", requires_grad=True)
    table = ops.rotary_table(5, 8, device="cuda")
    g, = torch.autograd.grad(ops.rotary(q, None, table), q, zeros(2, 5, 3, 8, device="cuda"))
    assert torch.equal(g, torch.zeros_like(q))
    leaf, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    for v in torch.autograd.grad(ops.rms_norm(leaf, wl), (leaf, wl), none):
        assert torch.equal(v, torch.zeros_like(v))
    assert torch.equal(ops.orthogonalize(none).float(), full)
    p = torch.zeros(6, 136, device="cuda")
    ops.muon_step([p], [none], [torch.zeros(6, 136, device="cuda")], lr=0.1)
    assert torch.equal(p, full)
    with pytest.raises(ValueError, match="nangila"):
        ops.muon_step([none], [x], [torch.zeros(6, 136, device="cuda")], lr=0.1)
