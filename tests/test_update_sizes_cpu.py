"""Updates of any size on the CPU: their norm is taken of values near one, whatever their size."""
import pytest
import torch

import _model_ops as plain
from nangila import ops
from nangila.optim import Muon

COEF = (3.4445, -4.7750, 2.0315)
# as for other sizes: the bf16 result's 2^-8, and fp32 products of 20 terms carried up by 485 at most
TOL = 2.0 ** -8 + 485 * 20 * 2.0 ** -24


@pytest.mark.parametrize("size", [1e-36, 1e-25, 1e-12, 1.0, 1e20, 1e38])
def test_sizes_of_the_input(size):
    u = torch.randn(12, 20)
    u = u / u.abs().max()
    want = plain.orthogonal(u, 5, COEF, 1e-30)
    got = ops.orthogonalize(u * size, eps=1e-36)
    assert float(torch.linalg.vector_norm(got.double() - want)) <= TOL * float(torch.linalg.vector_norm(want))


def test_a_step_with_a_large_gradient():
    p, g, m = torch.zeros(12, 20), torch.randn(12, 20), torch.zeros(12, 20)
    want = plain.orthogonal(g, 5, COEF, 1e-30)
    ops.muon_step([p], [g / g.abs().max() * 1e38], [m], lr=1.0, scale=None)
    assert float(torch.linalg.vector_norm(p.double() + want)) <= TOL * float(torch.linalg.vector_norm(want))


def test_values_that_are_not_finite_and_zeros():
    u = torch.randn(6, 8)
    assert (ops.orthogonalize(torch.zeros(6, 8)) == 0).all()
    for bad in (float("nan"), float("inf")):
        v = u.clone()
        v[2, 3] = bad
        assert torch.isnan(ops.orthogonalize(v)).any()


def test_ordinary_updates_are_what_they_were():
    for size in (1e-9, 1e-4, 1.0, 300.0):
        u = torch.randn(12, 20) * size
        x = u / torch.linalg.vector_norm(u).clamp(min=1e-7)
        for _ in range(5):
            gram = x @ x.mT
            x = COEF[0] * x + (COEF[1] * gram + COEF[2] * (gram @ gram)) @ x
        assert torch.equal(ops.orthogonalize(u), x.bfloat16())


def test_an_eps_that_float32_cannot_divide_by_is_refused():
    """Zeros over it would not be numbers, and with them the parameters."""
    z = torch.zeros(6, 8)
    p = torch.ones(6, 8)
    for eps in (1e-300, 1e-46, 1e-37, 0.0, -1.0, float("inf"), float("nan")):
        for call in (lambda: ops.orthogonalize(z, eps=eps), lambda: ops.muon_step([p], [z], [z.clone()], lr=0.1, eps=eps), lambda: Muon([torch.nn.Parameter(p)], eps=eps)):
            with pytest.raises(ValueError, match="nangila: eps"):
                call()
    assert (ops.orthogonalize(z, eps=1e-36) == 0).all() and (p == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(6, 8), (200, 65536), (300, 200)])
def test_zeros_over_the_smallest_eps_on_the_gpu(m, n):
    assert (ops.orthogonalize(torch.zeros(m, n, device="cuda"), eps=1e-36) == 0).all()
