"""What the updates' kernels lose against the formula in 64 bits, held to what their stated roundings cost (``_update_roundings``), and the variants that large matrices
and long lists take.

Tolerance. The restatement makes the kernels' roundings on the same input, with sums in 64 bits; its error against the formula is what the design costs there. The
kernels add up in fp32, in another order, which turns single roundings the other way: another draw of errors of the same size, whose norm over thousands of
elements hardly moves (restated with fp32 sums: 7 % at most over 120 inputs of 16 x 64 to 700 x 900). 1.25 times it is allowed, and 1e-4 for the fp32 sums themselves: 4096 values are
256 additions of the accumulator, 256 * 2^-24 = 1.5e-5, six of them weighted by the coefficients behind each result. A result in bf16 is off by half a step more, evenly spread: 2^-8 / sqrt(3).
"""
import pytest
import torch

import _model_ops as plain
from _update_roundings import rounded
from nangila import ops

COEF = (3.4445, -4.7750, 2.0315)
FIVE = [COEF] * 5
EPS = 1e-7
BF16 = 2.0 ** -8 / 3.0 ** 0.5


def rel(got, want):
    return float(torch.linalg.vector_norm(got.double() - want) / torch.linalg.vector_norm(want))


def update(m, n, fall, seed=0, device="cuda"):
    """Singular values that fall off as a power, and a little noise; 2: without it, so that they reach far down."""
    g = torch.Generator(device=device).manual_seed(seed * 7919 + m * 31 + n)
    left = torch.randn(m, min(m, n), device=device, generator=g) * (1.0 + torch.arange(min(m, n), device=device)).pow(-fall)
    u = left @ torch.randn(min(m, n), n, device=device, generator=g)
    return (u + (0.1 if fall < 1.5 else 0.0) * torch.randn(m, n, device=device, generator=g)) * 1e-4


def allowed(u, want):
    return 1.25 * rel(rounded(u, FIVE, EPS), want) + 1e-4


def unrounded(us):
    """The results in fp32: what a step of size one takes zeros to."""
    ps, ms = [torch.zeros_like(u) for u in us], [torch.zeros_like(u) for u in us]
    ops.muon_step(ps, us, ms, lr=1.0, momentum=0.0, scale=None)
    return [-p for p in ps]


@pytest.mark.parametrize("m,n,fall", [(300, 200, 0.0), (320, 512, 0.5), (320, 512, 2.0), (100, 1000, 0.5), (100, 1000, 2.0)])
def test_the_bound_tells_a_lost_half_and_coarser_operands(m, n, fall):
    """Mistakes planted in the restatement: X without its low half, operands in bf16."""
    u = update(m, n, fall, device="cpu")
    want = plain.orthogonal(u, 5, COEF, EPS)
    assert rel(rounded(u, FIVE, EPS, product=torch.float32), want) < allowed(u, want)
    assert rel(rounded(u, FIVE, EPS, low=False), want) > allowed(u, want)
    assert rel(rounded(u, FIVE, EPS, operand=torch.bfloat16), want) > 3 * allowed(u, want)


# The first five stay on the SMs, in one CTA or a cluster; 2051 x 300, 200 x 4000 and 4001 x 136 have the K of their Gram matrix split over clusters of four.
@pytest.mark.gpu
@pytest.mark.parametrize("fall", [0.0, 0.5, 2.0])
@pytest.mark.parametrize("m,n", [(128, 128), (352, 128), (100, 1000), (1024, 128), (63, 65), (300, 200), (320, 512), (517, 259), (768, 768), (2051, 300), (200, 4000), (4001, 136)])
def test_one_update(m, n, fall):
    u = update(m, n, fall)
    want = plain.orthogonal(u, 5, COEF, EPS)
    most = allowed(u, want)
    assert rel(unrounded([u])[0], want) < most
    assert rel(ops.orthogonalize(u), want) < most + BF16


# 2305 x 2177: one tile a pair of CTAs in the symmetric products (45 of 256 x 256 for 74 pairs), two in the others (90); three of it: two in the symmetric ones.
# 20 of 700 x 900: 120 and 240 tiles of pairs, several matrices in a launch. 30 of 381 x 301: tiles of 128 x 128, two of them a CTA, in the symmetric
# products (180 for 148 CTAs) and in the others (270).
@pytest.mark.gpu
@pytest.mark.parametrize("m,n,count", [(2305, 2177, 1), (2177, 2305, 1), (2177, 2305, 3), (700, 900, 20), (901, 700, 20), (381, 301, 30), (301, 381, 30)])
def test_many_tiles_a_cta(m, n, count):
    us = [update(m, n, 0.5, seed=i) for i in range(count)]
    fine, out = unrounded(us), ops.orthogonalize(us)
    for i in sorted({0, count // 2, count - 1}):
        want = plain.orthogonal(us[i], 5, COEF, EPS)
        most = allowed(us[i], want)
        assert rel(fine[i], want) < most and rel(out[i], want) < most + BF16
    for a, b in zip(out, ops.orthogonalize(us)):
        assert torch.equal(a, b)
    for a, b in zip(fine, out):  # the same but for the last rounding
        assert torch.equal(a.bfloat16(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,count", [(700, 900, 20), (301, 381, 30)])
def test_a_matrix_that_is_not_finite_spoils_no_other(m, n, count):
    us = [update(m, n, 0.5, seed=i) for i in range(count)]
    clean = ops.orthogonalize(us)
    us[3][m - 1, 0], us[count - 1][0, n - 1] = float("nan"), float("inf")
    out = ops.orthogonalize(us)
    for i in range(count):
        assert torch.equal(out[i], clean[i]) if i not in (3, count - 1) else not torch.isfinite(out[i].float()).all()


# 20 of 701 x 515: 180 tiles of pairs in the last product, three a pair, parameters read and written a value at a time; 520 x 704: runs of four; 30 of 384 x 300:
# 270 tiles of 128 x 128, two a CTA.
@pytest.mark.gpu
@pytest.mark.parametrize("ptype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,count", [(701, 515, 20), (520, 704, 20), (384, 300, 30), (2305, 2177, 1)])
def test_a_step_of_many_tiles_a_cta(m, n, count, ptype):
    g = torch.Generator(device="cuda").manual_seed(m)
    held = [torch.randn(m * n + 64, device="cuda", generator=g).mul_(0.1).to(ptype) for _ in range(count)]
    after = [h[m * n:].clone() for h in held]
    ps, ms = [h[:m * n].view(m, n) for h in held], [torch.randn(m, n, device="cuda", generator=g) * 1e-4 for _ in range(count)]
    gs = [(update(m, n, 0.5, seed=i) * 100).to(ptype) for i in range(count)]
    old_p, old_m = [p.clone() for p in ps], [v.clone() for v in ms]
    ops.muon_step(ps, gs, ms, lr=0.02, momentum=0.9, weight_decay=0.1)
    rate = 0.02 * 0.2 * max(m, n) ** 0.5
    for i in sorted({0, 1, count // 2, count - 1} & set(range(count))):
        wm = 0.9 * old_m[i].double() + gs[i].double()
        u = gs[i].double() + 0.9 * wm
        o = plain.orthogonal(u, 5, COEF, EPS)
        want = old_p[i].double() * (1 - 0.02 * 0.1) - rate * o
        assert rel(ms[i], wm) < 2.0 ** -22
        slack = rate * float(torch.linalg.vector_norm(o)) * allowed(u, o) + float(torch.linalg.vector_norm(want)) * plain.half_step(ptype)
        assert float(torch.linalg.vector_norm(ps[i].double() - want)) < slack
    for h, a in zip(held, after):
        assert torch.equal(h[m * n:], a)
