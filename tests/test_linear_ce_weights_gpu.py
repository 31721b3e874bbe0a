"""Losses weighted one by one: what a row of little weight gives to the classes that only such rows touch keeps its digits."""
import pytest
import torch

from tests._head_bounds import check_grads_anywhere
from tests._vocab_ops import head
from tests.test_linear_ce_kernel_gpu import DEV, run

pytestmark = pytest.mark.gpu


def two_kinds(n, d, rows, dtype, seed=0):
    """Every third row is of the first half of the classes, the others of the second: a first column that sets them e^80 apart."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, w = torch.randn(n, d, device=DEV, generator=g), torch.randn(rows, d, device=DEV, generator=g) / d ** 0.5
    heavy = torch.arange(n, device=DEV) % 3 == 0
    x[:, 0] = torch.where(heavy, 8.0, -8.0)
    w[:, 0] = torch.where(torch.arange(rows, device=DEV) < rows // 2, 5.0, -5.0)
    t = torch.randint(0, rows // 2, (n,), device=DEV, generator=g) + torch.where(heavy, 0, rows // 2)
    return x.to(dtype), w.to(dtype), t, heavy


def lost_below(x, up, want):
    """Rows of x are held with what lies below half a step of fp16's smallest lost, 2^-38 of the largest |upstream x|, for each token and probability (and at least 2^-55 of the largest
    weight: they are not made larger without end)."""
    live = up != 0
    largest = float((x.double().abs().amax(1) * up.double().abs())[live].max())
    return max(2.0 ** -38 * largest, 2.0 ** -55 * float(up.abs().max())) * want["share"][:, None]


def expect(x, w, t, up, b=None):
    want = head(x, w, t, b, reduction="none", upstream=up)
    p = torch.softmax(x.double() @ w.double().T + (0.0 if b is None else b.double()), 1)
    want["share"] = (p - torch.nn.functional.one_hot(t, w.size(0))).abs().sum(0)  # of all tokens, by class
    return want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("apart", [14, 20, 28])
@pytest.mark.parametrize("n,d,rows", [(3, 64, 40), (60, 8, 90), (200, 72, 600), (300, 64, 500), (1500, 136, 1000)])
def test_rows_of_little_weight(n, d, rows, apart, dtype):
    x, w, t, heavy = two_kinds(n, d, rows, dtype)
    up = torch.where(heavy, 1024.0, 1024.0 * 2.0 ** -apart) * (1.0 + torch.rand(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)))
    up[1::5] *= -1.0
    want = expect(x, w, t, up)
    assert float(want["dw"].abs().max()) < 60000
    _, grads = run(x, w, t, None, up, reduction="none")
    check_grads_anywhere(grads, want, x, w, d, dtype, also=lost_below(x, up, want) if dtype == torch.float16 else 0.0)
    if apart == 20:
        # the same from the light rows alone, whose classes the others' probabilities do not reach
        light = (~heavy).nonzero().squeeze(1)
        _, alone = run(x[light], w, t[light], None, up[light], reduction="none")
        of_light = slice(rows // 2, rows)
        # (each of them off by the bound from the same values)
        over = (grads[1][of_light].double() - alone[1][of_light].double()).abs()
        tol = want["dw_size"] * (6 * 2.0 ** (-11 if dtype == torch.float16 else -8) * 1.02) + 3 * want["dw"].abs() * 2.0 ** (-11 if dtype == torch.float16 else -8) + 2.0 ** -22
        assert bool((over <= tol[of_light]).all())


@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 4000.0, 60000.0])
@pytest.mark.parametrize("n", [40, 300])
def test_rows_of_any_size(n, size):
    # x up to half precision's largest value, and far below one: what rows are made larger by leaves them below it
    d, rows = 16, 50
    x, w, t, _ = two_kinds(n, d, rows, torch.float16)
    x, w = (size * x.float() / x.float().abs().amax(1, keepdim=True)).half(), (w.float() / max(1.0, size)).half()
    up = 2.0 ** -8 * 2.0 ** -torch.linspace(0, 12, n, device=DEV)
    b = torch.randn(rows, device=DEV)
    want = expect(x, w, t, up, b)
    _, grads = run(x, w, t, b, up, reduction="none")
    check_grads_anywhere(grads, want, x, w, d, torch.float16, also=lost_below(x, up, want))


def test_rows_that_add_nothing_do_not_set_the_size():
    x, w, t, heavy = two_kinds(300, 64, 500, torch.float16)
    up = torch.where(heavy, 1024.0, 1024.0 * 2.0 ** -20)
    want = expect(x, w, t, up)
    want = head(x, w, torch.where(torch.arange(300, device=DEV) % 6 == 0, -100, t), reduction="none", upstream=up) | {"share": want["share"]}
    t[::6] = -100
    for held in (60000.0, float("inf"), float("nan")):
        x[::6] = held
        _, grads = run(x, w, t, None, up, reduction="none")
        check_grads_anywhere(grads, want, x, w, 64, torch.float16, also=2.0 ** -38 * 2048.0 * 8 * want["share"][:, None])
    # weights of zero, and none but zeros
    for weights in (torch.where(heavy, 0.0, up), torch.zeros(300, device=DEV)):
        _, grads = run(x.nan_to_num(0.0), w, t, None, weights, reduction="none")
        zero = head(x.nan_to_num(0.0), w, t, reduction="none", upstream=weights) | {"share": want["share"]}
        check_grads_anywhere(grads, zero, x, w, 64, torch.float16, also=2.0 ** -38 * 8 * want["share"][:, None])
        assert not grads[0][weights == 0].any()


def test_weights_below_half_precision_reach_a_bias_in_single():
    x, w, t, _ = two_kinds(300, 64, 500, torch.float16)
    b = torch.zeros(500, device=DEV)
    up = torch.full((300,), 1e-30, device=DEV)
    want = expect(x, w, t, up, b)
    _, grads = run(x, w, t, b, up, reduction="none")
    assert not grads[0].any() and not grads[1].any()
    check_grads_anywhere(grads, want, x, w, 64, torch.float16)


def test_several_groups_of_tokens():
    n, d, rows = 3200, 64, 300001
    x, w, t, heavy = two_kinds(n, d, rows, torch.float16)
    up = torch.where(heavy, 1024.0, 1024.0 * 2.0 ** -20)
    want = expect(x, w, t, up)
    _, grads = run(x, w, t, None, up, reduction="none")
    check_grads_anywhere(grads, want, x, w, d, torch.float16, also=lost_below(x, up, want))
