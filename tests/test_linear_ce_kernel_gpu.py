"""The head's loss and its gradients against the formulas in 64 bits."""
import pytest
import torch

from nangila import ops
from tests._model_ops import half_step, rounding
from tests._vocab_ops import head

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def inputs(n, d, rows, dtype=torch.bfloat16, classes=None, bias=None, ignored=0.0, sure=6.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    classes = rows if classes is None else classes
    w = (torch.randn(rows, d, device=DEV, generator=g) / d ** 0.5).to(dtype)
    targets = torch.randint(0, classes, (n,), device=DEV, generator=g)
    known = w[targets].float()
    x = torch.randn(n, d, device=DEV, generator=g) + sure * torch.rand(n, 1, device=DEV, generator=g) * known / known.square().sum(-1, keepdim=True).clamp(min=0.1)
    if ignored:
        targets = torch.where(torch.rand(n, device=DEV, generator=g) < ignored, -100, targets)
    b = None if bias is None else (0.5 * torch.randn(rows, device=DEV, generator=g)).to(bias)
    return x.to(dtype), w, targets, b


def z_error(want, d):
    """How far a logit may be off: products of 16 at a time summed in float32, with what hardware may cut off instead of rounding (2^-22), and the bias."""
    size = float(want["z_size"].amax()) if want["z_size"].numel() else 0.0
    return (d / 16 + 17) * 2.0 ** -22 * size


def exp_error(want, d, rows):
    """Relative, of exp(z - lse) before its rounding: both logits, their products with log2(e), the exponential (2^-22), and the row's sum."""
    return 2 * z_error(want, d) + 6 * want["z_most"] * 2 * U + 2.0 ** -21 + (140 + rows / 64) * U


def check_losses(got, want, d, rows):
    # a sum's relative error is an absolute one of its logarithm, and the logarithm's own few steps
    tol = exp_error(want, d, rows) + 8 * U * (want["losses"].abs() + want["z_most"])
    err = (got.double().reshape(-1) - want["losses"]).abs()
    assert got.dtype == torch.float32
    assert torch.equal(got.reshape(-1).isnan(), want["losses"].isnan()) and bool((err <= tol)[~want["losses"].isnan()].all()), (err - tol).max()


def check_grads(grads, want, x, w, d, dtype):
    rows, n = w.size(0), x.numel() // d
    hs, exp = half_step(dtype), exp_error(want, d, rows)
    tiny = 2.0 ** -39 if dtype == torch.float16 else 2.0 ** -100  # fp16's subnormal steps under 2^15
    dx, dw = grads[0].double().reshape(-1, d), grads[1].double()
    # E's rounding, its error before that, the products' sums, the row's factor
    tol = want["dx_size"] * (hs * (1 + 2 * hs) + exp + (rows / 16 + 17) * 2.0 ** -22 + 8 * U) + tiny * want["u_size"] * w.double().abs().sum(0) + rounding(want["dx"], dtype) * 1.01
    assert bool(((dx - want["dx"]).abs() <= tol).all()), ("dx", ((dx - want["dx"]).abs() - tol).max())
    # as before, and the rounding of x times its row's factor
    tol = want["dw_size"] * (2 * hs * (1 + 2 * hs) + exp + (n / 16 + 17) * 2.0 ** -22 + 8 * U) + tiny * want["x_size"] + rounding(want["dw"], dtype) * 1.01
    assert bool(((dw - want["dw"]).abs() <= tol).all()), ("dw", ((dw - want["dw"]).abs() - tol).max())
    if len(grads) > 2:
        tol = want["db_size"] * (hs * (1 + 2 * hs) + exp + (n + 8) * U) + tiny * want["u_size"] + rounding(want["db"], grads[2].dtype) * 1.01
        assert bool(((grads[2].double() - want["db"]).abs() <= tol).all()), ("db", ((grads[2].double() - want["db"]).abs() - tol).max())


def run(x, w, targets, b=None, upstream=None, **options):
    leaves = [t.detach().clone().requires_grad_() for t in (x, w) + (() if b is None else (b,))]
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], targets, bias=None if b is None else leaves[2], **options)
    return loss, torch.autograd.grad(loss, leaves, upstream)


SIZES = [(1, 8, 1), (1, 64, 5), (2, 33, 130), (5, 1, 7), (127, 64, 1000), (128, 72, 129), (129, 100, 257), (255, 128, 128), (256, 200, 1024), (300, 768, 3001), (1023, 264, 4099), (513, 1000, 700)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d,rows", SIZES)
def test_losses_alone(dtype, n, d, rows):
    x, w, t, _ = inputs(n, d, rows, dtype)
    want = head(x, w, t)
    losses = ops.linear_cross_entropy(x, w, t, reduction="none")
    check_losses(losses, want, d, rows)
    total = ops.linear_cross_entropy(x, w, t, reduction="sum")
    assert total.shape == () and abs(float(total) - float(losses.double().sum())) <= 2 * U * float(losses.double().sum())
    mean = ops.linear_cross_entropy(x, w, t)
    assert abs(float(mean) - float(losses.double().mean())) <= 2 * U * float(losses.double().mean())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,d,rows", SIZES)
def test_gradients(dtype, reduction, n, d, rows):
    classes = max(1, rows - 3)
    x, w, t, b = inputs(n, d, rows, dtype, classes, torch.float32 if n % 2 else dtype, ignored=0.2)
    if reduction == "none":
        upstream = torch.randn(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
    else:
        upstream = torch.tensor(512.0 if dtype == torch.float16 else 1.0, device=DEV)
    want = head(x, w, t, b, classes, reduction=reduction, upstream=upstream)
    loss, grads = run(x, w, t, b, upstream, num_classes=classes, reduction=reduction)
    if reduction == "none":
        check_losses(loss, want, d, rows)
    check_grads(grads, want, x, w, d, dtype)
    assert not grads[1][classes:].any() and not grads[2][classes:].any() and not grads[0][t == -100].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_tiles_of_a_cta(dtype):
    n, d, rows = 4000, 136, 20011
    x, w, t, _ = inputs(n, d, rows, dtype)
    up = torch.tensor(1024.0, device=DEV)
    want = head(x, w, t, upstream=up)
    _, grads = run(x, w, t, None, up)
    check_grads(grads, want, x, w, d, dtype)
    _, again = run(x, w, t, None, up)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_several_groups_of_tokens():
    # rows of E of 2 x 300032 bytes: a gigabyte holds 1536 of them, three groups
    n, d, rows = 3200, 64, 300001
    x, w, t, b = inputs(n, d, rows, bias=torch.float32, ignored=0.1)
    want = head(x, w, t, b)
    _, grads = run(x, w, t, b)
    check_grads(grads, want, x, w, d, torch.bfloat16)
    del want
    up = torch.rand(n, device=DEV)
    want = head(x, w, t, b, reduction="none", upstream=up)
    loss, grads = run(x, w, t, b, up, reduction="none")
    check_losses(loss, want, d, rows)
    check_grads(grads, want, x, w, d, torch.bfloat16)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_ignored_rows_hold_anything(reduction):
    x, w, t, _ = inputs(300, 64, 500)
    t[::3] = -100
    t[1::50] = 500  # no class
    up = torch.rand(300, device=DEV) + 0.5 if reduction == "none" else None
    clean, grads = run(x, w, t, None, up, reduction=reduction)
    x[::3] = float("nan")
    x[3::6] = float("inf")
    x[1::50] = float("nan")
    loss, dirty = run(x, w, t, None, up, reduction=reduction)
    assert torch.equal(loss.nan_to_num(7.0), clean.nan_to_num(7.0))
    assert all(torch.equal(a, b) and bool(a.isfinite().all()) for a, b in zip(grads, dirty))
    assert not grads[0][::3].any() and not grads[0][1::50].any()
    if reduction == "none":
        assert not loss[t == -100].any() and torch.equal(loss.isnan(), t == 500)
        want = head(torch.nan_to_num(x, 0.0, 0.0, 0.0), w, t, reduction="none", upstream=up)
        check_losses(loss, want, 64, 500)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_all_ignored_and_no_tokens(dtype):
    x, w, t, b = inputs(40, 64, 50, dtype, bias=torch.float32)
    t.fill_(7)
    for reduction, value in (("mean", float("nan")), ("sum", 0.0)):
        loss, grads = run(x, w, t, b, ignore_index=7, reduction=reduction)
        assert torch.equal(loss.nan_to_num(5.0), torch.tensor(value, device=DEV).nan_to_num(5.0)) and not any(g.any() for g in grads)
    for reduction, value in (("mean", float("nan")), ("sum", 0.0)):
        loss, grads = run(x[:0], w, t[:0], b, reduction=reduction)
        assert torch.equal(loss.nan_to_num(5.0), torch.tensor(value, device=DEV).nan_to_num(5.0)) and grads[0].shape == (0, 64) and not any(g.any() for g in grads)
    loss, grads = run(x[:0], w, t[:0], b, torch.empty(0, device=DEV), reduction="none")
    assert loss.shape == (0,) and not any(g.any() for g in grads)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_targets_far_below_the_largest_logit(dtype, reduction):
    # losses from 0 to some hundreds: references that a first pass over a tile cannot serve
    n, d, rows = 700, 64, 600
    x, w, t, _ = inputs(n, d, rows, dtype)
    other = (t + 1) % rows
    away = w[other].float()
    x[5:400:7] = (200 * away / away.square().sum(-1, keepdim=True))[5:400:7].to(dtype)
    up = torch.rand(n, device=DEV) + 0.5 if reduction == "none" else torch.tensor(512.0 if dtype == torch.float16 else 1.0, device=DEV)
    want = head(x, w, t, reduction=reduction, upstream=up)
    assert float(want["losses"].max()) > 100 and float(want["losses"].min()) < 5
    loss, grads = run(x, w, t, None, up, reduction=reduction)
    if reduction == "none":
        check_losses(loss, want, d, rows)
    else:
        assert abs(float(loss) - float(want["loss"])) <= exp_error(want, d, rows) + 8 * U * (float(want["losses"].abs().max()) + want["z_most"])
    check_grads(grads, want, x, w, d, dtype)


@pytest.mark.parametrize("n", [3, 100])
def test_targets_far_below_the_largest_logit_of_few_rows(n):
    x, w, t, _ = inputs(n, 64, 600)
    away = w[(t + 1) % 600].float()
    x[1::2] = (200 * away / away.square().sum(-1, keepdim=True))[1::2].to(torch.bfloat16)
    want = head(x, w, t)
    assert float(want["losses"].max()) > 100
    loss, grads = run(x, w, t)
    assert abs(float(loss) - float(want["loss"])) <= exp_error(want, 64, 600) + 8 * U * (float(want["losses"].abs().max()) + want["z_most"])
    check_grads(grads, want, x, w, 64, torch.bfloat16)


@pytest.mark.parametrize("n,d,rows", [(3, 2048, 600), (100, 1000, 5000), (300, 2056, 700)])
def test_targets_far_below_the_largest_logit_of_wide_rows(n, d, rows):
    x, w, t, _ = inputs(n, d, rows)
    away = w[(t + 1) % rows].float()
    x[1::2] = (200 * away / away.square().sum(-1, keepdim=True))[1::2].to(torch.bfloat16)
    want = head(x, w, t)
    assert float(want["losses"].max()) > 100
    loss, grads = run(x, w, t)
    assert abs(float(loss) - float(want["loss"])) <= exp_error(want, d, rows) + 8 * U * (float(want["losses"].abs().max()) + want["z_most"])
    check_grads(grads, want, x, w, d, torch.bfloat16)
    again, twice = run(x, w, t)
    assert torch.equal(loss, again) and all(torch.equal(a, b) for a, b in zip(grads, twice))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_far_apart(dtype):
    # each row's own gradient keeps its digits, whatever the others' weights are: row by row the same as alone, up to the roundings of E and of the result
    n, d, rows = 300, 64, 500
    x, w, t, _ = inputs(n, d, rows, dtype)
    up = 4096.0 * 2.0 ** -torch.linspace(0, 14, n, device=DEV) * torch.where(torch.arange(n, device=DEV) % 3 == 0, -1.0, 1.0)
    up[5] = 0.0
    want = head(x, w, t, reduction="none", upstream=up)
    _, grads = run(x, w, t, None, up, reduction="none")
    hs, exp = half_step(dtype), exp_error(want, d, rows)
    # (fp16's subnormal steps: of E, 2^-25 under 2^14 at least, of a row's weight; of the result)
    small = 2.0 ** -39 * up.abs().double()[:, None] * w.double().abs().sum(0) if dtype == torch.float16 else 0.0
    tol = want["dx_size"] * (hs * (1 + 2 * hs) + exp + (rows / 16 + 17) * 2.0 ** -22 + 8 * U) + small + rounding(want["dx"], dtype) * 1.01
    assert bool(((grads[0].double() - want["dx"]).abs() <= tol).all()) and not grads[0][5].any()
    check_grads(grads, want, x, w, d, dtype)


def test_rows_near_half_precisions_largest_value():
    # the row of the largest weight as it is: nothing is doubled on the way
    n, d, rows = 40, 8, 50
    x, w, t, _ = inputs(n, d, rows, torch.float16)
    x, w = (60000.0 * x.float() / x.float().abs().amax(1, keepdim=True)).half(), (w.float() * 1e-4).half()
    up = torch.full((n,), 2.0 ** -8, device=DEV)
    want = head(x, w, t, reduction="none", upstream=up)
    _, grads = run(x, w, t, None, up, reduction="none")
    check_grads(grads, want, x, w, d, torch.float16)
    _, grads = run(x, w, t, None, torch.tensor(2.0 ** -8, device=DEV), reduction="sum")
    check_grads(grads, want, x, w, d, torch.float16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("n,d,rows", [(1, 64, 3000), (7, 72, 2000), (64, 256, 9000), (65, 1, 300), (130, 33, 5000), (256, 512, 3001)])
def test_classes_of_single_tokens_keep_their_digits(dtype, reduction, n, d, rows):
    # what few tokens give to their own classes is rounded once, in the result
    x, w, t, _ = inputs(n, d, rows, dtype, ignored=0.3)
    t[0] = 1
    up = torch.rand(n, device=DEV) + 0.5 if reduction == "none" else None
    want = head(x, w, t, reduction="sum" if up is None else "none", upstream=up)
    live = t != -100
    u = torch.ones(n, device=DEV).double() if up is None else up.double()
    g = torch.softmax(x.double() @ w.double().T, 1) * u[:, None]
    own = torch.nn.functional.one_hot(t.clamp(min=0), rows).bool() & live[:, None]
    to_others = torch.where(live[:, None] & ~own, g, 0.0)
    to_own = torch.where(own, to_others.sum(1, keepdim=True), 0.0)
    hs, exp, sums = half_step(dtype), exp_error(want, d, rows), (2 * n / 16 + 25) * 2.0 ** -22
    # the others' roundings and the target's, which is folded into the row; two roundings one behind the other of x times its factor
    tol = (to_others.T @ x.double().abs()) * (2 * hs * (1 + 2 * hs) + exp + sums) + (to_own.T @ x.double().abs()) * (2 * hs * hs + exp + sums) + rounding(want["dw"], dtype) * 1.01
    tol = tol + (2.0 ** -39 if dtype == torch.float16 else 2.0 ** -100) * want["x_size"] + (2.0 ** -24 * want["u_size"] if dtype == torch.float16 else 0.0)
    _, (_, dw) = run(x, w, t, None, up, reduction=reduction)
    assert bool(((dw.double() - want["dw"]).abs() <= tol).all()), ((dw.double() - want["dw"]).abs() - tol).max()


def test_a_model_that_is_sure():
    # losses down to 1e-23: what is left of the gradient is the sum of the others, not 1 - p
    n, d, rows = 200, 64, 300
    x, w, t, _ = inputs(n, d, rows)
    known = w[t].float()
    x = (torch.linspace(5, 80, n, device=DEV)[:, None] * known / known.square().sum(-1, keepdim=True)).to(torch.bfloat16)
    want = head(x, w, t, reduction="sum")
    loss, grads = run(x, w, t, reduction="none", upstream=torch.ones(n, device=DEV))
    rel = (loss.double() - want["losses"]).abs() / want["losses"]
    assert float(want["losses"].min()) < 1e-20 and float(rel.max()) <= exp_error(want, d, rows) + 8 * U + 6 * 80 * 2 * U
    check_grads(grads, want, x, w, d, torch.bfloat16)
    check_grads(run(x, w, t, reduction="sum")[1], want, x, w, d, torch.bfloat16)


def test_classes_closed_by_a_bias_of_minus_infinity():
    x, w, t, b = inputs(150, 64, 300, bias=torch.float32)
    t = t % 100
    b[100:] = -float("inf")
    want = head(x, w[:100], t, b[:100])
    _, grads = run(x, w, t, b)
    check_grads((grads[0], grads[1][:100], grads[2][:100]), want, x, w[:100], 64, torch.bfloat16)
    assert not grads[1][100:].any() and not grads[2][100:].any()
    losses = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    check_losses(losses, head(x, w[:100], t, b[:100]), 64, 300)


def test_values_that_are_not_finite_are_told():
    x, w, t, _ = inputs(300, 64, 200)
    x[17, 3] = float("nan")
    losses = ops.linear_cross_entropy(x, w, t, reduction="none")
    assert bool(losses[17].isnan()) and int(losses.isnan().sum()) == 1
    loss, grads = run(x, w, t)
    assert bool(loss.isnan()) and bool(grads[0][17].isnan().all()) and int(grads[0].isnan().any(1).sum()) == 1 and bool(grads[1].isnan().any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_an_upstream_gradient_that_is_not_finite_stays_in_its_row(dtype, bad):
    x, w, t, b = inputs(300, 64, 500, dtype, bias=torch.float32)
    t[::3] = -100
    up = torch.rand(300, device=DEV) + 0.5
    _, clean = run(x, w, t, b, up, reduction="none")
    up[::3] = bad
    _, grads = run(x, w, t, b, up, reduction="none")
    assert all(torch.equal(got, want) for got, want in zip(grads, clean))
    up[100] = bad
    _, grads = run(x, w, t, b, up, reduction="none")
    assert int((~grads[0].isfinite()).any(1).sum()) == 1 and not grads[0][100].isfinite().any()
    others, hs = torch.arange(300, device=DEV) != 100, half_step(dtype)
    want = head(x, w, t, b, reduction="none", upstream=torch.where(others & (t != -100), up, 0.0))
    small = 2.0 ** -39 * want["u_size"] * w.double().abs().sum(0) if dtype == torch.float16 else 0.0
    tol = want["dx_size"] * (hs * (1 + 2 * hs) + exp_error(want, 64, 500) + (500 / 16 + 17) * 2.0 ** -22 + 8 * U) + small + rounding(want["dx"], dtype) * 1.01
    assert bool(((grads[0].double() - want["dx"]).abs() <= tol)[others].all())
    assert not grads[1].isfinite().any() and not grads[2].isfinite().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_ignored_rows_get_nothing_from_an_upstream_gradient_that_is_not_finite(dtype, bad):
    x, w, t, _ = inputs(300, 64, 500, dtype)
    t[::3] = -100
    for reduction in ("mean", "sum"):
        _, (dx, dw) = run(x, w, t, None, torch.tensor(bad, device=DEV), reduction=reduction)
        live = t != -100
        assert not dx[~live].any() and not dx[live].isfinite().any(1).any() and not dw.isfinite().any(1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("n", [5, 150])
def test_targets_closed_by_a_bias_of_minus_infinity(dtype, reduction, n):
    # an infinite loss; its gradient is the softmax of the open classes, minus one at the target
    x, w, t, b = inputs(n, 64, 300, dtype, bias=torch.float32)
    t = t % 100
    t[::4] = 200
    b[100:] = -float("inf")
    losses = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    closed = torch.arange(n, device=DEV) % 4 == 0
    assert bool((losses[closed] == float("inf")).all())
    leaves = [v.double().requires_grad_() for v in (x, w, b)]
    probabilities = torch.softmax(leaves[0].detach() @ leaves[1].detach().T + leaves[2].detach(), 1)
    g = probabilities - torch.nn.functional.one_hot(t, 300)
    want = dict(head(x, w, t % 100, torch.where(b.isinf(), 0.0, b), reduction="sum"))
    want["dx"], want["dw"], want["db"] = g @ w.double(), g.T @ x.double(), g.sum(0)
    want["dx_size"], want["dw_size"], want["db_size"] = g.abs() @ w.double().abs(), g.abs().T @ x.double().abs(), g.abs().sum(0)
    loss, grads = run(x, w, t, b, torch.ones(n, device=DEV) if reduction == "none" else None, reduction=reduction)
    assert torch.equal(loss.isinf(), closed) if reduction == "none" else bool(loss.isinf())
    check_grads(grads, want, x, w, 64, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("n,rows", [(300, 500), (300, 33000), (40000, 16100)])
def test_padding_gets_zeros_whatever_the_rest_holds(dtype, reduction, n, rows):
    # (the last in more than one group of tokens, whose sums are joined)
    x, w, t, b = inputs(n, 16, rows, dtype, classes=rows - 100, bias=torch.float32)
    x[17, 3] = float("nan")
    w[rows - 50] = float("nan")
    up = torch.full((n,) if reduction == "none" else (), float("inf"), device=DEV)
    _, (dx, dw, db) = run(x, w, t, b, up, reduction=reduction, num_classes=rows - 100)
    assert not dw[rows - 100:].any() and not db[rows - 100:].any() and not dw[:rows - 100].isfinite().any(1).any()
    x[17, 3] = 0.0
    _, (dx, dw, db) = run(x, w, t, b, torch.ones_like(up), reduction=reduction, num_classes=rows - 100)
    assert bool(dx.isfinite().all() and dw.isfinite().all()) and not dw[rows - 100:].any() and not db[rows - 100:].any()


def test_shapes_strides_and_types():
    x, w, t, _ = inputs(120, 64, 90)
    want, grads = run(x, w, t)
    wide_x, wide_w = torch.zeros(120, 100, device=DEV, dtype=torch.bfloat16), torch.zeros(90, 80, device=DEV, dtype=torch.bfloat16)
    wide_x[:, 8:72], wide_w[:, :64] = x, w
    odd = torch.zeros(120, 65, device=DEV, dtype=torch.bfloat16)
    odd[:, 1:] = x
    for xs in (x.view(4, 30, 64), wide_x[:, 8:72], odd[:, 1:], x.T.contiguous().T):
        for ws in (w, wide_w[:, :64], w.T.contiguous().T):
            for ts in (t, t.int(), torch.stack((t, t), 1)[:, 0]):
                xs, ws = xs.detach().requires_grad_(), ws.detach().requires_grad_()
                loss = ops.linear_cross_entropy(xs, ws, ts.view(xs.shape[:-1]))
                dx, dw = torch.autograd.grad(loss, (xs, ws))
                assert torch.equal(loss, want) and torch.equal(dx.reshape(120, 64), grads[0]) and torch.equal(dw, grads[1])
    # one row for all tokens
    row = x[:1].detach().requires_grad_()
    loss = ops.linear_cross_entropy(row.expand(120, 64), w, t)
    dx, = torch.autograd.grad(loss, row)
    ref = head(x[:1].expand(120, 64), w, t)
    tol = (ref["dx_size"] * (half_step(torch.bfloat16) * 1.1 + exp_error(ref, 64, 90)) + 2 * rounding(ref["dx"], torch.bfloat16)).sum(0) + 4 * rounding(ref["dx"].sum(0), torch.bfloat16)
    assert bool(((dx[0].double() - ref["dx"].sum(0)).abs() <= tol).all())
    # a single token without a batch
    one = ops.linear_cross_entropy(x[0], w, t[0], reduction="none")
    assert one.shape == () and abs(float(one) - float(head(x[:1], w, t[:1])["losses"])) < 1e-4


def test_gradients_that_are_not_asked_for():
    x, w, t, b = inputs(200, 64, 300, bias=torch.float32)
    _, (dx, dw, db) = run(x, w, t, b)
    for which in range(1, 8):
        leaves = [v.detach().clone().requires_grad_(bool(which >> i & 1)) for i, v in enumerate((x, w, b))]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        wanted = [v for v in leaves if v.requires_grad]
        for got, expect in zip(torch.autograd.grad(loss, wanted), [g for g, v in zip((dx, dw, db), leaves) if v.requires_grad]):
            assert torch.equal(got, expect)


def test_the_upstream_gradient_and_a_second_pass():
    x, w, t, _ = inputs(300, 64, 500)
    leaves = [v.clone().requires_grad_() for v in (x, w)]
    loss = ops.linear_cross_entropy(*leaves, t)
    first = torch.autograd.grad(loss, leaves, torch.tensor(3.0, device=DEV), retain_graph=True)
    kept = [g.clone() for g in first]
    second = torch.autograd.grad(loss, leaves, torch.tensor(-7.0, device=DEV), retain_graph=True)
    third = torch.autograd.grad(loss, leaves, torch.tensor(1.0, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(first, kept))
    for grads, up in ((first, 3.0), (second, -7.0), (third, 1.0)):
        want = head(x, w, t, upstream=up)
        # (what was formed for one is rounded once more when it is multiplied)
        want["dx_size"], want["dw_size"] = want["dx_size"] + want["dx"].abs(), want["dw_size"] + want["dw"].abs()
        check_grads(grads, want, x, w, 64, torch.bfloat16)


def test_losses_changed_in_place():
    x, w, t, _ = inputs(100, 64, 200)
    up = torch.rand(100, device=DEV)
    leaves = [v.clone().requires_grad_() for v in (x, w)]
    losses = ops.linear_cross_entropy(*leaves, t, reduction="none")
    losses *= 2.0
    got = torch.autograd.grad(losses, leaves, up)
    for a, b in zip(got, run(x, w, t, None, 2.0 * up, reduction="none")[1]):
        assert torch.equal(a, b)


def test_captured_passes_replayed_on_other_inputs():
    x, w, t, _ = inputs(400, 128, 700)
    leaves = [v.clone().requires_grad_() for v in (x, w)]
    up = torch.tensor(2.0, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.linear_cross_entropy(*leaves, t), leaves, up)
    torch.cuda.current_stream().wait_stream(side)
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward):
        loss = ops.linear_cross_entropy(*leaves, t)
    with torch.cuda.graph(backward):
        grads = torch.autograd.grad(loss, leaves, up)
    for seed in (1, 2):
        nx, nw, nt, _ = inputs(400, 128, 700, seed=seed)
        with torch.no_grad():
            leaves[0].copy_(nx), leaves[1].copy_(nw), t.copy_(nt)
        forward.replay()
        backward.replay()
        backward.replay()
        want = head(nx, nw, nt, upstream=2.0)
        assert abs(float(loss) - float(want["loss"])) <= 1e-5 * float(want["loss"])
        want["dx_size"], want["dw_size"] = want["dx_size"] + want["dx"].abs(), want["dw_size"] + want["dw"].abs()
        check_grads(grads, want, nx, nw, 128, torch.bfloat16)


def test_differences():
    # the gradient along a direction against a central difference of the loss, which is smooth: third derivatives are below 1 here
    x, w, t, _ = inputs(64, 64, 90)
    loss, (dx, dw) = run(x, w, t, reduction="sum")
    g = torch.Generator(device=DEV).manual_seed(3)
    for leaf, grad, which in ((x, dx, 0), (w, dw, 1)):
        # steps that the 16-bit values hold: powers of two of their own last place are too small, so the difference is taken between two rounded points
        step = torch.randn(leaf.shape, device=DEV, generator=g) * 0.05
        high, low = (leaf.float() + step).to(leaf.dtype), (leaf.float() - step).to(leaf.dtype)
        ends = [ops.linear_cross_entropy(*((v, w) if which == 0 else (x, v)), t, reduction="none").double().sum() for v in (high, low)]
        middle = (high.double() + low.double()) / 2 - leaf.double()
        slope = ((high.double() - low.double()) * grad.double()).sum()
        scale = float(((high.double() - low.double()).abs() * grad.double().abs()).sum())
        # the third-order term of a step of 0.05 sqrt(64) in each logit, the middle's shift, the gradient's own rounding
        assert abs(float(ends[0] - ends[1] - slope)) <= 0.02 * scale + float((middle.abs() * grad.double().abs()).sum())


def test_autocast_casts():
    x, w, t, b = inputs(100, 64, 200, bias=torch.float32)
    x32, w32 = x.float().requires_grad_(), w.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = ops.linear_cross_entropy(x32, w32, t, bias=b)
    dx, dw = torch.autograd.grad(loss, (x32, w32))
    want, grads = run(x, w, t, b)
    assert torch.equal(loss, want) and dx.dtype == torch.float32 and torch.equal(dx.to(x.dtype), grads[0]) and torch.equal(dw.to(w.dtype), grads[1])


def test_other_streams():
    x, w, t, _ = inputs(1000, 256, 3000)
    want, grads = run(x, w, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loss, got = run(x, w, t)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(loss, want) and all(torch.equal(a, b) for a, b in zip(grads, got))
