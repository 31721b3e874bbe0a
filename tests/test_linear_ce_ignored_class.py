"""The head's loss where the target that is ignored is itself a class (a padding token's number): such rows add nothing, whatever they hold."""
import pytest
import torch

from nangila import ops
from tests._head_bounds import check_grads_anywhere
from tests._vocab_ops import head
from tests.test_linear_ce_kernel_gpu import DEV, check_losses, inputs, run

HELD = ["nan", "inf", "far"]


def spoil(x, w, rows, held):
    """What the ignored rows hold: values that are not finite, or finite ones whose logits pass 100."""
    if held == "far":
        along = w[1].float()
        x[rows] = (200 * along / along.square().sum()).to(x.dtype)
    else:
        x[rows] = float(held)


def upstream_of(reduction, n, dtype):
    if reduction == "none":
        return torch.rand(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)) + 0.5
    return torch.tensor(512.0 if dtype == torch.float16 else 1.0, device=DEV)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("held", HELD)
def test_on_the_cpu(held, last, reduction):
    g = torch.Generator().manual_seed(2)
    x, w, b = torch.randn(12, 8, generator=g), torch.randn(11, 8, generator=g), torch.randn(11, generator=g)
    ignore, t = 9 if last else 0, torch.randint(1, 9, (12,), generator=g)
    t[::3] = ignore
    results = []
    for dirty in (False, True):
        if dirty:
            spoil(x, w, slice(None, None, 3), held)
        leaves = [v.clone().requires_grad_() for v in (x, w, b)]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], num_classes=10, ignore_index=ignore, reduction=reduction)
        results.append((loss, *torch.autograd.grad(loss, leaves, torch.ones_like(loss))))
    assert all(torch.equal(clean, dirty) and bool(dirty.isfinite().all()) for clean, dirty in zip(*results))
    want = head(torch.where((t == ignore)[:, None], 0.0, x), w, t, b, 10, ignore, reduction, torch.ones(12) if reduction == "none" else None)
    for got, name in zip(results[1][1:], ("dx", "dw", "db")):
        assert torch.allclose(got.double(), want[name], atol=1e-5), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n", [3, 100, 300])
def test_they_add_nothing(n, bias, last, reduction, dtype):
    rows, classes, d = 700, 650, 64
    ignore = classes - 1 if last else 0
    x, w, t, b = inputs(n, d, rows, dtype, classes, torch.float32 if bias else None)
    t = t.clamp(1, classes - 2)
    t[::3] = ignore
    up = upstream_of(reduction, n, dtype)
    want = head(x, w, t, b, classes, ignore, reduction, up)
    options = dict(num_classes=classes, ignore_index=ignore, reduction=reduction)
    clean, grads = run(x, w, t, b, up, **options)
    if reduction == "none":
        check_losses(clean, want, d, rows)
    check_grads_anywhere(grads, want, x, w, d, dtype)
    assert not grads[0][::3].any()
    for held in HELD:
        spoil(x, w, slice(None, None, 3), held)
        loss, dirty = run(x, w, t, b, up, **options)
        assert torch.equal(loss, clean), held
        assert all(torch.equal(a, c) and bool(c.isfinite().all()) for a, c in zip(grads, dirty)), held


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,reduction", [(torch.bfloat16, "mean"), (torch.bfloat16, "none"), (torch.float16, "sum")])
def test_in_several_groups_of_tokens(dtype, reduction):
    # (1536 rows of E fill a gigabyte; every seventh token is ignored)
    n, d, rows = 3200, 64, 300001
    x, w, t, b = inputs(n, d, rows, dtype, bias=torch.float32)
    t = t.clamp(1, rows - 2)
    t[::7] = 0
    up = upstream_of(reduction, n, dtype)
    clean, grads = run(x, w, t, b, up, ignore_index=0, reduction=reduction)
    for held in HELD:
        spoil(x, w, slice(None, None, 7), held)
        loss, dirty = run(x, w, t, b, up, ignore_index=0, reduction=reduction)
        assert torch.equal(loss, clean) and all(torch.equal(a, c) and bool(c.isfinite().all()) for a, c in zip(grads, dirty)), held
        assert not dirty[0][::7].any()
