"""The loss that comes with its gradients: means and sums with a bias, padded classes, ignored tokens and tokens without a class, against the formula in 64 bits."""
import pytest
import torch

from nangila import ops
from tests._vocab_ops import head
from tests.test_linear_ce_kernel_gpu import DEV, SIZES, U, exp_error, inputs

pytestmark = pytest.mark.gpu


def allowed(want, live, d, rows, mean, count):
    """Each token's loss is off by the relative error of its row's sum and by the logarithm's few steps; what they add up to in 64 bits is rounded once."""
    each = exp_error(want, d, rows) + 8 * U * (want["losses"].nan_to_num(0.0).abs() + want["z_most"])
    return float(each[live].sum()) / (count if mean else 1) + 2 * U * abs(float(want["loss"]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [None, torch.float32, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("n,d,rows", SIZES + [(2600, 64, 12000)])
def test_means_and_sums(dtype, bias, reduction, n, d, rows):
    classes = max(1, rows - 3)
    x, w, t, b = inputs(n, d, rows, dtype, classes, bias, ignored=0.2 if n > 2 else 0.0)
    if n > 100:  # some far above their reference, which a first pass cannot serve
        away = w[(t.clamp(min=0) + 1) % classes].float()
        x[3::40] = (150 * away / away.square().sum(-1, keepdim=True).clamp(min=0.1))[3::40].to(dtype)
    if not bool((t != -100).any()):
        t[0] = 0
    want = head(x, w, t, b, classes, reduction=reduction)
    leaves = [v.detach().clone().requires_grad_() for v in (x, w)] + ([] if b is None else [b.clone().requires_grad_()])
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2] if b is not None else None, num_classes=classes, reduction=reduction)
    live = t != -100
    tol = allowed(want, live, d, rows, reduction == "mean", int(live.sum()))
    assert loss.requires_grad and loss.dtype == torch.float32 and loss.shape == ()
    assert abs(float(loss.detach()) - float(want["loss"])) <= tol
    with torch.no_grad():  # by itself it is as near
        alone = ops.linear_cross_entropy(x, w, t, bias=b, num_classes=classes, reduction=reduction)
    assert abs(float(alone) - float(want["loss"])) <= tol


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_a_target_that_is_no_class_is_told(reduction):
    x, w, t, b = inputs(300, 64, 500, classes=490, bias=torch.float32)
    t[7] = 490
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], num_classes=490, reduction=reduction)
    assert bool(loss.detach().isnan()) and all(bool(g.isfinite().all()) for g in torch.autograd.grad(loss, leaves))


def test_in_several_groups_of_tokens():
    x, w, t, b = inputs(3200, 64, 300001, bias=torch.float32, ignored=0.1)
    for reduction in ("mean", "sum"):
        want = head(x, w, t, b, reduction=reduction)
        leaves = [v.clone().requires_grad_() for v in (x, w, b)]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], reduction=reduction).detach()
        live = t != -100
        assert abs(float(loss) - float(want["loss"])) <= allowed(want, live, 64, 300001, reduction == "mean", int(live.sum()))
        assert loss.device.type == torch.device(DEV).type
