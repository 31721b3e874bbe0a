"""The vocabulary's operators with what follows PyTorch's operations from outside, and with tensors whose values are not in memory: refused or the same."""
import pytest
import torch
import torch.autograd.forward_ad as forward
from torch.fx.experimental.proxy_tensor import make_fx

from nangila import ops

neg, zeros = torch._neg_view, torch._efficientzerotensor


def calls(device):
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    x, r, w, b = (torch.randn(*s, device=device).to(dtype) for s in ((6, 64), (6, 64), (50, 64), (50,)))
    ids = torch.tensor([1, 4, 4, 0, 2, 7], device=device)
    return [(lambda a, c: ops.dropout(a, 0.5, seed=1, residual=c), (x, r)), (lambda a: ops.embedding(ids, a), (w,)),
            (lambda a, c, e: ops.linear_cross_entropy(a, c, ids, bias=e), (x, w, b)), (lambda a, c: ops.linear_cross_entropy(a, c, ids, reduction="none"), (x, w))]


def test_tangents_on_the_cpu():
    for call, args in calls("cpu"):
        tangents = [torch.randn_like(a) for a in args]
        with forward.dual_level():
            out = forward.unpack_dual(call(*(forward.make_dual(a, t) for a, t in zip(args, tangents)))).tangent
        leaves = [a.clone().requires_grad_() for a in args]
        y = call(*leaves)
        up = torch.randn_like(y)
        back = torch.autograd.grad(y, leaves, up)
        # the same bilinear form from both sides, in float32
        left, right = (out * up).sum(), sum((g * t).sum() for g, t in zip(back, tangents))
        assert torch.allclose(left, right, rtol=1e-4, atol=1e-4)


def test_masks_are_not_traced():
    x = torch.randn(4, 8)
    with pytest.raises(NotImplementedError, match="nangila.*traced"):
        torch.jit.trace(lambda a: ops.dropout(a, 0.5), (x,), check_trace=False)


@pytest.mark.gpu
def test_tangents_and_tracers_are_refused_by_the_kernels():
    for call, args in calls("cuda"):
        for i in range(len(args)):
            with forward.dual_level():
                dual = [forward.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
                with pytest.raises(NotImplementedError, match="nangila.*tangent"):
                    call(*dual)
        with pytest.raises(NotImplementedError, match="nangila.*traced"):
            torch.jit.trace(call, args, check_trace=False)
        with pytest.raises(NotImplementedError, match="nangila.*traced"):
            make_fx(call)(*args)
        y = call(*(a.clone().requires_grad_() for a in args))
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(y.float().sum(), y.grad_fn.next_functions[0][0].variable, create_graph=True)
        call(*args)


@pytest.mark.gpu
def test_transforms_are_refused_by_the_kernels():
    for call, args in calls("cuda"):
        for transform in (lambda g: torch.vmap(g)(torch.stack((args[0], args[0]))), lambda g: torch.func.grad(lambda v: g(v).float().sum())(args[0])):
            with pytest.raises((RuntimeError, TypeError)):
                transform(lambda v: call(v, *args[1:]))


@pytest.mark.gpu
def test_values_that_are_not_in_memory():
    for call, args in calls("cuda"):
        assert torch.equal(call(*(neg(a) for a in args)), call(*(-a for a in args)))
        leaves = [a.clone().requires_grad_() for a in args]
        up = torch.randn_like(call(*args))
        back, want, none = (torch.autograd.grad(call(*leaves), leaves, g) for g in (neg(up), -up, zeros(list(up.shape), dtype=up.dtype, device="cuda")))
        for a, b, c in zip(back, want, none):
            assert torch.equal(a, b) and not torch.as_tensor(c).any()
    w, ids = torch.randn(50, 64, device="cuda"), torch.tensor([1, 2, 0], device="cuda")
    assert torch.equal(ops.embedding(neg(-ids), w), ops.embedding(ids, w))


@pytest.mark.gpu
def test_devices_have_to_agree():
    x, w, t = torch.randn(4, 64, device="cuda").to(torch.bfloat16), torch.randn(9, 64).to(torch.bfloat16), torch.zeros(4, dtype=torch.long)
    for bad in (lambda: ops.linear_cross_entropy(x, w, t.cuda()), lambda: ops.linear_cross_entropy(x, w.cuda(), t), lambda: ops.embedding(t, w.cuda()), lambda: ops.dropout(x, seed=t[:1]),
                lambda: ops.dropout(x, residual=x.cpu()), lambda: ops.linear_cross_entropy(x, w.cuda(), t.cuda(), bias=torch.zeros(9))):
        with pytest.raises(ValueError, match="nangila.* on "):
            bad()
    with pytest.raises(TypeError, match="not float32"):
        ops.linear_cross_entropy(x.float(), w.float().cuda(), t.cuda())


@pytest.mark.gpu
def test_inference_mode():
    with torch.inference_mode():
        for call, args in calls("cuda"):
            call(*args)
