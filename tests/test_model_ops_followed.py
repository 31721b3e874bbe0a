"""What follows PyTorch's operations from outside (forward-mode derivatives, tracers, tensors that wrap others): CPU tensors take operations that it sees, the
kernels refuse instead of losing it."""
import pytest
import torch
import torch.autograd.forward_ad as forward
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from nangila import ops
from nangila.models import Llama, LlamaConfig


def inputs(device):
    x, r, w = torch.randn(4, 128, device=device), torch.randn(4, 128, device=device), torch.randn(128, device=device)
    q, k = torch.randn(1, 6, 2, 8, device=device), torch.randn(1, 6, 1, 8, device=device)
    return x, r, w, q, k, ops.rotary_table(6, 8, device=device)


def calls(x, r, w, q, k, table):
    """(function, its tensors) of every operator whose result depends on all of them."""
    return [(lambda a, b: ops.rms_norm(a, b), (x, w)), (lambda a, b, c: ops.add_rms_norm(a, b, c), (x, r, w)), (lambda a, b, c: ops.rms_norm_fp8(a, c, residual=b), (x, r, w)),
            (lambda a, b: ops.rotary(a, b, table), (q, k)), (lambda a, t: ops.rotary(a, None, t), (q, table)), (lambda a: ops.orthogonalize(a), (x,)),
            (lambda a, b: ops.orthogonalize([a, b]), (x, r)),
            (lambda a, b, c: ops.muon_step([a], [b], [c], lr=0.1), (x, r, torch.zeros_like(x)))]


def test_tangents_on_the_cpu():
    x, r, w, q, k, table = inputs("cpu")
    tx, tr, tw, tq = (torch.randn_like(v) for v in (x, r, w, q))
    with forward.dual_level():
        y, h = ops.add_rms_norm(forward.make_dual(x, tx), forward.make_dual(r, tr), forward.make_dual(w, tw))
        turned = ops.rotary(forward.make_dual(q, tq), None, table)
        ty, th, tt = (forward.unpack_dual(v).tangent for v in (y, h, turned))
    hd, td = (x + r).double(), (tx + tr).double()
    rstd = (hd.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    want = (td * rstd - hd * rstd ** 3 * (hd * td).mean(-1, keepdim=True)) * w + hd * rstd * tw
    size = (td.abs() * rstd + hd.abs() * rstd ** 3 * (hd * td).abs().mean(-1, keepdim=True)) * w.abs() + (hd * rstd * tw).abs()
    assert torch.equal(th, tx + tr)
    assert ((ty.double() - want).abs() <= size * 2.0 ** -16).all()  # fp32: sums of 128 terms and a dozen roundings, below 2^-16 of the terms' sizes
    assert torch.equal(tt, ops.rotary(tq, None, table))


@pytest.mark.gpu
def test_tangents_are_refused_by_the_kernels():
    for call, args in calls(*inputs("cuda")):
        for i in range(len(args)):
            keep = [a.clone() for a in args]
            with forward.dual_level():
                dual = [forward.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
                with pytest.raises(NotImplementedError, match="nangila.*tangent"):
                    call(*dual)
            for a, b in zip(args, keep):
                assert torch.equal(a, b)
        call(*args)  # and none of it stays behind


@pytest.mark.gpu
def test_a_gradient_with_a_tangent_is_refused():
    x, r, w, q, k, table = inputs("cuda")
    for out, leaf in ((ops.rms_norm(x.requires_grad_(), w), x), (ops.rotary(q.requires_grad_(), None, table), q)):
        with forward.dual_level():
            up = forward.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="nangila.*tangent"):
                torch.autograd.grad(out, leaf, up, retain_graph=True)
        torch.autograd.grad(out, leaf, torch.ones_like(out))


@pytest.mark.gpu
def test_the_decoder_does_not_lose_a_tangent():
    cfg = LlamaConfig.tiny()
    cfg.fused = True
    m = Llama(cfg).cuda()
    idx = torch.randint(0, 1024, (1, 8), device="cuda")
    names = [n for n, _ in m.named_parameters()]
    with forward.dual_level():
        duals = {n: forward.make_dual(p.detach(), torch.ones_like(p)) for n, p in m.named_parameters() if n == names[0]}
        with pytest.raises(NotImplementedError, match="nangila.*tangent"):
            torch.func.functional_call(m, duals, (idx,))


@pytest.mark.gpu
def test_tracers_are_refused_by_the_kernels():
    for call, args in calls(*inputs("cuda")):
        with pytest.raises(NotImplementedError, match="nangila.*traced"):
            torch.jit.trace(call, args, check_trace=False)
        with pytest.raises(NotImplementedError, match="nangila.*traced"):
            make_fx(call)(*args)
        mode = FakeTensorMode(allow_non_fake_inputs=True)
        with mode, pytest.raises(NotImplementedError, match="nangila.*traced"):
            call(*args)
        with pytest.raises((TypeError, NotImplementedError), match="nangila"):
            with mode:
                call(*(mode.from_tensor(a) for a in args))
        call(*args)


@pytest.mark.gpu
def test_transforms_are_refused_by_the_kernels():
    x, r, w, q, k, table = inputs("cuda")
    for f in (lambda v: ops.rms_norm(v, w).sum(), lambda v: ops.add_rms_norm(v, r[0], w)[0].sum()):
        for transform in (lambda g: torch.vmap(g)(x), lambda g: torch.func.grad(g)(x[0]), lambda g: torch.func.jvp(g, (x[0],), (x[0],))):
            with pytest.raises((RuntimeError, TypeError)):
                transform(f)


@pytest.mark.gpu
def test_modes_that_only_look_on_change_nothing():
    from torch.utils.flop_counter import FlopCounterMode

    x, r, w, q, k, table = inputs("cuda")
    want = ops.rms_norm(x, w)
    with FlopCounterMode(display=False):
        assert torch.equal(ops.rms_norm(x, w), want)
    with torch.inference_mode():
        assert torch.equal(ops.rms_norm(x, w), want)
