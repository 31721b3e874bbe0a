"""The model and update operators on CPU tensors: their formulas in torch operations, and what they refuse."""
import os
import subprocess
import sys

import pytest
import torch

import _model_ops as plain
from nangila import ops
from nangila.models import Llama, LlamaConfig
from nangila.ops.muon import update_scale
from nangila.optim import Muon

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COEF = (3.4445, -4.7750, 2.0315)


# ---- RMS norm -------------------------------------------------------------------------------------------------------

def test_norm_is_the_formula_and_has_its_gradients():
    # fp32 sums of 24 terms: below 2^-18 of the terms
    x, r = torch.randn(5, 24, requires_grad=True), torch.randn(5, 24, requires_grad=True)
    w = torch.randn(24, requires_grad=True)
    y, h = ops.add_rms_norm(x, r, w, eps=1e-5)
    assert torch.equal(h, x + r)
    want = plain.norm(h.detach(), w.detach(), 1e-5)
    assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -18).all()
    dy, dh = torch.randn(5, 24), torch.randn(5, 24)
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (dy, dh))
    wx, ww, sx, sw = plain.norm_grads(h.detach(), w.detach(), 1e-5, dy, dh)
    assert torch.equal(dx, dr)
    assert ((dx.double() - wx).abs() <= sx * 2.0 ** -17).all() and ((dw.double() - ww).abs() <= sw * 2.0 ** -17).all()
    assert torch.equal(ops.rms_norm(h, w, eps=1e-5), y)


@pytest.mark.parametrize("group", [None, 128])
def test_eight_bits_is_the_formula(group):
    x, w = torch.randn(6, 256).bfloat16(), torch.randn(256).bfloat16()
    x[1] = 0
    x[2, 200] = float("nan")
    q, scale = ops.rms_norm_fp8(x, w, group=group)
    assert q.shape == x.shape and scale.shape == (6, 2 if group else 1)
    keep = [0, 1, 3, 4, 5]
    f = plain.norm(x[keep], w, 1e-5).view(5, -1, group or 256)
    s = scale[keep].double().view(5, -1)
    got = q[keep].double().view(f.shape) * s.unsqueeze(-1)
    assert ((got - f).abs() <= f.abs() * (2.0 ** -4 + 2.0 ** -15) + s.unsqueeze(-1) * 2.0 ** -10 * 1.01).all()
    assert torch.isnan(scale[2]).all() and torch.isnan(q[2].float()).all()
    out = ops.rms_norm_fp8(x, w, residual=x, group=group)
    assert len(out) == 3 and torch.equal(out[2][keep], (x + x)[keep])


def test_norm_refusals():
    x, w = torch.randn(4, 16), torch.ones(16)
    bad = [
        (TypeError, lambda: ops.rms_norm(x.double(), w)),
        (TypeError, lambda: ops.rms_norm(x, w.long())),
        (TypeError, lambda: ops.rms_norm(x.to_sparse(), w)),
        (TypeError, lambda: ops.add_rms_norm(x, x.bfloat16(), w)),
        (ValueError, lambda: ops.rms_norm(x, torch.ones(15))),
        (ValueError, lambda: ops.rms_norm(x, torch.ones(1, 16))),
        (ValueError, lambda: ops.rms_norm(torch.tensor(1.0), torch.ones(1))),
        (ValueError, lambda: ops.rms_norm(torch.ones(2, 0), torch.ones(0))),
        (ValueError, lambda: ops.rms_norm(torch.ones(1, 32769), torch.ones(32769))),
        (ValueError, lambda: ops.add_rms_norm(x, x[:1], w)),
        (ValueError, lambda: ops.rms_norm(x, w, eps=-1.0)),
        (ValueError, lambda: ops.rms_norm(x, w, eps=float("nan"))),
        (ValueError, lambda: ops.rms_norm_fp8(x, w, group=64)),
        (ValueError, lambda: ops.rms_norm_fp8(x, w, group=128)),
        (RuntimeError, lambda: ops.rms_norm_fp8(x.clone().requires_grad_(), w)),
    ]
    for kind, call in bad:
        with pytest.raises(kind, match="nangila"):
            call()
    with torch.no_grad():
        ops.rms_norm_fp8(x.clone().requires_grad_(), w)


# ---- rotary positions -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("d,rot", [(16, 16), (20, 8), (6, 2)])
def test_rotary_is_the_formula_and_has_its_gradient(d, rot, layout):
    table = ops.rotary_table(30, rot)
    q, k = torch.randn(2, 7, 3, d, requires_grad=True), torch.randn(2, 7, 1, d)
    pos = torch.randint(0, 30, (2, 7))
    for given, at in ((None, torch.arange(7)[None]), (pos, pos), (pos[0].int(), pos[:1])):
        oq, ok = ops.rotary(q, k, table, positions=given, layout=layout)
        for got, x in ((oq, q.detach()), (ok, k)):
            want, size = plain.turned(x, table, at, layout)
            assert ((got.double() - want).abs() <= size * 2.0 ** -21).all()
        up = torch.randn(q.shape)
        g, = torch.autograd.grad(oq, q, up)
        want, size = plain.turned(up, table, at, layout, inverse=True)
        assert ((g.double() - want).abs() <= size * 2.0 ** -21).all()


def test_the_interleaved_layout_is_the_models_rotation():
    from nangila.models.llama import apply_rope, rope_table

    x = torch.randn(2, 9, 3, 16)
    # the model's table forms its angles in fp32: at positions below 9 they are off by 9 * 2^-23 at most
    assert torch.allclose(ops.rotary(x, None, ops.rotary_table(9, 16)), apply_rope(x, rope_table(9, 16, 10000.0, x.device)), rtol=0, atol=4.0 * 9 * 2.0 ** -23 * x.abs().max())


def test_positions_outside_the_table():
    q = torch.randn(1, 3, 1, 8)
    out = ops.rotary(q, None, ops.rotary_table(4, 4), positions=torch.tensor([-1, 3, 4]))
    assert torch.isnan(out[0, [0, 2], :, :4]).all() and torch.equal(out[..., 4:], q[..., 4:]) and torch.isfinite(out[0, 1]).all()


def test_tables():
    full = ops.rotary_table(50, 8, theta=500.0).double()
    inv = 500.0 ** (-torch.arange(0, 8, 2).double() / 8)
    angle = torch.arange(50).double()[:, None] * inv
    assert torch.allclose(full, torch.stack((angle.cos(), angle.sin()), -1), rtol=0, atol=2.0 ** -24)
    linear = ops.rotary_table(50, 8, theta=500.0, scaling="linear", factor=4.0).double()
    assert torch.allclose(linear, torch.stack(((angle / 4).cos(), (angle / 4).sin()), -1), rtol=0, atol=2.0 ** -24)
    # ntk: the fastest pair as before, the slowest slowed by the factor
    ntk = ops.rotary_table(50, 8, theta=500.0, scaling="ntk", factor=4.0).double()
    assert torch.allclose(ntk[:, 0], full[:, 0], rtol=0, atol=2.0 ** -23)
    assert torch.allclose(ntk[:, 3], linear[:, 3], rtol=0, atol=2.0 ** -22)
    # yarn: fast pairs as before, slow ones slowed, all larger by the attention factor
    yarn = ops.rotary_table(50, 64, scaling="yarn", factor=8.0, original_seq=4096).double() / (0.1 * torch.log(torch.tensor(8.0)).double() + 1)
    plain_table, slow = ops.rotary_table(50, 64).double(), ops.rotary_table(50, 64, scaling="linear", factor=8.0).double()
    assert torch.allclose(yarn[:, 0], plain_table[:, 0], rtol=0, atol=2.0 ** -22) and torch.allclose(yarn[:, -1], slow[:, -1], rtol=0, atol=2.0 ** -22)
    # far positions: an angle formed in fp32 would be off by 2^20 * 2^-24 there
    far = ops.rotary_table(1_000_001, 2)[-1, 0].double()
    exact = torch.tensor(1_000_000.0, dtype=torch.float64)
    assert torch.allclose(far, torch.stack((exact.cos(), exact.sin())), rtol=0, atol=2.0 ** -24)


def test_rotary_refusals():
    q, table = torch.randn(1, 4, 2, 8), ops.rotary_table(4, 8)
    bad = [
        (TypeError, lambda: ops.rotary(q.double(), None, table)),
        (TypeError, lambda: ops.rotary(q, q.bfloat16(), table)),
        (TypeError, lambda: ops.rotary(q, None, table, positions=torch.zeros(4))),
        (ValueError, lambda: ops.rotary(q[0], None, table)),
        (ValueError, lambda: ops.rotary(q, q[:, :3], table)),
        (ValueError, lambda: ops.rotary(q, q[..., :4], table)),
        (ValueError, lambda: ops.rotary(q, None, table.double())),
        (ValueError, lambda: ops.rotary(q, None, table[..., 0])),
        (ValueError, lambda: ops.rotary(q, None, ops.rotary_table(4, 10))),
        (ValueError, lambda: ops.rotary(q, None, ops.rotary_table(3, 8))),
        (ValueError, lambda: ops.rotary(q, None, table.clone().requires_grad_())),
        (ValueError, lambda: ops.rotary(q, None, table, positions=torch.zeros(3, dtype=torch.long))),
        (ValueError, lambda: ops.rotary(q, None, table, positions=torch.zeros(2, 4, dtype=torch.long))),
        (ValueError, lambda: ops.rotary(q, None, table, layout="pairs")),
        (ValueError, lambda: ops.rotary_table(0, 8)),
        (ValueError, lambda: ops.rotary_table(4, 7)),
        (ValueError, lambda: ops.rotary_table(4, 8, theta=-1.0)),
        (ValueError, lambda: ops.rotary_table(4, 8, factor=2.0)),
        (ValueError, lambda: ops.rotary_table(4, 8, scaling="linear", factor=0.5)),
        (ValueError, lambda: ops.rotary_table(4, 8, scaling="other", factor=2.0)),
        (ValueError, lambda: ops.rotary_table(4, 2, scaling="ntk", factor=2.0)),
        (ValueError, lambda: ops.rotary_table(4, 8, scaling="yarn", factor=2.0)),
        (ValueError, lambda: ops.rotary_table(4, 8, scaling="yarn", factor=2.0, original_seq=64, beta_fast=1.0)),
    ]
    for kind, call in bad:
        with pytest.raises(kind, match="nangila"):
            call()


# ---- orthogonalised updates --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,n", [(1, 1), (1, 6), (12, 20), (20, 12), (16, 16)])
def test_orthogonalize_is_the_formula(m, n):
    # bf16 result: 2^-8; fp32 products of 20 terms carried up by 485 at most: 485 * 20 * 2^-24
    u = torch.randn(m, n)
    want = plain.orthogonal(u, 5, COEF, 1e-7)
    got = ops.orthogonalize(u)
    assert got.dtype == torch.bfloat16 and torch.linalg.vector_norm(got.double() - want) <= (2.0 ** -8 + 485 * 20 * 2.0 ** -24) * torch.linalg.vector_norm(want)
    many = ops.orthogonalize([u, u.bfloat16(), u.t()])
    assert torch.equal(many[0], got) and many[2].shape == (n, m)
    assert torch.equal(ops.orthogonalize(u[None].expand(2, m, n))[1], got)
    assert (ops.orthogonalize(torch.zeros(m, n)) == 0).all()


def test_orthogonalize_refusals():
    u = torch.randn(4, 6)
    bad = [
        (TypeError, lambda: ops.orthogonalize(u.double())),
        (TypeError, lambda: ops.orthogonalize([u, 3])),
        (TypeError, lambda: ops.orthogonalize(u.to_sparse())),
        (ValueError, lambda: ops.orthogonalize(u[0])),
        (ValueError, lambda: ops.orthogonalize(u[:0])),
        (ValueError, lambda: ops.orthogonalize(torch.empty(0, 0, 3))),
        (ValueError, lambda: ops.orthogonalize(torch.empty(65537, 1))),
        (ValueError, lambda: ops.orthogonalize(u, steps=0)),
        (ValueError, lambda: ops.orthogonalize(u, steps=33)),
        (ValueError, lambda: ops.orthogonalize(u, coefficients=(1.0, 2.0))),
        (ValueError, lambda: ops.orthogonalize(u, steps=2, coefficients=[(1.0, 2.0, 3.0)])),
        (ValueError, lambda: ops.orthogonalize(u, coefficients=(float("nan"), 0.0, 0.0))),
        (ValueError, lambda: ops.orthogonalize(u, eps=0.0)),
    ]
    for kind, call in bad:
        with pytest.raises(kind, match="nangila"):
            call()


def test_muon_step_is_the_formula():
    p, g, m = torch.randn(12, 8), torch.randn(12, 8), torch.randn(12, 8)
    wm = 0.9 * m.double() + g.double()
    wp = p.double() * (1 - 0.1 * 0.01) - 0.1 * 0.2 * 12 ** 0.5 * plain.orthogonal(g.double() + 0.9 * wm, 5, COEF, 1e-7)
    ops.muon_step([p], [g], [m], lr=0.1, momentum=0.9, weight_decay=0.01)
    assert torch.allclose(m.double(), wm, rtol=0, atol=2.0 ** -20) and torch.allclose(p.double(), wp, rtol=0, atol=485 * 12 * 2.0 ** -24)
    assert update_scale(8, 2, "spectral") == 2.0 and update_scale(2, 8, "spectral") == 1.0 and update_scale(2, 8, None) == 1.0


def test_muon_step_refusals_change_nothing():
    p, g, m = torch.randn(4, 6), torch.randn(4, 6), torch.zeros(4, 6)
    both = torch.zeros(8, 6)
    bad = [
        (ValueError, lambda: ops.muon_step([p], [g], [], lr=0.1)),
        (ValueError, lambda: ops.muon_step([p, p], [g, g], [m, torch.zeros(4, 6)], lr=0.1)),
        (ValueError, lambda: ops.muon_step([p, torch.zeros(4, 6)], [g, g], [m, m], lr=0.1)),
        (ValueError, lambda: ops.muon_step([p], [m], [m], lr=0.1)),
        (ValueError, lambda: ops.muon_step([both[:4]], [g], [both[3:7]], lr=0.1)),
        (ValueError, lambda: ops.muon_step([p], [torch.randn(6, 4)], [m], lr=0.1)),
        (ValueError, lambda: ops.muon_step([torch.randn(6, 4).t()], [g], [m], lr=0.1)),
        (TypeError, lambda: ops.muon_step([p], [g], [m.bfloat16()], lr=0.1)),
        (TypeError, lambda: ops.muon_step([p.double()], [g], [m], lr=0.1)),
        (ValueError, lambda: ops.muon_step([p], [g], [m], lr=float("inf"))),
        (ValueError, lambda: ops.muon_step([p], [g], [m], lr=0.1, momentum=-0.5)),
        (ValueError, lambda: ops.muon_step([p], [g], [m], lr=0.1, scale="other")),
        (ValueError, lambda: ops.muon_step([p, torch.randn(5)], [g, torch.randn(5)], [m, torch.zeros(5)], lr=0.1)),
    ]
    keep = p.clone(), m.clone()
    for kind, call in bad:
        with pytest.raises(kind, match="nangila"):
            call()
    assert torch.equal(p, keep[0]) and torch.equal(m, keep[1])
    ops.muon_step([p, torch.zeros(4, 6)], [g, g], [m, torch.zeros(4, 6)], lr=0.1)  # one gradient for two is read twice


def test_muon_optimizer_keeps_its_momentum_in_float32():
    p = torch.nn.Parameter(torch.randn(6, 4).bfloat16())
    q = torch.nn.Parameter(torch.randn(3, 3))  # no gradient: left alone
    opt = Muon([p, q], lr=0.01)
    for _ in range(3):
        p.grad = torch.randn(6, 4).bfloat16()
        opt.step()
    state = opt.state_dict()
    other = Muon([torch.nn.Parameter(p.detach().clone()), torch.nn.Parameter(q.detach().clone())], lr=1.0)
    other.load_state_dict(state)
    mine, theirs = opt.state[p]["momentum_buffer"], other.state[other.param_groups[0]["params"][0]]["momentum_buffer"]
    assert mine.dtype == theirs.dtype == torch.float32 and torch.equal(mine, theirs) and mine.data_ptr() != theirs.data_ptr()
    assert other.param_groups[0]["lr"] == 0.01 and len(opt.state[q]) == 0
    p2 = other.param_groups[0]["params"][0]
    p.grad = torch.randn(6, 4).bfloat16()
    p2.grad = p.grad.clone()
    opt.step(), other.step()
    assert torch.equal(p, p2)
    assert opt.step(lambda: 3.0) == 3.0
    for kind, call in ((ValueError, lambda: Muon([torch.nn.Parameter(torch.randn(4))])), (ValueError, lambda: Muon([p], lr=-1.0)), (ValueError, lambda: Muon([p], steps=0)),
                       (ValueError, lambda: Muon([p], scale="x")), (ValueError, lambda: opt.add_param_group({"params": [torch.nn.Parameter(torch.randn(2, 2, 2))]}))):
        with pytest.raises(kind):
            call()
    assert len(opt.param_groups) == 1


def test_sharded_tensors_are_refused():
    import torch.distributed as dist
    from torch.distributed.device_mesh import DeviceMesh
    from torch.distributed.tensor import DTensor, Replicate

    own = not dist.is_initialized()
    if own:
        dist.init_process_group("gloo", rank=0, world_size=1, store=dist.HashStore())
    try:
        d = DTensor.from_local(torch.randn(4, 6), DeviceMesh("cpu", [0]), [Replicate()])
        table = ops.rotary_table(4, 4)
        for call in (lambda: ops.rms_norm(d, torch.ones(6)), lambda: ops.rotary(d.to_local().view(1, 4, 1, 6), None, DTensor.from_local(table, DeviceMesh("cpu", [0]), [Replicate()])),
                     lambda: ops.orthogonalize(d), lambda: ops.orthogonalize([d]), lambda: ops.muon_step([d], [torch.randn(4, 6)], [torch.zeros(4, 6)], lr=0.1),
                     lambda: Muon([torch.nn.Parameter(d)])):
            with pytest.raises(TypeError, match="nangila"):
                call()
    finally:
        if own:
            dist.destroy_process_group()


# ---- where they are used -------------------------------------------------------------------------------------------------

def test_the_decoder_gives_the_same_with_them():
    torch.manual_seed(0)
    a = Llama(LlamaConfig.tiny())
    cfg = LlamaConfig.tiny()
    cfg.fused = True
    b = Llama(cfg)
    b.load_state_dict(a.state_dict())
    idx = torch.randint(0, 1024, (2, 24))
    la, lb = a(idx, idx), b(idx, idx)
    la.backward(), lb.backward()
    # fp32 throughout, two blocks: a few hundred roundings of 2^-24 on terms near one
    assert abs(float(la) - float(lb)) < 1e-4
    for p, q in zip(a.parameters(), b.parameters()):
        assert float(torch.linalg.vector_norm(p.grad - q.grad)) <= 1e-3 * float(torch.linalg.vector_norm(p.grad)) + 1e-7


def test_the_decoders_position_options():
    cfg = LlamaConfig(n_layer=1, n_head=2, n_kv_head=1, d_model=32, d_mlp=48, vocab_size=64, max_seq=16, fused=True, rope_layout="half", rope_dim=8, rope_scaling="yarn",
                      rope_factor=4.0, rope_original_seq=16)
    m = Llama(cfg)
    idx = torch.randint(0, 64, (1, 20))
    m(idx, idx).backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())
    with pytest.raises(ValueError, match="fused"):
        LlamaConfig(rope_layout="half")


def test_ddp_example_with_muon(tmp_path):
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", MASTER_ADDR="127.0.0.1", MASTER_PORT="29593")
    ck = str(tmp_path / "run.pt")
    for steps in ("6", "8"):  # the second run resumes
        r = subprocess.run([sys.executable, "examples/train_ddp_gpt2.py", "--tiny", "--steps", steps, "--warmup-steps", "2", "--micro-batch", "2", "--optimizer", "muon",
                            "--checkpoint", ck, "--save-every", "6"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
