"""One training step of the decoder with its norms, rotary positions and orthogonal updates together, and the examples that use them."""
import os
import subprocess
import sys

import pytest
import torch

import _model_ops as plain
from nangila.models import Llama, LlamaConfig
from nangila.optim import Muon

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def models(**more):
    torch.manual_seed(0)
    a = Llama(LlamaConfig.tiny()).cuda()
    cfg = LlamaConfig.tiny()
    cfg.fused = True
    for k, v in more.items():
        setattr(cfg, k, v)
    b = Llama(cfg).cuda()
    b.load_state_dict(a.state_dict())
    return a, b


def test_forward_backward_and_update():
    # fp32: the kernels' norms and rotations differ from PyTorch's by a few 2^-24, which two blocks carry to the gradients
    a, b = models()
    idx = torch.randint(0, 1024, (2, 96), device="cuda")
    la, lb = a(idx, idx), b(idx, idx)
    la.backward(), lb.backward()
    assert abs(la.item() - lb.item()) < 1e-4
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.linalg.vector_norm(p.grad - q.grad) <= 1e-3 * torch.linalg.vector_norm(p.grad) + 1e-7
    matrices = [p for p in b.blocks.parameters() if p.dim() == 2]
    opt = Muon(matrices, lr=0.01, weight_decay=0.1)
    before = [p.detach().clone() for p in matrices]
    opt.step()
    for p, old in zip(matrices, before):
        g = p.grad.double()
        o = plain.orthogonal(g + 0.95 * g, 5, (3.4445, -4.7750, 2.0315), 1e-7)
        rate = 0.01 * 0.2 * max(p.shape) ** 0.5
        want = old.double() * (1 - 0.01 * 0.1) - rate * o
        # 7.5e-3 of the update: five steps of roundings to fp16 (see the kernel's own tests)
        assert torch.linalg.vector_norm(p.detach().double() - want) <= 7.5e-3 * rate * torch.linalg.vector_norm(o) + 2.0 ** -24 * torch.linalg.vector_norm(want)


@pytest.mark.parametrize("layout,rot", [("interleaved", None), ("half", 16)])
def test_steps_in_bf16(layout, rot):
    _, b = models(rope_layout=layout, rope_dim=rot)
    b = Llama(b.cfg).cuda().bfloat16()
    matrices = [p for p in b.blocks.parameters() if p.dim() == 2]
    held = {id(p) for p in matrices}
    opts = [Muon(matrices, lr=1e-3), torch.optim.AdamW([p for p in b.parameters() if id(p) not in held], lr=1e-3)]
    for _ in range(3):
        idx = torch.randint(0, 1024, (2, 97), device="cuda")
        b(idx[:, :-1], idx[:, 1:]).backward()
        for o in opts:
            o.step()
            o.zero_grad()
    assert all(torch.isfinite(p).all() for p in b.parameters())


def test_under_autocast_the_residual_stream_keeps_its_type():
    _, b = models()
    idx = torch.randint(0, 1024, (2, 32), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = b(idx, idx)
    loss.backward()
    assert torch.isfinite(loss) and all(torch.isfinite(p.grad).all() for p in b.parameters())


@pytest.mark.parametrize("args", [["examples/train_ddp_gpt2.py", "--tiny", "--steps", "6", "--warmup-steps", "2", "--micro-batch", "2", "--optimizer", "muon"],
                                  ["examples/train_fsdp_llama.py", "--tiny", "--steps", "3", "--micro-batch", "2", "--fused"],
                                  ["bench/train_bench.py", "--config", "llama-1.3b-fsdp", "--small", "--fused", "--steps", "2", "--warmup", "3"]])
def test_the_commands_that_use_them_run(args):
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29597")
    r = subprocess.run([sys.executable, *args], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
