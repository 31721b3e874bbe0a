"""The models with their vocabulary's operators and dropout: the same results as without where nothing is dropped, what goes into a step together, and what is refused."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch
import torch.nn.functional as F

from nangila import ops
from nangila.models import GPT2, BertMLM, Llama, LlamaConfig
from nangila.models.bert import BertConfig, mask_tokens
from nangila.models.gpt2 import GPT2Config
from tests._model_ops import half_step
from tests._vocab_ops import embedding_grad, head, kept, share

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def models(**options):
    gpt2, bert, llama = GPT2Config.tiny(), BertConfig.tiny(), LlamaConfig.tiny()
    for cfg in (gpt2, bert, llama):
        for k, v in options.items():
            if hasattr(cfg, k):
                setattr(cfg, k, v)
    return {"gpt2": lambda: GPT2(gpt2), "bert": lambda: BertMLM(bert), "llama": lambda: Llama(llama)}


def batch(name, device="cpu"):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(5, 1000, (3, 40), generator=g)
    if name == "bert":
        x, y = mask_tokens(ids, BertConfig.tiny(), generator=g)
        return x.to(device), y.to(device)
    return ids[:, :-1].to(device), ids[:, 1:].to(device)


def step(name, device="cpu", dtype=torch.float32, seed=0, **options):
    torch.manual_seed(seed)
    m = models(**options)[name]().to(device=device, dtype=dtype)
    loss = m(*batch(name, device))
    loss.backward()
    return m, loss.detach(), {n: p.grad for n, p in m.named_parameters()}


@pytest.mark.parametrize("name", ["gpt2", "bert", "llama"])
def test_the_same_without_logits_on_the_cpu(name):
    _, loss, grads = step(name)
    _, fused, got = step(name, fused_vocab=True)
    assert abs(float(loss) - float(fused)) <= 1e-5  # float32 sums in another order, of losses near 7
    for n, g in grads.items():
        assert torch.allclose(g, got[n], rtol=1e-3, atol=1e-6), n


@pytest.mark.parametrize("name", ["gpt2", "bert"])
def test_dropout_is_for_training(name):
    m, loss, _ = step(name, dropout=0.2)
    _, plain, _ = step(name)
    assert float(loss) != float(plain)
    m.eval()
    torch.manual_seed(0)
    still = models()[name]().eval()
    still.load_state_dict(m.state_dict())
    x, y = batch(name)
    assert torch.equal(m(x, y), still(x, y))
    # the masks follow PyTorch's generator
    a, b, c = (step(name, dropout=0.2)[1] for _ in range(3))
    assert torch.equal(a, b) and torch.equal(b, c)


def test_recomputed_activations_get_the_same_masks():
    torch.manual_seed(0)
    cfg = GPT2Config.tiny()
    cfg.dropout = 0.3
    m = GPT2(cfg)
    x = torch.randn(2, 10, cfg.d_model, requires_grad=True)
    grads = []
    for again in (False, True):
        torch.manual_seed(5)
        y = torch.utils.checkpoint.checkpoint(m.blocks[0], x, use_reentrant=False) if again else m.blocks[0](x)
        grads.append(torch.autograd.grad(y.square().sum(), x)[0])
    assert torch.equal(*grads)


def test_commands_refuse_options_without_effect():
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29598")
    r = subprocess.run([sys.executable, "bench/train_bench.py", "--config", "resnet50-powersgd", "--fused-vocab", "--small"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 2 and "--fused-vocab" in r.stderr


def test_the_example_takes_them():
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", MASTER_ADDR="127.0.0.1", MASTER_PORT="29597")
    r = subprocess.run([sys.executable, "examples/train_ddp_gpt2.py", "--tiny", "--steps", "6", "--warmup-steps", "2", "--micro-batch", "2", "--dropout", "0.1", "--fused-vocab"],
                       cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["gpt2", "bert", "llama"])
def test_the_same_without_logits_on_the_gpu(name):
    """Against the same model in float32 on the CPU: both bf16 paths are off by the roundings on the way, the fused one by no more than half as much again."""
    _, want, exact = step(name)
    worst = {}
    for fused in (False, True):
        torch.manual_seed(0)
        m = models(fused_vocab=fused)[name]().cuda().to(torch.bfloat16)
        loss = m(*batch(name, "cuda"))
        loss.backward()
        assert abs(float(loss) - float(want)) <= 0.05
        worst[fused] = {n: float((p.grad.float().cpu() - exact[n]).norm() / exact[n].norm().clamp(min=1e-6)) for n, p in m.named_parameters()}
    for n, e in worst[True].items():
        assert e <= 1.5 * worst[False][n] + 2 * half_step(torch.bfloat16), (n, e, worst[False][n])


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["gpt2", "bert"])
def test_autocast_with_dropout(name):
    torch.manual_seed(0)
    m = models(fused_vocab=True, dropout=0.1)[name]().cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = m(*batch(name, "cuda"))
    loss.backward()
    assert bool(loss.isfinite()) and all(p.grad is not None and p.grad.dtype == torch.float32 and bool(p.grad.isfinite().all()) for p in m.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_the_three_together(dtype, reduction):
    """Looked up, scaled, dropped with a residual, and the loss of the tied table: gradients against the formulas in 64 bits, taken from where each operator's inputs are as they were rounded."""
    n, d, rows, classes, p = 700, 136, 1500, 1403, 0.2
    g = torch.Generator(device="cuda").manual_seed(0)
    table = (torch.randn(rows, d, device="cuda", generator=g) / d ** 0.5).to(dtype).requires_grad_()
    r = torch.randn(n, d, device="cuda", generator=g).to(dtype)
    ids = torch.randint(0, rows, (n,), device="cuda", generator=g)
    targets = torch.randint(0, classes, (n,), device="cuda", generator=g)
    targets[::7] = -100
    up = torch.rand(n, device="cuda", generator=g) + 0.5 if reduction == "none" else torch.tensor(256.0, device="cuda")
    e = ops.embedding(ids, table, scale=8.0, padding_idx=3)
    x = ops.dropout(e, p, seed=11, residual=r)
    loss = ops.linear_cross_entropy(x, table, targets, num_classes=classes, reduction=reduction)
    dtable, dx = torch.autograd.grad(loss, (table, x), up)
    keep = kept((n, d), p, 11).cuda()
    assert torch.equal(x.detach(), (r.float() + torch.where(keep, e.detach().float() * float(torch.tensor(1 / share(p))), 0.0)).to(dtype))
    want = head(x.detach(), table.detach(), targets, None, classes, reduction=reduction, upstream=up)
    # dx as in the loss's own tests (a rounding of E and one of the result, exponents good to 2^-12 at these sizes); what reaches the table is dx dropped and summed by token, rounded twice more
    hs = half_step(dtype)
    size = want["dx_size"] * (hs + 2.0 ** -12) + want["dx"].abs() * hs + 2.0 ** -24
    assert bool(((dx.double() - want["dx"]).abs() <= size * 1.01).all())
    de = torch.where(keep, dx.double() / share(p), 0.0)
    looked, looked_size, count = embedding_grad(ids, de, rows, 8.0, 3)
    tol = looked_size * (hs * 1.01 + (count[:, None] + 4) * 2.0 ** -24) + looked.abs() * hs + want["dw_size"] * (2 * hs + 2.0 ** -12) + want["dw"].abs() * hs
    total = looked + want["dw"]
    tol = (tol + total.abs() * hs) * 1.02 + 2.0 ** -20
    assert bool(((dtable.double() - total).abs() <= tol).all()), ((dtable.double() - total).abs() - tol).max()


@pytest.mark.gpu
def test_a_captured_training_step():
    """A whole step of GPT-2 with masks from a tensor, replayed on other tokens: the same as run outside."""
    torch.manual_seed(0)
    table = torch.randn(1024, 128, device="cuda").mul(0.02).to(torch.bfloat16).requires_grad_()
    ids, targets, seed = torch.randint(0, 1000, (2, 64), device="cuda"), torch.randint(0, 1000, (2, 64), device="cuda"), torch.tensor(3, device="cuda")

    def run(seed):
        x = ops.dropout(ops.embedding(ids, table, scale=50.0), 0.1, seed=seed)
        loss = ops.linear_cross_entropy(x, table, targets, num_classes=1000)
        return loss, torch.autograd.grad(loss, table)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = run(seed)
    for s in (3, 4):
        seed.fill_(s), ids.random_(0, 1000), targets.random_(0, 1000)
        graph.replay()
        want, dtable = run(s)
        assert torch.equal(loss, want) and torch.equal(grad, dtable)


def _all_three(ids, table, targets, seed):
    x = ops.dropout(ops.embedding(ids, table, scale=50.0), 0.1, seed=seed)
    loss = ops.linear_cross_entropy(x, table, targets, num_classes=1000)
    return loss.detach(), torch.autograd.grad(loss, table)[0]


@pytest.mark.gpu
def test_two_threads_at_once():
    torch.manual_seed(0)
    work = []
    for i in range(2):
        table = torch.randn(1024, 128, device="cuda").mul(0.02).to(torch.float16 if i else torch.bfloat16).requires_grad_()
        work.append((torch.randint(0, 1000, (3, 70 + 30 * i), device="cuda"), table, torch.randint(0, 1000, (3, 70 + 30 * i), device="cuda"), 5 + i))
    want = [_all_three(*w) for w in work]
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = [_all_three(*work[i]) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(loss, want[i][0]) and torch.equal(grad, want[i][1]) for loss, grad in out)

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(run, range(2)))


@pytest.mark.gpu
def test_two_captured_graphs_replayed_at_once():
    torch.manual_seed(0)
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i, stream in enumerate(streams):
        table = torch.randn(1024, 128, device="cuda").mul(0.02).to(torch.bfloat16).requires_grad_()
        inputs = (torch.randint(0, 1000, (2, 300), device="cuda"), table, torch.randint(0, 1000, (2, 300), device="cuda"), torch.tensor(7 + i, device="cuda"))
        want = [t.clone() for t in _all_three(*inputs)]
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = _all_three(*inputs)
        graphs.append((graph, got, want, inputs))  # (a graph does not hold what it reads)
    for _ in range(20):
        for stream, (graph, *_) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _ in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
