"""Gradients that the forward pass forms along with the loss are tensors that autograd has saved: for hooks, checkpoints, and passes that keep the graph."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from nangila import ops
from tests._head_bounds import check_grads_anywhere
from tests._vocab_ops import head
from tests.test_linear_ce_kernel_gpu import DEV, inputs

pytestmark = pytest.mark.gpu


def leaves_of(*tensors):
    return [v.detach().clone().requires_grad_() for v in tensors]


def passes(x, w, t, b, up, through=None):
    leaves = leaves_of(x, w, b)
    loss = (through or (lambda f, *a: f(*a)))(lambda u, v, c: ops.linear_cross_entropy(u, v, t, bias=c), *leaves)
    return torch.autograd.grad(loss, leaves, up)


def test_hooks_see_them():
    x, w, t, b = inputs(300, 64, 500, bias=torch.float16)
    up = torch.tensor(3.0, device=DEV)
    want = passes(x, w, t, b, up)
    packed = []

    def pack(v):
        packed.append((v.shape, v.dtype))
        return v.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v.to(DEV)):
        got = passes(x, w, t, b, up)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    # (inputs and gradients alike)
    assert packed.count(((300, 64), torch.bfloat16)) == 2 and packed.count(((500, 64), torch.bfloat16)) == 2 and packed.count(((500,), torch.float32)) == 1


def test_a_checkpoint_keeps_none_of_them():
    n, d, rows = 256, 512, 20000
    x, w, t, b = inputs(n, d, rows, bias=torch.float32)
    up = torch.tensor(2.0, device=DEV)
    want = passes(x, w, t, b, up)
    leaves = leaves_of(x, w, b)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = checkpoint(lambda u, v, c: ops.linear_cross_entropy(u, v, t, bias=c), *leaves, use_reentrant=False)
    assert torch.cuda.memory_allocated() - before < rows * d  # (half of what dw takes)
    got = torch.autograd.grad(loss, leaves, up)
    assert all(torch.equal(a, c) for a, c in zip(want, got))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_passes_that_keep_the_graph(dtype):
    x, w, t, b = inputs(300, 64, 500, dtype, bias=torch.float32)
    leaves = leaves_of(x, w, b)
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    results = []
    for up, keep in ((256.0, True), (3.0, True), (256.0, True), (3.0, False)):
        grads = torch.autograd.grad(loss, leaves, torch.tensor(up, device=DEV), retain_graph=keep)
        check_grads_anywhere(grads, head(x, w, t, b, upstream=up), x, w, 64, dtype, results=2)
        results.append([g.clone() for g in grads])
        for g in grads:  # they are the caller's
            g.fill_(float("nan"))
    for first, second in ((0, 2), (1, 3)):
        assert all(torch.equal(a, c) for a, c in zip(results[first], results[second]))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaves)


def test_one_at_a_time():
    x, w, t, b = inputs(300, 64, 500, bias=torch.float32)
    up = torch.tensor(0.5, device=DEV)
    want = passes(x, w, t, b, up)
    leaves = leaves_of(x, w, b)
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    for i, leaf in enumerate(leaves):
        got, = torch.autograd.grad(loss, leaf, up, retain_graph=i < 2)
        assert torch.equal(got, want[i])


def test_accumulated_into_the_leaves():
    x, w, t, b = inputs(300, 64, 500, bias=torch.float32)
    want = passes(x, w, t, b, None)
    leaves = leaves_of(x, w, b)
    for _ in range(2):
        ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2]).backward()
    assert all(torch.equal(v.grad, 2 * g) for v, g in zip(leaves, want))
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    for v in leaves:
        v.grad = None
    loss.backward(retain_graph=True)
    loss.backward()
    assert all(torch.equal(v.grad, 2 * g) for v, g in zip(leaves, want))
