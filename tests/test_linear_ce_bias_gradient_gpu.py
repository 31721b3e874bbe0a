"""The bias's gradient of the head's loss is rounded once, to the bias's type, when the upstream gradient is known."""
import pytest
import torch

from nangila import ops
from tests._head_bounds import check_grads_anywhere
from tests._vocab_ops import head
from tests.test_linear_ce_kernel_gpu import DEV, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("upstream", [65536.0, 3.0, 1 / 3, 1.0, 0.0])
@pytest.mark.parametrize("n", [60, 3000])
def test_one_rounding_behind_the_upstream_gradient(n, upstream, bias):
    # over 3000 tokens values of 1e-5 for an upstream gradient of one: subnormal in half precision, of which scaled losses lie far above
    d, rows, classes = 64, 900, 870
    x, w, t, b = inputs(n, d, rows, torch.bfloat16, classes, bias, ignored=0.2)
    up = torch.tensor(upstream, device=DEV)
    want = head(x, w, t, b, classes, upstream=upstream)
    _, grads = run(x, w, t, b, up, num_classes=classes)
    assert grads[2].dtype == bias and not grads[2][classes:].any()
    check_grads_anywhere(grads, want, x, w, d, torch.bfloat16, results=2)  # (dx and dw have been rounded for one)
    # the same sums, rounded here
    _, exact = run(x, w, t, b.float(), up, num_classes=classes)
    assert torch.equal(grads[2], exact[2].to(bias))


def test_replayed_and_taken_twice():
    x, w, t, b = inputs(300, 64, 500, bias=torch.float16)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    first, second = (torch.autograd.grad(loss, leaves, torch.tensor(up, device=DEV), retain_graph=True) for up in (4096.0, 2048.0))
    for grads, up in ((first, 4096.0), (second, 2048.0)):
        check_grads_anywhere(grads, head(x, w, t, b, upstream=up), x, w, 64, torch.bfloat16)
    # passes that are captured leave what the forward pass has formed (no eager graph of the same leaves may live meanwhile)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    side, factor = torch.cuda.Stream(), torch.tensor(4096.0, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2]), leaves, factor)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        grads = torch.autograd.grad(loss, leaves, factor)
    for up in (4096.0, 2048.0):
        factor.fill_(up)
        graph.replay()
        graph.replay()
        check_grads_anywhere(grads, head(x, w, t, b, upstream=up), x, w, 64, torch.bfloat16)
        assert torch.equal(grads[2].double() / up, first[2].double() / 4096.0)
