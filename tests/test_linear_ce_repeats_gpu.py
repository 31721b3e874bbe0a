"""The same call gives the same bits, whichever CTAs take which tiles."""
import pytest
import torch

from tests.test_linear_ce_kernel_gpu import DEV, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("n,d,rows", [(16, 2048, 5000), (200, 512, 9000), (1229, 1024, 30592), (4096, 768, 8000)])
def test_twenty_times(n, d, rows, reduction, dtype):
    x, w, t, b = inputs(n, d, rows, dtype, rows - 70, torch.float32, ignored=0.1)
    up = torch.rand(n, device=DEV) if reduction == "none" else torch.tensor(64.0, device=DEV)
    loss, grads = run(x, w, t, b, up, num_classes=rows - 70, reduction=reduction)
    for _ in range(20):
        again, others = run(x, w, t, b, up, num_classes=rows - 70, reduction=reduction)
        assert torch.equal(loss, again) and all(torch.equal(a, c) for a, c in zip(grads, others))
