"""The head's loss with few classes, few columns or few tokens, where roundings do not average out: each gradient within the bound of its own roundings."""
import pytest
import torch

from tests._head_bounds import check_grads_anywhere
from tests._vocab_ops import head
from tests.test_linear_ce_kernel_gpu import DEV, check_losses, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 33])
@pytest.mark.parametrize("d", [1, 3, 8])
def test_each_term_has_its_roundings(d, rows, reduction, dtype):
    for seed, n in enumerate((1, 2, 5, 40, 129, 257, 300, 700)):
        x, w, t, b = inputs(n, d, rows, dtype, None, torch.float32 if seed % 2 else None, seed=seed)
        g = torch.Generator(device=DEV).manual_seed(seed)
        up = torch.rand(n, device=DEV, generator=g) + 0.5 if reduction == "none" else torch.tensor(16.0, device=DEV)
        want = head(x, w, t, b, reduction=reduction, upstream=up)
        loss, grads = run(x, w, t, b, up, reduction=reduction)
        if reduction == "none":
            check_losses(loss, want, d, rows)
        check_grads_anywhere(grads, want, x, w, d, dtype)
