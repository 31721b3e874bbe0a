"""Numbers of heads that the kernels' 32-bit counts do not hold."""
import pytest
import torch

from nangila import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [2 ** 30 + 1, 2 ** 31, 2 ** 32 + 1])
def test_too_many_heads_are_refused(heads):
    table = ops.rotary_table(1, 2, device="cuda")
    one, many = torch.zeros(1, 1, 1, 2, device="cuda"), torch.zeros(1, 1, 1, 2, device="cuda").expand(1, 1, heads, 2)  # (one head's memory)
    for call in (lambda: ops.rotary(many, None, table), lambda: ops.rotary(one, many, table)):
        with pytest.raises(ValueError, match="nangila.*heads"):
            call()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_many_heads(layout):
    """Around the 65536 heads up to which a group of tokens takes them all together."""
    table = ops.rotary_table(3, 8, device="cuda")
    for heads in (65535, 65536, 65537):
        q = torch.randn(1, 3, heads, 8, device="cuda")
        got = ops.rotary(q, None, table, layout=layout)
        for h in (0, 1, heads // 2, heads - 1):
            assert torch.equal(got[:, :, h], ops.rotary(q[:, :, h:h + 1], None, table, layout=layout)[:, :, 0])
