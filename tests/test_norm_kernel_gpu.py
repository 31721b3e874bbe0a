"""RMS norm on the GPU against its formula in 64 bits: outputs, gradients, the 8-bit form, layouts, streams and graphs.

Tolerances. Squares and products are summed in fp32 over chains of at most 64 values a thread, 5 + 16 over threads: a sum of positive terms is
off by less than 96 * 2^-24 of itself, rstd by half of that and the 2 units of its approximation, and each result has five more fp32
roundings: 2^-17 of the terms' sizes covers it. On top comes the result's own rounding, half a step of its type. The weight's gradient is a sum
over rows of chains of at most rows / CTAs, 4, parts / 16 and 16 values, below 2^8 here: 2^-16 of the sum of its terms' sizes.
"""
import pytest
import torch

import _model_ops as plain
from _model_ops import rounding

pytestmark = pytest.mark.gpu
EPS = 1e-5
F32 = 2.0 ** -17
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def ops():
    from nangila import ops as o

    return o


def make(rows, d, dtype, seed=0, wdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + d)
    x = torch.randn(*((rows,) if isinstance(rows, int) else rows), d, device="cuda", generator=g).to(dtype)
    r = torch.randn(x.shape, device="cuda", generator=g).to(dtype)
    w = (1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(wdtype or dtype)
    return x, r, w, g


def assert_near(got, want, slack):
    bad = (got.double() - want).abs() > slack
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / slack.clamp(min=1e-300)).max()))


def check_all(x, r, w, dy, dh, dtype):
    y, h = ops().add_rms_norm(x, r, w, eps=EPS)
    assert torch.equal(h, (x.detach().float() + r.detach().float()).to(dtype))
    want = plain.norm(h.detach(), w.detach(), EPS)
    assert_near(y, want, rounding(want, dtype) + want.abs() * F32)
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (dy, dh))
    wx, ww, sx, sw = plain.norm_grads(h.detach(), w.detach(), EPS, dy, dh)
    assert dx.dtype == dtype and dw.dtype == w.dtype and dx.shape == x.shape
    assert_near(dx.reshape(wx.shape), wx, rounding(wx, dtype) + sx * F32)
    assert torch.equal(dx, dr)
    assert_near(dw, ww, rounding(ww, w.dtype) + sw * 2 * F32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 8), (3, 7), (5, 33), (1, 2048), (257, 128), (130, 520), (17, 1000), (9, 1001), (1500, 2048), (33, 4096), (6, 5632), (3, 8200),
                                    (2, 16384), (2, 20000), (1, 32768), (2, 32767), (3, 6),
                                    (5, 66), (11, 1004), (7, 1002), (300, 250), (3, 4100), (3, 3001), (2, 6002), (2, 16388), (2, 9999)])
def test_add_norm_and_gradients(rows, d, dtype):
    x, r, w, g = make(rows, d, dtype)
    dy = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    dh = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    check_all(x.requires_grad_(), r.requires_grad_(), w.requires_grad_(), dy, dh, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wdtype", TYPES)
def test_norm_without_residual_and_weight_of_another_type(dtype, wdtype):
    x, _, w, g = make(70, 264, dtype, wdtype=wdtype)
    x.requires_grad_(), w.requires_grad_()
    y = ops().rms_norm(x, w, eps=EPS)
    want = plain.norm(x.detach(), w.detach(), EPS)
    assert y.dtype == dtype
    assert_near(y, want, rounding(want, dtype) + want.abs() * F32)
    dy = torch.randn(70, 264, device="cuda", generator=g).to(dtype)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wx, ww, sx, sw = plain.norm_grads(x.detach(), w.detach(), EPS, dy)
    assert_near(dx, wx, rounding(wx, dtype) + sx * F32)
    assert dw.dtype == wdtype
    assert_near(dw, ww, rounding(ww, wdtype) + sw * 2 * F32)


def test_gradient_against_differences():
    # central differences of the 64-bit formula at 1e-4: their own error is of the order 1e-8; fp32's 2^-17 of terms near one is larger
    x, r, w, g = make(4, 24, torch.float32)
    dy, dh = torch.randn(4, 24, device="cuda", generator=g), torch.randn(4, 24, device="cuda", generator=g)
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(ops().add_rms_norm(x, r, w, eps=EPS), (x, w), (dy, dh))

    def loss(xv, wv):
        hv = xv + r.double()
        return float((plain.norm(hv, wv, EPS) * dy.double()).sum() + (hv * dh.double()).sum())

    xd, wd, step = x.detach().double(), w.detach().double(), 1e-4
    for i, j in [(0, 0), (1, 5), (3, 23), (2, 11)]:
        e = torch.zeros_like(xd)
        e[i, j] = step
        assert float(dx[i, j]) == pytest.approx((loss(xd + e, wd) - loss(xd - e, wd)) / (2 * step), abs=1e-4)
    e = torch.zeros_like(wd)
    e[7] = step
    assert float(dw[7]) == pytest.approx((loss(xd, wd + e) - loss(xd, wd - e)) / (2 * step), abs=1e-4)


@pytest.mark.parametrize("which", ["y", "h"])
def test_a_gradient_that_arrives_at_one_output_only(which):
    x, r, w, g = make(20, 512, torch.bfloat16)
    x.requires_grad_(), w.requires_grad_()
    y, h = ops().add_rms_norm(x, r, w, eps=EPS)
    up = torch.randn(20, 512, device="cuda", generator=g).bfloat16()
    dx, dw = torch.autograd.grad(y if which == "y" else h, (x, w), up, allow_unused=True)
    if which == "h":
        assert torch.equal(dx, up) and dw is None
    else:
        wx, ww, sx, sw = plain.norm_grads(h.detach(), w.detach(), EPS, up)
        assert_near(dx, wx, rounding(wx, torch.bfloat16) + sx * F32)


def test_only_what_is_wanted_gets_a_gradient():
    x, r, w, g = make(12, 64, torch.float32)
    y, h = ops().add_rms_norm(x, r, w.requires_grad_(), eps=EPS)
    (y.sum() + h.sum()).backward()
    _, ww, _, sw = plain.norm_grads(h.detach(), w.detach(), EPS, torch.ones_like(y))
    assert x.grad is None and r.grad is None
    assert_near(w.grad, ww, sw * 2 * F32)
    x.requires_grad_()
    y = ops().rms_norm(x, w.detach(), eps=EPS)
    y.sum().backward()
    wx, _, sx, _ = plain.norm_grads(x.detach(), w.detach(), EPS, torch.ones_like(y))
    assert_near(x.grad, wx, rounding(wx, torch.float32) + sx * F32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d,group", [(1, 128, 128), (5, 384, 128), (300, 2048, 128), (3, 5632, 128), (2, 32768, 128), (1, 1, None), (7, 33, None), (40, 1000, None),
                                          (2, 1001, None), (64, 2048, None), (3, 16385, None), (9, 1004, None), (5, 1002, None), (4, 250, None),
                                          (3, 4099, None), (2, 6002, None)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_eight_bits(rows, d, group, dtype, with_residual):
    # q: half a step of e4m3 is 2^-4 of the value, or 2^-10 of the scale among the subnormals; the scale and the value carry fp32's error
    x, r, w, _ = make(rows, d, dtype)
    x[0] *= 1e-3  # rows of different size
    out = ops().rms_norm_fp8(x, w, eps=EPS, residual=r if with_residual else None, group=group)
    q, scale = out[:2]
    h = x
    if with_residual:
        h = out[2]
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
    f = plain.norm(h, w, EPS).view(rows, -1, group or d)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (rows, d // group if group else 1)
    s = f.abs().amax(-1).clamp(min=1e-12) / 448
    sc = scale.view(s.shape)
    assert_near(sc, s, s * 2 * F32)
    got = q.double().view(f.shape) * sc.double().unsqueeze(-1)
    assert_near(got, f, f.abs() * (2.0 ** -4 + 3 * F32) + s.unsqueeze(-1) * 2.0 ** -10 * (1 + F32))
    assert torch.isfinite(q.float()).all()


def test_eight_bits_of_zeros_and_of_values_that_are_not_finite():
    x = torch.randn(4, 256, device="cuda").bfloat16()
    w = torch.ones(256, device="cuda").bfloat16()
    x[1] = 0
    x[2, 130] = float("nan")
    x[3, 5] = float("inf")
    q, scale = ops().rms_norm_fp8(x, w, eps=EPS, group=128)
    assert (q[1].float() == 0).all() and (scale[1] > 0).all() and torch.isfinite(scale[:2]).all()
    assert torch.isfinite(q[0].float()).all()
    # one value spoils rstd, and with it the row (nan), or makes it zero and itself nan (inf)
    assert torch.isnan(scale[2]).all() and torch.isnan(q[2].float()).all()
    assert torch.isnan(scale[3, 0]) and torch.isnan(q[3, :128].float()).all()
    assert (q[3, 128:].float() == 0).all()
    q, scale = ops().rms_norm_fp8(x, w, eps=EPS)
    assert torch.isnan(scale[2:]).all() and torch.isnan(q[2:].float()).all() and (q[1].float() == 0).all()


def test_values_that_are_not_finite_stay_in_their_row():
    x = torch.randn(6, 2048, device="cuda").bfloat16()
    x[2, 7] = float("nan")
    x[4, 9] = float("inf")
    w = torch.ones(2048, device="cuda").bfloat16()
    y = ops().rms_norm(x, w)
    assert torch.isnan(y[2]).all() and torch.isnan(y[4, 9]) and (y[4, :9] == 0).all()
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], ops().rms_norm(x[keep].contiguous(), w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    """Rows far apart, rows that start anywhere, transposed and expanded tensors, gradients of any layout."""
    base = torch.randn(40, 1032, device="cuda").to(dtype)
    w = torch.randn(1024, device="cuda").to(dtype)
    for x in (base[:, :1024], base[:, 8:1032], base[:, 3:1027], base[::2, 1:1025], torch.randn(1024, 24, device="cuda").to(dtype).t(),
              base[5, :1024].expand(7, 1024), base[:, :1024].view(8, 5, 1024), base[:, :1024].view(8, 5, 1024).transpose(0, 1), base[3, :1024]):
        y = ops().rms_norm(x, w)
        assert y.shape == x.shape and y.is_contiguous()
        want = plain.norm(x, w, EPS)
        assert_near(y, want, rounding(want, dtype) + want.abs() * F32)
        q, _ = ops().rms_norm_fp8(x, w, group=128)
        assert torch.equal(q.view(torch.uint8), ops().rms_norm_fp8(x.contiguous(), w, group=128)[0].view(torch.uint8))
    flat = torch.randn(1025, device="cuda").to(dtype)
    want = plain.norm(base[:, :1024], flat[1:], EPS)
    assert_near(ops().rms_norm(base[:, :1024], flat[1:]), want, rounding(want, dtype) + want.abs() * F32)
    x = base[:, :1024].clone().requires_grad_()
    for dy in (torch.ones(1, 1, device="cuda", dtype=dtype).expand(40, 1024), torch.randn(1024, 40, device="cuda").to(dtype).t(), base[:, 5:1029]):
        a, = torch.autograd.grad(ops().rms_norm(x, w), x, dy)
        b, = torch.autograd.grad(ops().rms_norm(x, w), x, dy.contiguous())
        wx, _, sx, _ = plain.norm_grads(x.detach(), w, EPS, dy)
        for got in (a, b):
            assert_near(got, wx, rounding(wx, dtype) + sx * F32)


def test_a_broadcast_input_gets_the_sum_of_its_gradients():
    row = torch.randn(1, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda")
    dy = torch.randn(5, 64, device="cuda")
    ops().rms_norm(row.expand(5, 64), w, eps=EPS).backward(dy)
    wx, _, sx, _ = plain.norm_grads(row.detach().expand(5, 64), w, EPS, dy)
    assert_near(row.grad[0], wx.sum(0), sx.sum(0) * 2 * F32)


def test_the_same_tensor_twice():
    x, _, w, g = make(20, 264, torch.float32)
    x.requires_grad_()
    dy = torch.randn(20, 264, device="cuda", generator=g)
    y, h = ops().add_rms_norm(x, x, w, eps=EPS)
    assert torch.equal(h, x.detach() * 2)
    dx, = torch.autograd.grad((y, h), x, (dy, dy))
    wx, _, sx, _ = plain.norm_grads(h.detach(), w, EPS, dy, dy)
    assert_near(dx, 2 * wx, rounding(2 * wx, torch.float32) + 2 * sx * F32)


def test_nothing_to_do():
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y, h = ops().add_rms_norm(x, x.detach(), w)
    (y.sum() + h.sum()).backward()
    assert y.shape == h.shape == (0, 16) and x.grad.shape == (0, 16) and torch.equal(w.grad, torch.zeros(16, device="cuda"))
    q, s = ops().rms_norm_fp8(torch.empty(2, 0, 128, device="cuda"), torch.ones(128, device="cuda"), group=128)
    assert q.shape == (2, 0, 128) and s.shape == (2, 0, 1)


def test_same_bits_every_time_and_on_another_stream():
    x, r, w, g = make(3000, 2048, torch.bfloat16)
    x.requires_grad_(), w.requires_grad_()

    def run():
        y, h = ops().add_rms_norm(x, r, w)
        return (y, h) + torch.autograd.grad((y, h), (x, w), (r, r))

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured_and_replayed_on_new_inputs():
    x, r, w, g = make(64, 1024, torch.bfloat16)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()

    def run():
        y, h = ops().add_rms_norm(xs, r, ws)
        q, s = ops().rms_norm_fp8(xs.detach(), ws.detach(), group=128)
        return (y, h, q, s) + torch.autograd.grad((y, h), (xs, ws), (r, r))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    with torch.no_grad():
        xs.copy_(torch.randn(64, 1024, device="cuda", generator=g))
    graph.replay()
    for a, b in zip(held, run()):
        assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)


def test_no_second_derivative_and_no_stale_saved_values():
    x, r, w, _ = make(4, 32, torch.float32)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="again"):
        torch.autograd.grad(ops().rms_norm(x, w).sum(), x, create_graph=True)
    y, h = ops().add_rms_norm(x, r, w)
    h.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_more_rows_than_one_wave_and_offsets_past_32_bits():
    rows, d = 1_100_000, 2048  # 2.25 G elements: offsets need 64 bits
    x = torch.ones(rows, d, device="cuda", dtype=torch.bfloat16)
    x[-1] = 3
    w = torch.full((d,), 2.0, device="cuda", dtype=torch.bfloat16)
    y = ops().rms_norm(x, w, eps=0.0)
    assert float(y[-1].min()) == float(y[-1].max()) == 2.0 and float(y[::100_000].min()) == 2.0
