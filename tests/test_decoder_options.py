"""The decoder's configuration: options that would have no effect are refused, whenever they are set."""
import pytest
import torch

from nangila.models import Llama, LlamaConfig
from nangila.models.llama import DecoderBlock

SMALL = dict(n_layer=1, n_head=2, n_kv_head=1, d_model=32, d_mlp=48, vocab_size=64, max_seq=16)


@pytest.mark.parametrize("options", [dict(rope_factor=4.0), dict(rope_original_seq=128), dict(rope_factor=4.0, rope_original_seq=128), dict(rope_layout="half"), dict(rope_dim=8),
                                     dict(rope_scaling="ntk", rope_factor=2.0)])
def test_what_needs_fused(options):
    with pytest.raises(ValueError, match="fused"):
        LlamaConfig(**SMALL, **options)
    cfg = LlamaConfig(**SMALL)
    for k, v in options.items():
        setattr(cfg, k, v)
    for build in (Llama, DecoderBlock):  # set later, past the first check
        with pytest.raises(ValueError, match="fused"):
            build(cfg)


@pytest.mark.parametrize("options", [dict(rope_factor=4.0), dict(rope_original_seq=128), dict(rope_scaling="linear", rope_factor=2.0, rope_original_seq=64), dict(rope_layout="pairs"),
                                     dict(rope_dim=0), dict(rope_dim=7), dict(rope_dim=18), dict(rope_dim=-2)])
def test_what_fused_refuses(options):
    with pytest.raises(ValueError, match="nangila: rope"):
        LlamaConfig(**SMALL, fused=True, **options)


def test_fused_cleared_again():
    cfg = LlamaConfig(**SMALL, fused=True, rope_layout="half")
    cfg.fused = False
    with pytest.raises(ValueError, match="fused"):
        Llama(cfg)


def test_a_model_keeps_what_it_was_built_from():
    torch.manual_seed(0)
    cfg = LlamaConfig(**SMALL, fused=True, rope_layout="half")
    m = Llama(cfg)
    idx = torch.randint(0, 64, (1, 12))
    want = m(idx)
    m._rope = None
    cfg.fused, cfg.rope_layout, cfg.rope_theta = False, "interleaved", 5.0
    assert torch.equal(m(idx), want)


def test_all_columns_can_be_named():
    for dim in (2, 16, None):
        m = Llama(LlamaConfig(**SMALL, fused=True, rope_dim=dim))
        m(torch.randint(0, 64, (1, 12)))
        assert m._rope.shape[1] == (dim or 16) // 2


@pytest.mark.parametrize("fused", [False, True])
def test_training_after_an_evaluation_in_inference_mode(fused):
    m = Llama(LlamaConfig(**SMALL, fused=fused))
    idx = torch.randint(0, 64, (1, 12))
    with torch.inference_mode():
        want = m(idx)
    out = m(idx)
    out.sum().backward()
    assert torch.equal(out, want) and all(p.grad is not None for p in m.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
def test_training_after_an_evaluation_in_inference_mode_on_the_gpu(fused):
    m = Llama(LlamaConfig(**SMALL, fused=fused)).cuda()
    idx = torch.randint(0, 64, (1, 12), device="cuda")
    with torch.inference_mode():
        m(idx)
    m(idx).sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())
