"""Llama-style decoder (RMSNorm, rotary position embedding, SwiGLU MLP, untied head, no biases), the
model of the fully-sharded benchmark: 24 layers, d_model 2048, 16 heads, SwiGLU 5632, vocabulary
32000, sequence 2048 (about 1.3 B parameters).

The reference's FSDP examples wrap Hugging Face Llama checkpoints (examples/train_fsdp_llm.py); here
the architecture is defined directly and initialised randomly. Each :class:`DecoderBlock` is the unit
``fully_shard`` wraps.

``LlamaConfig(fused=True)`` takes the norms (with the residual's addition inside a block) and the rotary positions through
``nangila.ops``: one kernel each, forward and backward, where PyTorch's operations make several passes. Results agree with the other
path up to the last rounding (the benchmark's step on one GPU: 126 -> 90 ms). It also opens the positions' options: the half layout, part of the head, scaling for long contexts.
"""
from __future__ import annotations

from dataclasses import dataclass, replace
from typing import Optional, Union

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


@dataclass
class LlamaConfig:
    n_layer: int = 24
    n_head: int = 16
    n_kv_head: int = 16
    d_model: int = 2048
    d_mlp: int = 5632
    vocab_size: int = 32000
    max_seq: int = 2048
    rope_theta: float = 10000.0
    eps: float = 1e-5
    fused: bool = False                      # nangila.ops for norms and positions; what follows needs it
    rope_layout: str = "interleaved"         # or "half"
    rope_dim: Optional[int] = None           # turned columns of a head; None: all
    rope_scaling: Optional[str] = None       # "linear", "ntk" or "yarn" (nangila.ops.rotary_table)
    rope_factor: float = 1.0
    rope_original_seq: Optional[int] = None

    def __post_init__(self):
        self.check()

    def check(self) -> None:
        """Refuses options that would have no effect. Models and blocks check again what they are built from, for fields can be set in between."""
        if not self.fused and (self.rope_layout, self.rope_dim, self.rope_scaling, self.rope_factor, self.rope_original_seq) != ("interleaved", None, None, 1.0, None):
            raise ValueError("nangila: rope_layout, rope_dim, rope_scaling, rope_factor and rope_original_seq need fused=True")
        if self.rope_scaling is None and self.rope_factor != 1.0:
            raise ValueError("nangila: rope_factor needs a rope_scaling")
        if self.rope_scaling != "yarn" and self.rope_original_seq is not None:
            raise ValueError("nangila: rope_original_seq needs rope_scaling='yarn'")
        if self.rope_layout not in ops.positions.LAYOUTS:
            raise ValueError(f"nangila: rope_layout must be one of {ops.positions.LAYOUTS}, got {self.rope_layout!r}")
        head_dim = self.d_model // self.n_head
        if self.rope_dim is not None and not (2 <= self.rope_dim <= head_dim and self.rope_dim % 2 == 0):
            raise ValueError(f"nangila: rope_dim must be even and 2 to {head_dim} (a head's columns), got {self.rope_dim}")

    @staticmethod
    def llama_1_3b() -> "LlamaConfig":
        return LlamaConfig()

    @staticmethod
    def tiny() -> "LlamaConfig":
        return LlamaConfig(n_layer=2, n_head=4, n_kv_head=2, d_model=128, d_mlp=352, vocab_size=1024, max_seq=128)


class RMSNorm(nn.Module):
    def __init__(self, d: int, eps: float):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d))
        self.eps = eps

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return F.rms_norm(x, (x.size(-1),), self.weight, self.eps)


def rope_table(seq: int, head_dim: int, theta: float, device) -> torch.Tensor:
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    ang = torch.outer(torch.arange(seq, device=device, dtype=torch.float32), inv)
    return torch.stack((ang.cos(), ang.sin()), dim=-1)  # [seq, head_dim / 2, 2]


def apply_rope(x: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """x: [b, t, h, d]; rotates consecutive (even, odd) pairs."""
    b, t, h, d = x.shape
    xf = x.float().view(b, t, h, d // 2, 2)
    cos, sin = table[:t, None, :, 0], table[:t, None, :, 1]
    out = torch.stack((xf[..., 0] * cos - xf[..., 1] * sin, xf[..., 0] * sin + xf[..., 1] * cos), dim=-1)
    return out.view(b, t, h, d).to(x.dtype)


class Angles:
    """The table of the fused path, float32: not a tensor among a block's inputs, which FSDP's mixed precision takes to the parameters' type."""

    def __init__(self, table: torch.Tensor):
        self.table = table


class DecoderBlock(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        cfg.check()
        self.h, self.kv = cfg.n_head, cfg.n_kv_head
        self.hd = cfg.d_model // cfg.n_head
        self.fused, self.layout = cfg.fused, cfg.rope_layout
        self.norm1 = RMSNorm(cfg.d_model, cfg.eps)
        self.wq = nn.Linear(cfg.d_model, self.h * self.hd, bias=False)
        self.wk = nn.Linear(cfg.d_model, self.kv * self.hd, bias=False)
        self.wv = nn.Linear(cfg.d_model, self.kv * self.hd, bias=False)
        self.wo = nn.Linear(self.h * self.hd, cfg.d_model, bias=False)
        self.norm2 = RMSNorm(cfg.d_model, cfg.eps)
        self.gate = nn.Linear(cfg.d_model, cfg.d_mlp, bias=False)
        self.up = nn.Linear(cfg.d_model, cfg.d_mlp, bias=False)
        self.down = nn.Linear(cfg.d_mlp, cfg.d_model, bias=False)

    def forward(self, x: torch.Tensor, rope: Union[torch.Tensor, Angles]) -> torch.Tensor:
        if self.fused:
            return self._fused(x, rope)
        b, t, _ = x.shape
        y = self.norm1(x)
        q = apply_rope(self.wq(y).view(b, t, self.h, self.hd), rope).transpose(1, 2)
        k = apply_rope(self.wk(y).view(b, t, self.kv, self.hd), rope).transpose(1, 2)
        v = self.wv(y).view(b, t, self.kv, self.hd).transpose(1, 2)
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=self.kv != self.h)
        x = x + self.wo(a.transpose(1, 2).reshape(b, t, self.h * self.hd))
        y = self.norm2(x)
        return x + self.down(F.silu(self.gate(y)) * self.up(y))

    def _fused(self, x: torch.Tensor, rope: Angles) -> torch.Tensor:
        b, t, _ = x.shape
        y = ops.rms_norm(x, self.norm1.weight, eps=self.norm1.eps)
        q, k = ops.rotary(self.wq(y).view(b, t, self.h, self.hd), self.wk(y).view(b, t, self.kv, self.hd), rope.table, layout=self.layout)
        v = self.wv(y).view(b, t, self.kv, self.hd).transpose(1, 2)
        a = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v, is_causal=True, enable_gqa=self.kv != self.h)
        a = self.wo(a.transpose(1, 2).reshape(b, t, self.h * self.hd))
        # (under autocast the projection has another type than the residual stream)
        y, x = ops.add_rms_norm(a.to(x.dtype), x, self.norm2.weight, eps=self.norm2.eps)
        return x + self.down(F.silu(self.gate(y)) * self.up(y))


class Llama(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.cfg = cfg = replace(cfg)  # checked; what is set in the caller's later does not change a model that is built
        self.embed = nn.Embedding(cfg.vocab_size, cfg.d_model)
        self.blocks = nn.ModuleList([DecoderBlock(cfg) for _ in range(cfg.n_layer)])
        self.norm = RMSNorm(cfg.d_model, cfg.eps)
        self.head = nn.Linear(cfg.d_model, cfg.vocab_size, bias=False)
        for m in self.modules():
            if isinstance(m, (nn.Linear, nn.Embedding)):
                nn.init.normal_(m.weight, std=0.02)
        self._rope: torch.Tensor | None = None

    def forward(self, idx: torch.Tensor, targets: torch.Tensor | None = None):
        t = idx.size(1)
        if self._rope is None or self._rope.device != idx.device or self._rope.size(0) < t:
            with torch.inference_mode(False):  # (a table made by an evaluation serves the training that follows)
                self._rope = self._table(max(t, self.cfg.max_seq), idx.device)
        x = self.embed(idx)
        rope = Angles(self._rope) if self.cfg.fused else self._rope
        for blk in self.blocks:
            x = blk(x, rope)
        logits = self.head(ops.rms_norm(x, self.norm.weight, eps=self.norm.eps) if self.cfg.fused else self.norm(x))
        if targets is None:
            return logits
        from ..ops.fused_ce import fused_cross_entropy  # fused kernels for bf16 logits on a GPU, PyTorch's path otherwise

        return fused_cross_entropy(logits.view(-1, logits.size(-1)), targets.reshape(-1))

    def _table(self, seq: int, device) -> torch.Tensor:
        cfg = self.cfg
        head_dim = cfg.d_model // cfg.n_head
        if not cfg.fused:
            return rope_table(seq, head_dim, cfg.rope_theta, device)
        return ops.rotary_table(seq, head_dim if cfg.rope_dim is None else cfg.rope_dim, cfg.rope_theta, device, scaling=cfg.rope_scaling, factor=cfg.rope_factor,
                                original_seq=cfg.rope_original_seq)

    def num_params(self) -> int:
        return sum(p.numel() for p in self.parameters())
