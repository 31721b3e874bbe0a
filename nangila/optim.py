"""Muon: momentum, made orthogonal, as the update of matrix parameters (``nangila.ops.muon_step``)."""
from __future__ import annotations

from typing import Any, Callable, Dict, Iterable, Optional, Union

import torch

from .ops.muon import COEFFICIENTS, _check_eps, _schedule, muon_step, update_scale


class Muon(torch.optim.Optimizer):
    """Muon for 2-D parameters; embeddings, heads, biases and norms belong to another optimizer.

    Every step takes ``M <- momentum M + G``, makes ``G + momentum M`` (``M`` without ``nesterov``) orthogonal by ``steps`` Newton-Schulz steps, and
    ``P <- P (1 - lr weight_decay) - lr s O`` with ``s`` after ``scale`` (``nangila.ops.muon.update_scale``; ``"rms"`` makes an update as large as AdamW's, whose
    learning rate then fits). The momentum is float32 whatever the parameters' type. On CUDA all parameters of one shape go through the kernels
    together. It works on whole matrices: under DistributedDataParallel (with or without a compression hook) every rank takes the same
    step; sharded parameters (``fully_shard``) are refused."""

    def __init__(self, params: Iterable, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                 coefficients=COEFFICIENTS, eps: float = 1e-7, scale: Optional[str] = "rms"):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=coefficients, eps=eps,
                                      scale=scale))

    def add_param_group(self, param_group: Dict[str, Any]) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            for name in ("lr", "momentum", "weight_decay"):
                if not group[name] >= 0:
                    raise ValueError(f"nangila: {name} must not be negative, got {group[name]}")
            _schedule(group["steps"], group["coefficients"])
            _check_eps(group["eps"])
            update_scale(1, 1, group["scale"])
            for p in group["params"]:
                if type(p).__name__ == "DTensor":
                    raise TypeError("nangila: Muon needs whole matrices, not the shards of a DTensor")
                if p.dim() != 2 or not p.is_contiguous():
                    raise ValueError(f"nangila: Muon takes packed 2-D parameters, got shape {tuple(p.shape)}; give the others to another optimizer")
        except Exception:
            self.param_groups.pop()
            raise

    @torch.no_grad()
    def step(self, closure: Optional[Callable[[], float]] = None) -> Optional[float]:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            for p in params:
                if p.grad.is_sparse:
                    raise RuntimeError("nangila: Muon does not take sparse gradients")
                if "momentum_buffer" not in self.state[p]:
                    self.state[p]["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            muon_step(params, [p.grad for p in params], [self.state[p]["momentum_buffer"] for p in params], lr=float(group["lr"]), momentum=group["momentum"],
                      nesterov=group["nesterov"], weight_decay=group["weight_decay"], steps=group["steps"], coefficients=group["coefficients"],
                      eps=group["eps"], scale=group["scale"])
        return loss

    def load_state_dict(self, state_dict: Dict[str, Union[Dict, list]]) -> None:
        super().load_state_dict(state_dict)
        # the base class takes the state to the parameters' type; the momentum stays in float32
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, own):
            entry = state_dict["state"].get(i, {})
            if "momentum_buffer" in entry:
                self.state[p]["momentum_buffer"] = torch.empty(p.shape, dtype=torch.float32, device=p.device).copy_(entry["momentum_buffer"])
