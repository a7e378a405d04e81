"""Optimisers beside the clip + Adam kernels: hidden matrices by orthogonalised momentum, the rest by Adam.

The reference trains with Adam alone (cradle_vae/models/utils/perturbation_lightning_module.py:147-150); this one is chosen
with ``lightning_module_kwargs.optimizer: muon``.
"""
from __future__ import annotations

import math
from collections import defaultdict
from typing import Dict, List, Tuple

import torch

from . import ops


def split_parameters(module: torch.nn.Module) -> Tuple[List[torch.nn.Parameter], List[torch.nn.Parameter]]:
    """(hidden matrices, the rest): the weights of the MLP trunks behind their first layer -- maps of one hidden layer to the
    next -- against input layers (whose columns are genes, treatments), output heads, norms, biases and tables."""
    hidden, rest = [], []
    for name, p in module.named_parameters():
        if not p.requires_grad:
            continue
        head, _, tail = name.rpartition("mlp.layers.")
        inner = p.dim() == 2 and bool(head or tail != name) and not tail.startswith("0.")
        (hidden if inner else rest).append(p)
    return hidden, rest


def _state_dtype(p: torch.Tensor) -> torch.dtype:
    return torch.promote_types(p.dtype, torch.float32)


def _widened(tensors: List[torch.Tensor]) -> List[torch.Tensor]:
    """The tensors themselves, or copies in fp32 of 16-bit ones."""
    return [t.to(_state_dtype(t)) for t in tensors]


def _narrowed(params: List[torch.Tensor], wide: List[torch.Tensor]) -> None:
    for p, w in zip(params, wide):
        if w.dtype != p.dtype:
            p.copy_(w)


class Muon(torch.optim.Optimizer):
    """Hidden matrices W (m, n): buf <- momentum buf + g;  W <- (1 - lr weight_decay) W - lr 0.2 sqrt(max(m, n)) O, O the
    Newton-Schulz orthogonalisation (``ops.orthogonalize``) of g + momentum buf -- the factor gives an update the root mean
    square of a typical Adam update (0.2), so one ``lr`` serves both groups.  Matrices of one shape go through one
    call.  Other parameters: Adam with L2 weight decay, as ``torch.optim.Adam``.  States are fp32 beside 16-bit parameters, which
    are rounded once a step."""

    def __init__(self, hidden, rest=(), lr: float = 1e-3, momentum: float = 0.95, weight_decay: float = 1e-6, steps: int = 5,
                 betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8):
        hidden, rest = list(hidden), list(rest)
        bad = [tuple(p.shape) for p in hidden if p.dim() != 2]
        if bad:
            raise ValueError(f"Muon: only matrices can be orthogonalised, got shapes {bad}")
        if not 0 <= momentum < 1 or lr < 0 or not 1 <= int(steps) <= 64:
            raise ValueError(f"Muon: lr={lr}, momentum={momentum}, steps={steps}")
        groups = [dict(params=ps, orthogonal=o) for ps, o in ((hidden, True), (rest, False)) if ps]
        super().__init__(groups, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, steps=int(steps), betas=betas, eps=eps))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            (self._orthogonal if group["orthogonal"] else self._adam)(group)
        return loss

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)  # (casts states to their parameter's type)
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip((i for g in state_dict["param_groups"] for i in g["params"]), params):
            for k, v in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(v):
                    self.state[p][k] = v.to(device=p.device, dtype=_state_dtype(p), copy=True)

    def _orthogonal(self, group) -> None:
        by_shape: Dict[tuple, List[torch.nn.Parameter]] = defaultdict(list)
        for p in group["params"]:
            if p.grad is not None:
                by_shape[(tuple(p.shape), p.dtype, p.device)].append(p)
        for (shape, _, _), params in by_shape.items():
            bufs = []
            for p in params:
                st = self.state[p]
                if not st:
                    st["momentum"] = torch.zeros_like(p, dtype=_state_dtype(p), memory_format=torch.contiguous_format)
                bufs.append(st["momentum"])
            grads = _widened([p.grad for p in params])
            torch._foreach_mul_(bufs, group["momentum"])
            torch._foreach_add_(bufs, grads)
            update = torch.stack(torch._foreach_add(grads, bufs, alpha=group["momentum"]))
            ops.orthogonalize(update, steps=group["steps"], out=update)
            wide = _widened(params)
            if group["weight_decay"]:
                torch._foreach_mul_(wide, 1.0 - group["lr"] * group["weight_decay"])
            torch._foreach_add_(wide, list(update.unbind(0)), alpha=-group["lr"] * 0.2 * math.sqrt(max(shape)))
            _narrowed(params, wide)

    def _adam(self, group) -> None:
        b1, b2 = group["betas"]
        for p in group["params"]:
            if p.grad is None:
                continue
            st = self.state[p]
            if not st:
                st["step"] = 0
                st["exp_avg"], st["exp_avg_sq"] = (torch.zeros_like(p, dtype=_state_dtype(p)) for _ in range(2))
            st["step"] += 1
            (g,), (wide,) = _widened([p.grad]), _widened([p])
            g = g.add(wide, alpha=group["weight_decay"]) if group["weight_decay"] else g
            st["exp_avg"].lerp_(g, 1 - b1)
            st["exp_avg_sq"].mul_(b2).addcmul_(g, g, value=1 - b2)
            denom = (st["exp_avg_sq"].sqrt() / math.sqrt(1 - b2 ** st["step"])).add_(group["eps"])
            wide.addcdiv_(st["exp_avg"], denom, value=-group["lr"] / (1 - b1 ** st["step"]))
            _narrowed([p], [wide])


OPTIMIZERS = ("adam", "muon")


def make_optimizer(name: str, module: torch.nn.Module, lr: float, weight_decay: float) -> torch.optim.Optimizer:
    if name == "adam":
        return torch.optim.Adam(module.parameters(), lr=lr, weight_decay=weight_decay)
    if name == "muon":
        return Muon(*split_parameters(module), lr=lr, weight_decay=weight_decay)
    raise ValueError(f"optimizer={name!r}: expected one of {OPTIMIZERS}")
