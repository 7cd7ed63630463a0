"""Optimiser for the block's matrices: momentum whose update is orthogonalised on ``bibo_moe_orthogonalize``.

    matrices = [p for p in layer.parameters() if p.requires_grad and p.dim() >= 2]   # gate_proj, gate_up_proj, down_proj
    opt = bibo_b200.Muon(matrices, lr=0.02)

A stacked parameter [E, m, n] is E matrices, each orthogonalised by itself (``gate_up_proj`` and ``down_proj`` of
``BiBoFusedExperts``).  Vectors and scalars (``radial_theta``, norm weights) belong to another optimiser and are refused.
"""
from __future__ import annotations

import torch

from . import functional as Fn

__all__ = ["Muon"]


class Muon(torch.optim.Optimizer):
    """One step, for a parameter w with gradient g and momentum buffer v (fp32):

        v <- momentum v + g;   u = g + momentum v (nesterov) or v
        w <- (1 - lr weight_decay) w - lr max(1, m/n)^0.5 orthogonalize(u)
    """

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients=Fn.NEWTON_SCHULZ, eps: float = 1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            lr, momentum, weight_decay = group["lr"], group["momentum"], group["weight_decay"]
            if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
                raise ValueError(f"Muon: lr={lr}, momentum={momentum}, weight_decay={weight_decay}")
            for p in group["params"]:
                if p.dim() < 2:
                    raise ValueError(f"Muon takes matrices and stacks of them, got a parameter of shape {tuple(p.shape)}")
            try:
                Fn.check_polynomials(group["steps"], group["coefficients"], group["eps"])
            except RuntimeError as e:
                raise ValueError(f"Muon: {e}") from None
        except ValueError:
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        keys = [k for group in state_dict["param_groups"] for k in group["params"]]
        for key, p in zip(keys, [p for group in self.param_groups for p in group["params"]]):
            buf = state_dict["state"].get(key, {}).get("momentum_buffer")
            if buf is not None:                     # torch casts a state to the parameter's type; the momentum stays in fp32
                self.state[p]["momentum_buffer"] = buf.to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:              # nothing is stepped, and no momentum touched, where something is refused
            for p in group["params"]:
                if p.grad is not None and p.numel() and (not p.is_cuda or p.grad.layout != torch.strided or p.is_complex()):
                    raise RuntimeError(f"Muon: a parameter of shape {tuple(p.shape)} on {p.device} with a gradient of {p.grad.dtype}, "
                                       f"{p.grad.layout}: it takes dense real ones on CUDA devices (there is no CPU implementation)")
        for group in self.param_groups:
            momentum = group["momentum"]
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():   # every replay would clear the momentum
                        raise RuntimeError("Muon: take a step, or load a state, before a step is captured in a graph")
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                buf = state["momentum_buffer"]
                buf.mul_(momentum).add_(p.grad)
                u = torch.add(p.grad, buf, alpha=momentum).float() if group["nesterov"] else buf
                u = Fn.orthogonalize(u.contiguous(), group["steps"], group["coefficients"], group["eps"])
                if group["weight_decay"]:
                    p.mul_(1 - group["lr"] * group["weight_decay"])
                p.add_(u, alpha=-group["lr"] * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5)
        return loss
