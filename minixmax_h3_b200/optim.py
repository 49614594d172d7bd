"""Muon: the optimiser whose step for a matrix is the orthogonal factor of its
averaged gradient, by ``ops.orthogonalize``.

For the matrices of trained layers (``block.TrainableCrossAttention.matrices``);
norms, biases and embeddings go to another optimiser.  No reference counterpart.
"""
from __future__ import annotations

import torch

from . import ops


class Muon(torch.optim.Optimizer):
    """m <- momentum m + (1 - momentum) g;  u = m, or with nesterov
    momentum m + (1 - momentum) g again;  p <- (1 - lr weight_decay) p -
    lr sqrt(max(1, rows / columns)) orthogonalize(u).

    Parameters are matrices, or stacks [..., m, n] of them, each
    orthogonalised by itself.  Those of one shape are orthogonalised in one
    call.  Averages are fp32; ``dtype`` is the type that an update is rounded
    to and orthogonalised in.  bf16's rounding is felt by what is small beside
    an update's large directions, fp32 costs 4 to 15 % more; fp16 does not hold
    the range of averaged gradients and is taken as fp32.  Gradients and
    parameters may be of any floating type: a parameter is updated in its own,
    so what is below its rounding is lost there.  State and steps follow the parameters' devices; a step can be
    captured into a CUDA graph once the averages exist."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5,
                 coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7,
                 dtype: torch.dtype = torch.bfloat16):
        if not lr >= 0.0 or not 0.0 <= momentum < 1.0 or not weight_decay >= 0.0:
            raise ValueError("Muon: lr and weight_decay are not negative, momentum is in [0, 1)")
        if dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise ValueError("Muon: updates are orthogonalised in bf16, fp16 or fp32")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coefficients=tuple(coefficients), eps=eps, dtype=dtype))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2 or not p.is_floating_point():
                self.param_groups.pop()
                raise ValueError(f"Muon is for matrices [..., m, n]: a parameter of shape {tuple(p.shape)}")

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # (which has rounded the averages to their parameters' types)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                average = state_dict["state"][i]["average"]
                self.state[p]["average"] = average.to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike: dict = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    if p.grad.is_sparse:
                        raise RuntimeError("Muon has no sparse gradients")
                    alike.setdefault((p.shape, p.device), []).append(p)
            for (shape, _), params in alike.items():
                self._update(group, shape, params)
        return loss

    def _update(self, group, shape, params) -> None:
        momentum = group["momentum"]
        grads, averages = [], []
        for p in params:
            state = self.state[p]
            if not state:
                state["average"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
            grads.append(p.grad.float())
            averages.append(state["average"])
        torch._foreach_lerp_(averages, grads, 1.0 - momentum)
        updates = torch._foreach_lerp(grads, averages, momentum) if group["nesterov"] else averages
        u = torch.stack(list(updates))
        if group["dtype"] != torch.float16:  # (1e-8 would be nothing, 1e5 infinite)
            u = u.to(group["dtype"])
        u = ops.orthogonalize(u, steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"], out=u)
        rows, columns = shape[-2:]
        if group["weight_decay"]:
            torch._foreach_mul_(params, 1.0 - group["lr"] * group["weight_decay"])
        scale = -group["lr"] * max(1.0, rows / columns) ** 0.5
        for p, o in zip(params, u.unbind()):
            p.add_(o.to(torch.float32) if p.dtype == torch.float32 else o, alpha=scale)
