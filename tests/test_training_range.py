"""CPU: values and settings that a trained layer meets beyond the ordinary ones.  No kernel runs."""
from __future__ import annotations

import pytest
import torch

from minixmax_h3_b200 import ops, optim


def plain(x, *, steps, coefficients, eps, out=None):
    a, b, c = coefficients
    y = x.double()
    y = y / (torch.linalg.matrix_norm(y)[..., None, None] + eps)
    for _ in range(steps):
        g = y @ y.mT
        y = a * y + (b * g + c * (g @ g)) @ y
    y = y.to(x.dtype)
    return y if out is None else out.copy_(y)


@pytest.mark.parametrize("size", [1e-12, 1e-9, 1e-5, 1.0, 1e6, 1e9])
def test_muon_fp16_holds_any_gradient(monkeypatch, size):
    """Averages beyond f16's range, and below its smallest numbers, move the parameters as in fp32: beside the
    largest element of the movement by a rounding to f16 and one of the parameter at most."""
    monkeypatch.setattr(ops, "orthogonalize", plain)
    g = torch.Generator().manual_seed(0)
    grads = [size * torch.randn(s, generator=g) for s in ((24, 30), (24, 30), (40, 9))]
    grads[1] = grads[1] * 1e-3  # of one call with the first
    moved = {}
    for dtype in (torch.float32, torch.float16):
        params = [torch.zeros_like(t).requires_grad_() for t in grads]
        opt = optim.Muon(params, lr=1.0, dtype=dtype)
        for p, t in zip(params, grads):
            p.grad = t.clone()
        opt.step()
        moved[dtype] = [p.detach() for p in params]
    for a, b in zip(moved[torch.float16], moved[torch.float32]):
        assert b.abs().max() > 0 and (a - b).abs().max() <= (2.0 ** -11 + 2.0 ** -24) * b.abs().max()
