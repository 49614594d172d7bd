"""What a trained layer and its quantised form do with gradients, devices and
sizes.  The CPU part runs no kernel."""
from __future__ import annotations

import pytest
import torch

from minixmax_h3_b200 import block, modules, ops

BF16, F16 = torch.bfloat16, torch.float16


# ----------------------------------------------------------------------------- gradients that are not there


def test_a_norm_that_wants_gradients_raises(monkeypatch):
    """The projection behind the norm is quantised and would drop them without a word."""
    class Plain(modules.QuantLinear):
        def forward(self, x):
            return torch.zeros(*x.shape[:-1], self.out_features)

    class Layers(modules.Ops):
        QuantLinear = Plain

    monkeypatch.setattr(modules, "layer_norm", lambda x, w, b, eps: torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, eps))
    monkeypatch.setattr(ops, "cross_attention", lambda q, k, v, **kw: torch.zeros_like(q))
    layer = block.CrossAttention(64, 1, 64, 32, operations=Layers, norm=True)
    x, cond = torch.zeros(1, 2, 64), torch.zeros(1, 3, 32)
    assert layer(x, cond).shape == x.shape
    for p in (layer.norm.weight, layer.norm.bias):
        p.requires_grad_(True)
        with pytest.raises(RuntimeError, match="no gradients"):
            layer(x, cond)
        with torch.no_grad():
            assert layer(x, cond).shape == x.shape
        p.requires_grad_(False)
    layer.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradients"):
        layer(x, cond)
    bare = block.CrossAttention(64, 1, 64, 32, operations=Layers).requires_grad_(True)
    assert bare(x, cond).shape == x.shape
