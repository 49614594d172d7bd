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


# ----------------------------------------------------------------------------- rotations move with their layer


def test_rotations_move(monkeypatch):
    rope = ops.Rotary.build(32, factor=1.5, interleaved=True, device="cpu")
    assert rope.to("cpu") is rope
    far = rope.to("meta")
    assert far.turns.is_meta and (far.sections, far.interleaved, far.factor) == (rope.sections, True, 1.5)
    layers = [block.CrossAttention(64, 1, 64, 32, rope=rope), block.TrainableCrossAttention(64, 1, 64, 32, rope=rope)]
    moves = []
    monkeypatch.setattr(ops.Rotary, "to", lambda self, device: moves.append(torch.device(device)) or self)
    for layer in layers:
        outer = torch.nn.Sequential(torch.nn.Sequential(layer))
        outer.to("cpu", torch.float64)
        assert moves.pop() == torch.device("cpu") and layer.rope is rope and rope.turns.dtype == torch.int64
        outer.half().share_memory()
        assert len(moves) == 2 and rope.turns.dtype == torch.int64
        moves.clear()
        outer.to("meta")  # values would be lost
        assert not moves and not layer.rope.turns.is_meta
        outer.to_empty(device="cpu")
        assert moves.pop() == torch.device("cpu") and torch.equal(layer.rope.turns, rope.turns)
        moves.clear()
    block.CrossAttention(64, 1, 64, 32).to("cpu")
    assert not moves


@pytest.mark.gpu
def test_layer_built_elsewhere(cuda):
    """Built on the CPU, moved and called: the same bits as built in its place."""
    torch.manual_seed(0)
    here = block.TrainableCrossAttention(128, 2, 64, 128, rope=ops.Rotary.build(64, device="cpu"))
    there = block.TrainableCrossAttention(128, 2, 64, 128, rope=ops.Rotary.build(64, device=cuda), device=cuda)
    there.load_state_dict(here.state_dict())
    here = here.to(cuda)
    x, cond = torch.randn(2, 9, 128, device=cuda), torch.randn(2, 5, 128, device=cuda)
    where = {"positions": torch.arange(9, device=cuda), "cond_positions": torch.arange(5, device=cuda)}
    assert torch.equal(here(x, cond, **where), there(x, cond, **where))
