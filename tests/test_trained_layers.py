"""What a trained layer and its quantised form do with gradients, devices and
sizes.  The CPU part runs no kernel."""
from __future__ import annotations

import pytest
import torch

from minixmax_h3_b200 import attention, block, modules, ops

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


# ----------------------------------------------------------------------------- quantised forms


def test_sizes_that_cannot_be_quantised(monkeypatch):
    """The products take K in multiples of 128 (int8) or 256 (nvfp4): said where the layer is made, not at its first call."""
    made = []
    monkeypatch.setattr(block, "load_quant_linear", lambda ql, w, fmt: made.append((tuple(w.shape), fmt)))
    good = {"hidden": 256, "heads": 4, "head_dim": 64, "cond_dim": 512}
    for fmt in ("int8_tensorwise", "nvfp4"):
        block.TrainableCrossAttention(**good).quantized(fmt)
    assert made == [(s, f) for f in ("int8_tensorwise", "nvfp4") for s in ((256, 256), (512, 512), (256, 256))]
    made.clear()
    for name, value, fmts in (("hidden", 192, ("int8_tensorwise", "nvfp4")), ("cond_dim", 160, ("int8_tensorwise", "nvfp4")),
                              ("heads", 3, ("int8_tensorwise", "nvfp4")), ("hidden", 384, ("nvfp4",)),
                              ("cond_dim", 128, ("nvfp4",)), ("heads", 2, ("nvfp4",))):
        layer = block.TrainableCrossAttention(**{**good, name: value})
        for fmt in fmts:
            with pytest.raises(ValueError, match="multiples of"):
                layer.quantized(fmt)
    with pytest.raises(ValueError):
        block.TrainableCrossAttention(**good).quantized("other")
    assert not made


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,dtype", [("int8_tensorwise", BF16), ("int8_tensorwise", F16), ("nvfp4", BF16), ("nvfp4", F16)])
def test_quantised_layer_is_its_parts(cuda, fmt, dtype):
    """Of bf16 and fp16 layers, in both formats: dense, with keys encoded once, and through the 8-bit cache."""
    torch.manual_seed(1)
    rope = ops.Rotary.build(32, interleaved=True, device=cuda)
    layer = block.TrainableCrossAttention(256, 4, 128, 512, kv_heads=2, rope=rope, compute_dtype=dtype, device=cuda)
    layer.norm.weight.data.normal_(1.0, 0.1)
    layer.norm.bias.data.normal_(0.0, 0.1)
    q8 = layer.quantized(fmt)
    x, cond = torch.randn(2, 37, 256, device=cuda, dtype=dtype), torch.randn(2, 21, 512, device=cuda, dtype=dtype)
    at, cond_at = torch.arange(37, device=cuda), torch.arange(21, device=cuda) + 4
    lens = torch.tensor([21, 9], dtype=torch.int32, device=cuda)
    h = ops.layer_norm(x, layer.norm.weight, layer.norm.bias, layer.norm.eps)
    q = ops.rotary(q8.q_proj(h.view(74, 256)).view(2, 37, 4, 128), None, at, rope)[0]
    kv = q8.kv_proj(cond.view(42, 512)).view(2, 21, 2, 2, 128)
    k, v = ops.rotary(kv[:, :, 0], None, cond_at, rope)[0], kv[:, :, 1]
    want = q8.out_proj(ops.cross_attention(q, k, v, kv_lens=lens).view(74, 512)).view(2, 37, 256)
    got = q8(x, cond, cond_lens=lens, positions=at, cond_positions=cond_at)
    assert got.dtype == dtype and torch.equal(got, want)
    kept = q8.encode(cond, cond_positions=cond_at)
    assert torch.equal(q8(x, kv=kept, cond_lens=lens, positions=at), want)
    cache = ops.KV8Cache.empty(2, 2, 128, device=cuda)
    table = torch.tensor([[1], [0]], dtype=torch.int32, device=cuda)
    q8.fill(cache, cond, table, torch.zeros(2, dtype=torch.int32, device=cuda), new_lens=lens, cond_positions=cond_at)
    o = ops.kv8_attention(q, cache, table, lens)
    got = q8(x, cache=cache, block_table=table, cond_lens=lens, positions=at)
    assert torch.equal(got, q8.out_proj(o.view(74, 512)).view(2, 37, 256))


# ----------------------------------------------------------------------------- rotary's gradients


def test_rotary_turns_only_gradients_that_are_there(monkeypatch):
    """One of two results used, or one of two inputs that requires a gradient: the other's is not turned."""
    turned = []

    def plain(q, k, positions, rope, *, inverse=False):
        turned.append((tuple(q.shape), None if k is None else tuple(k.shape), inverse))
        return (-q if inverse else 2 * q), None if k is None else (-k if inverse else 2 * k)

    monkeypatch.setattr(ops, "rotary", plain)
    rope, p = ops.Rotary.build(4, device="cpu"), torch.zeros(2, dtype=torch.int32)
    q, k = torch.randn(1, 2, 3, 8), torch.randn(1, 2, 1, 8)
    for wanted in ("q", "k", "qk"):
        for used in ("q", "k", "qk"):
            a, b = q.clone().requires_grad_("q" in wanted), k.clone().requires_grad_("k" in wanted)
            out = attention.rotary(a, b, p, rope)
            turned.clear()
            sum((o ** 2).sum() for o, n in zip(out, "qk") if n in used).backward()
            there = [n for n in "qk" if n in wanted and n in used]
            want = {0: [], 1: [(tuple((q if there == ["q"] else k).shape), None, True)],
                    2: [(tuple(q.shape), tuple(k.shape), True)]}[len(there)]
            assert turned == want
            for t, n in ((a, "q"), (b, "k")):
                if n not in wanted:
                    assert t.grad is None
                else:
                    assert torch.equal(t.grad, -4 * t.detach() if n in there else torch.zeros_like(t))
    # and their own gradients
    a = q.clone().requires_grad_()
    g = torch.randn_like(q).requires_grad_()
    da, = torch.autograd.grad(attention.rotary(a, k, p, rope)[0], a, g, create_graph=True)
    assert torch.equal(torch.autograd.grad(da, g, torch.ones_like(da))[0], 2 * torch.ones_like(q))
