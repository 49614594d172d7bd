"""GPU: the trained layer beside the same layer of elementary torch operations
in the same type (products in 16 bits, norm, rotations and softmax in 32, each
result rounded once): both round in the same places, so against 64 bits the
kernels' error is at most twice the plain layer's, in Frobenius norm, for the
result and for each parameter's gradient by itself."""
from __future__ import annotations

import math

import pytest
import torch

from minixmax_h3_b200 import _lib, block, ops

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def layer_of(p, x, cond, lens, at, cond_at, heads, kv_heads, eps, dtype):
    """The layer; dtype torch.float64: no rounding.  Halves turned, theta 10000."""
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    d = p["q_proj"].shape[0] // heads

    def turn(t, where):
        n = d // 2
        a = where.double()[:, None] * 10000.0 ** (-torch.arange(n, device=t.device, dtype=torch.float64) / n)
        c, s = (f(a).to(wide)[:, None] for f in (torch.cos, torch.sin))
        u, v = t.to(wide).split(n, -1)
        return torch.cat([u * c - v * s, v * c + u * s], -1).to(dtype)

    h = x.to(dtype).to(wide)
    h = (h - h.mean(-1, keepdim=True)) * (h.var(-1, correction=0, keepdim=True) + eps).rsqrt()
    h = (h * p["norm.weight"].to(wide) + p["norm.bias"].to(wide)).to(dtype)
    cond = cond.to(dtype)
    q = turn((h @ p["q_proj"].to(dtype).T).unflatten(-1, (heads, d)), at)
    k = turn((cond @ p["k_proj"].to(dtype).T).unflatten(-1, (kv_heads, d)), cond_at)
    v = (cond @ p["v_proj"].to(dtype).T).unflatten(-1, (kv_heads, d))
    k, v = (t.repeat_interleave(heads // kv_heads, 2) for t in (k, v))
    s = torch.einsum("bshd,bkhd->bhsk", q.to(wide), k.to(wide)) / math.sqrt(d)
    s = s.masked_fill(torch.arange(cond.shape[1], device=x.device) >= lens[:, None, None, None], -math.inf)
    w = torch.softmax(s, -1).to(dtype)
    o = torch.einsum("bhsk,bkhd->bshd", w.to(wide), v.to(wide)).to(dtype).flatten(2)
    return o @ p["out_proj"].to(dtype).T


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim,tokens,keys", [(64, 70, 33), (128, 300, 129), (64, 1, 5)])
def test_layer_rounds_no_more_than_a_plain_one(cuda, dtype, head_dim, tokens, keys):
    torch.manual_seed(tokens)
    hidden, cond_dim, heads, kv_heads = 192, 160, 4, 2
    rope = ops.Rotary.build(head_dim, device=cuda)
    layer = block.TrainableCrossAttention(hidden, heads, head_dim, cond_dim, kv_heads=kv_heads, rope=rope,
                                          compute_dtype=dtype, device=cuda)
    layer.norm.weight.data.normal_(1.0, 0.2)
    layer.norm.bias.data.normal_(0.0, 0.2)
    x = torch.randn(3, tokens, hidden, device=cuda) + 0.5
    cond = torch.randn(3, keys, cond_dim, device=cuda)
    lens = torch.tensor([keys, keys // 2 + 1, 2], dtype=torch.int32, device=cuda)
    at, cond_at = torch.arange(tokens, device=cuda) + 7, torch.arange(keys, device=cuda)
    dy = torch.randn(3, tokens, hidden, device=cuda).to(dtype)

    x, cond = x.to(dtype), cond.to(dtype)
    y = layer(x, cond, cond_lens=lens, positions=at, cond_positions=cond_at)
    got = (y, *torch.autograd.grad(y, list(layer.parameters()), dy))
    got, others = [t.detach() for t in got], []
    for t in (torch.float64, dtype):
        p = {n: v.detach().to(torch.float64 if t == torch.float64 else torch.float32).requires_grad_()
             for n, v in layer.named_parameters()}
        z = layer_of(p, x, cond, lens, at, cond_at, heads, kv_heads, layer.norm.eps, t)
        others.append((z.detach(), *torch.autograd.grad(z, list(p.values()), dy.to(t))))
    names = ["result", *(n for n, _ in layer.named_parameters())]
    for name, g, w, plain in zip(names, got, *others):
        here, there = (float((t.double() - w).norm() / w.norm()) for t in (g, plain))
        assert here <= 2 * there, (name, here, there)
    assert y.dtype == dtype and _lib.device_status() == (0, 0, 0, 0)
