"""GPU: layer norm, rotary positions, cross attention and Muon together, as a
conditioned layer is trained and then used."""
from __future__ import annotations

import math

import pytest
import torch

from minixmax_h3_b200 import _lib, block, ops, optim
from minixmax_h3_b200 import torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def layer_and_inputs(cuda, head_dim=64, seed=0, dtype=BF16, hidden=192, cond_dim=160):
    torch.manual_seed(seed)
    rope = ops.Rotary.build(head_dim // 2, interleaved=True, device=cuda)
    layer = block.TrainableCrossAttention(hidden, 4, head_dim, cond_dim, kv_heads=2, rope=rope, compute_dtype=dtype, device=cuda)
    x, cond = torch.randn(2, 70, hidden, device=cuda), torch.randn(2, 33, cond_dim, device=cuda)
    where = {"cond_lens": torch.tensor([33, 20], dtype=torch.int32, device=cuda),
             "positions": torch.arange(70, device=cuda), "cond_positions": torch.arange(33, device=cuda) + 5}
    return layer, x, cond, where


def reference(layer, x, cond, where):
    """The layer in 64 bits, from parameters that require gradients; and the largest score."""
    p = {n: t.detach().double().requires_grad_() for n, t in layer.named_parameters()}
    h = (x - x.mean(-1, keepdim=True)) / (x.var(-1, correction=0, keepdim=True) + layer.norm.eps).sqrt()
    h = h * p["norm.weight"] + p["norm.bias"]
    d, hkv = layer.head_dim, layer.kv_heads

    def turn(t, at):
        n = d // 4
        a = at.double()[:, None] * torch.tensor([10000.0 ** (-2 * i / (2 * n)) for i in range(n)], dtype=torch.float64,
                                                device=t.device)
        z = torch.view_as_complex(t[..., :2 * n].unflatten(-1, (n, 2)).contiguous())
        z = torch.view_as_real(z * torch.polar(torch.ones_like(a), a)[None, :, None]).flatten(-2)
        return torch.cat([z, t[..., 2 * n:]], -1)

    q = turn((h @ p["q_proj"].T).unflatten(-1, (-1, d)), where["positions"])
    k = turn((cond @ p["k_proj"].T).unflatten(-1, (-1, d)), where["cond_positions"])
    v = (cond @ p["v_proj"].T).unflatten(-1, (-1, d))
    q = q.unflatten(2, (hkv, -1))
    s = torch.einsum("bsgnd,bkgd->bgnsk", q, k) / math.sqrt(d)
    s = s.masked_fill(torch.arange(cond.shape[1], device=x.device) >= where["cond_lens"][:, None, None, None, None], -math.inf)
    o = torch.einsum("bgnsk,bkgd->bsgnd", torch.softmax(s, -1), v).flatten(2)
    return o @ p["out_proj"].T, p, float(s.detach()[s > -math.inf].abs().max())


@pytest.mark.parametrize("dtype,head_dim", [(BF16, 64), (torch.float16, 128)])
def test_layer_against_64_bits(cuda, dtype, head_dim):
    """Output and gradients, in Frobenius norms.  A product's operands and its
    result are rounded (u = eps / 2 each in norm): h, w, q, rotated q, likewise k,
    the weights p, v, o, the output's weight and the result - 14 roundings - and a
    score is off by 8 u of its largest value, which moves p by as much.  Backward
    the same once more, for values and for gradients: twice that."""
    layer, x, cond, where = layer_and_inputs(cuda, head_dim, dtype=dtype)
    y = layer(x, cond, **where)
    dy = torch.randn_like(y)
    grads = torch.autograd.grad(y, list(layer.parameters()), dy)
    want, p, top = reference(layer, x.to(dtype).double(), cond.to(dtype).double(), where)
    wanted = torch.autograd.grad(want, list(p.values()), dy.double())
    u = torch.finfo(dtype).eps / 2
    off = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert y.dtype == dtype and off(y, want) <= (14 + 8 * top) * u
    for (name, _), got, w in zip(layer.named_parameters(), grads, wanted):
        assert off(got, w) <= 2 * (14 + 8 * top) * u, name
    assert _lib.device_status() == (0, 0, 0, 0)


def test_layer_is_its_parts(cuda):
    """The same bits as the operators called one by one, forward and backward."""
    layer, x, cond, where = layer_and_inputs(cuda)
    y = layer(x, cond, **where)
    dy = torch.randn_like(y)
    got = dict(zip((n for n, _ in layer.named_parameters()), torch.autograd.grad(y, list(layer.parameters()), dy)))
    w = {n: t.detach().to(BF16) for n, t in layer.named_parameters() if "norm" not in n}
    xb, cb = x.to(BF16), cond.to(BF16)
    stats = torch.empty(2, 140, device=cuda)
    h = ops.layer_norm(xb, layer.norm.weight, layer.norm.bias, layer.norm.eps, stats=stats)
    q0, k0, v = ((t @ w[n].T).unflatten(-1, (-1, 64)) for t, n in ((h, "q_proj"), (cb, "k_proj"), (cb, "v_proj")))
    q = ops.rotary(q0, None, where["positions"], layer.rope)[0]
    k = ops.rotary(k0, None, where["cond_positions"], layer.rope)[0]
    lse = torch.empty(2, 4, 70, device=cuda)
    o = ops.cross_attention(q, k, v, kv_lens=where["cond_lens"], lse=lse)
    assert torch.equal(y, o.flatten(2) @ w["out_proj"].T)
    do = (dy @ w["out_proj"]).unflatten(-1, (4, 64))
    dq, dk, dv = ops.cross_attention_bwd(do, q, k, v, o, lse, kv_lens=where["cond_lens"])
    dq = ops.rotary(dq, None, where["positions"], layer.rope, inverse=True)[0].flatten(2)
    dk = ops.rotary(dk, None, where["cond_positions"], layer.rope, inverse=True)[0].flatten(2)
    want = {"out_proj": dy.flatten(0, 1).T @ o.flatten(2).flatten(0, 1), "q_proj": dq.flatten(0, 1).T @ h.flatten(0, 1),
            "k_proj": dk.flatten(0, 1).T @ cb.flatten(0, 1), "v_proj": dv.flatten(2).flatten(0, 1).T @ cb.flatten(0, 1)}
    _, want["norm.weight"], want["norm.bias"] = ops.layer_norm_bwd(dq @ w["q_proj"], xb, stats, layer.norm.weight)
    for n, g in got.items():
        assert torch.equal(g, want[n].float()), n


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_muon_moves_the_layer(cuda, dtype):
    """A step of Muon is ops.orthogonalize of the averages, one call a shape; a captured step the same bits."""
    layer, x, cond, where = layer_and_inputs(cuda)
    before = [p.detach().clone() for p in layer.matrices()]
    opt = optim.Muon(layer.matrices(), lr=0.03, momentum=0.8, weight_decay=0.1, dtype=dtype)
    launches = _lib.LAUNCHES[0]
    (layer(x, cond, **where).float() ** 2).mean().backward()
    launches = _lib.LAUNCHES[0]
    opt.step()
    assert _lib.LAUNCHES[0] - launches == 3  # q and out of two shapes, k and v of one
    for p, old in zip(layer.matrices(), before):
        average = torch.lerp(torch.zeros_like(p.grad), p.grad, 0.2)
        u = ops.orthogonalize(torch.lerp(p.grad, average, 0.8).to(dtype)[None])[0].float()
        m, n = p.shape
        want = (old * (1 - 0.03 * 0.1)).add(u, alpha=-0.03 * max(1.0, m / n) ** 0.5)
        assert torch.equal(p.detach(), want)
    # captured: the parameters' gradients are the graph's inputs
    grads = [torch.randn_like(p) for p in layer.matrices()]
    for p, g in zip(layer.matrices(), grads):
        p.grad = g
    twin = [p.detach().clone().requires_grad_() for p in layer.matrices()]
    other = optim.Muon(twin, lr=0.03, momentum=0.8, weight_decay=0.1, dtype=dtype)
    for p, q, g in zip(layer.matrices(), twin, grads):
        q.grad = g
        other.state[q]["average"] = opt.state[p]["average"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(2):
        graph.replay()
        other.step()
        assert all(torch.equal(p, q) for p, q in zip(layer.matrices(), twin))
        for g in grads:
            g.mul_(-0.5)


def test_captured_training_step(cuda):
    """Forward and backward through autograd, captured and replayed on other inputs."""
    layer, x, cond, where = layer_and_inputs(cuda)
    params, dy = list(layer.parameters()), torch.randn(2, 70, 192, device=cuda).to(BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(layer(x, cond, **where), params, dy)  # its results are gone before the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, cond, **where)
        grads = torch.autograd.grad(y, params, dy)
    for _ in range(2):
        x.normal_()
        cond.normal_()
        graph.replay()
        want = layer(x, cond, **where)
        wanted = torch.autograd.grad(want, params, dy)
        assert torch.equal(y, want) and all(torch.equal(g, w) for g, w in zip(grads, wanted))


def test_quantized_layer(cuda):
    """The layer for inference is its parts: norm, quantised projections, rotations, attention - dense, with keys
    encoded once, and through the 8-bit cache, chunk and single token."""
    # (the int8 products take K in multiples of 128)
    layer, x, cond, where = layer_and_inputs(cuda, 128, hidden=256, cond_dim=384)
    q8 = layer.quantized()
    x, cond = x.to(BF16), cond.to(BF16)
    assert torch.equal(q8.norm.weight, layer.norm.weight) and q8.rope is layer.rope
    h = ops.layer_norm(x, layer.norm.weight, layer.norm.bias, layer.norm.eps)
    q = ops.rotary(q8.q_proj(h.view(140, 256)).view(2, 70, 4, 128), None, where["positions"], layer.rope)[0]
    kv = q8.kv_proj(cond.view(66, 384)).view(2, 33, 2, 2, 128)
    k, v = ops.rotary(kv[:, :, 0], None, where["cond_positions"], layer.rope)[0], kv[:, :, 1]
    o = ops.cross_attention(q, k, v.contiguous(), kv_lens=where["cond_lens"])
    want = q8.out_proj(o.view(140, 512)).view(2, 70, 256)
    assert torch.equal(q8(x, cond, **where), want)
    kept = q8.encode(cond, cond_positions=where["cond_positions"])
    assert torch.equal(kept[0], k) and torch.equal(kept[1], v)
    assert torch.equal(q8(x, kv=kept, cond_lens=where["cond_lens"], positions=where["positions"]), want)
    cache = ops.KV8Cache.empty(2, 2, 128, device=cuda)
    table = torch.tensor([[1], [0]], dtype=torch.int32, device=cuda)
    q8.fill(cache, cond, table, torch.zeros(2, dtype=torch.int32, device=cuda), new_lens=where["cond_lens"],
            cond_positions=where["cond_positions"])
    for s in (slice(0, 70), slice(69, 70)):
        got = q8(x[:, s], cache=cache, block_table=table, cond_lens=where["cond_lens"], positions=where["positions"][s])
        o = ops.kv8_attention(q[:, s], cache, table, where["cond_lens"])
        n = o.shape[1]
        assert torch.equal(got, q8.out_proj(o.reshape(2 * n, 512)).view(2, n, 256))
    # what training needs still raises
    with pytest.raises(RuntimeError):
        q8(x.requires_grad_(), cond, **where)


def test_custom_operators(cuda):
    """torch.ops.h3b.*: the same bits as ops, and their gradients."""
    x = torch.randn(2, 9, 3, 64, device=cuda, requires_grad=True)
    p = torch.arange(9, device=cuda)
    rope = ops.Rotary.build(32, factor=1.5, device=cuda)
    y = torch.ops.h3b.rotary(x, p, rope.turns, list(rope.sections), False, rope.factor, False)
    assert torch.equal(y, ops.rotary(x, None, p, rope)[0])
    g = torch.randn_like(y).requires_grad_()
    dx, = torch.autograd.grad(y, x, g, create_graph=True)
    assert torch.equal(dx, ops.rotary(g, None, p, rope, inverse=True)[0])
    u = torch.randn_like(dx)
    assert torch.equal(torch.autograd.grad(dx, g, u)[0], ops.rotary(u, None, p, rope)[0])
    w, b = torch.randn(64, device=cuda, requires_grad=True), torch.randn(64, device=cuda, requires_grad=True)
    y, stats = torch.ops.h3b.layer_norm(x, w, b, 1e-5)
    assert torch.equal(y, ops.layer_norm(x, w, b))
    got = torch.autograd.grad(y, (x, w, b), g.detach())
    assert all(torch.equal(s, t) for s, t in zip(got, ops.layer_norm_bwd(g.detach(), x.detach(), stats.detach(), w.detach())))
    y, stats = torch.ops.h3b.layer_norm(x, None, None, 1e-5)
    got, = torch.autograd.grad(y, x, g.detach())
    assert torch.equal(got, ops.layer_norm_bwd(g.detach(), x.detach(), stats)[0])
    with pytest.raises(RuntimeError, match="stats"):
        torch.ops.h3b.layer_norm(x, w, b, 1e-5)[1].sum().backward()
    m = torch.randn(2, 30, 50, device=cuda)
    assert torch.equal(torch.ops.h3b.orthogonalize(m, 4, 1.5, -0.5, 0.0, 1e-7),
                       ops.orthogonalize(m, steps=4, coefficients=(1.5, -0.5, 0.0)))
