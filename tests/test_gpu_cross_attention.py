"""GPU: cross attention (forward, backward, autograd) against the formulas in
64 bits on the CPU.

Tolerance: |error| in the 2-norm over |result| of each output.  An output
is off by its own rounding, u = 2^-9 (bf16) or 2^-12 (f16) at most (the half
unit of an 8 or 11 bit significand, relative), and by the rounding of the
16-bit weights P (or dS) that enter the products, at most u more; scores,
sums and statistics are fp32 (2^-24, far below).  With few keys the gradients
also hold delta, rounded at most twice.  So 4 u bounds every output."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def formula(q, k, v, keep=None, scale=None, do=None):
    """fp64 on the CPU: o, lse and with do the gradients; keep bool [B, Skv]."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    b, s_q, h, d = q.shape
    g = h // k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    if keep is not None:
        k = torch.where(keep.cpu()[:, :, None, None], k, torch.zeros_like(k))
        v = torch.where(keep.cpu()[:, :, None, None], v, torch.zeros_like(v))
    kk, vv = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, kk) * scale
    if keep is not None:
        s = s.masked_fill(~keep.cpu()[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:-1], -math.inf, dtype=torch.float64)
    p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
    o = torch.einsum("bhij,bjhd->bihd", p, vv)
    if do is None:
        return o, lse
    do = do.detach().double().cpu()
    dp = torch.einsum("bihd,bjhd->bhij", do, vv)
    delta = (do * o).sum(-1).permute(0, 2, 1)
    ds = p * (dp - delta[..., None]) * scale
    dq = torch.einsum("bhij,bjhd->bihd", ds, kk)
    shape = (b, k.shape[1], k.shape[2], g, d)
    dk = torch.einsum("bhij,bihd->bjhd", ds, q).reshape(shape).sum(3)
    dv = torch.einsum("bhij,bihd->bjhd", p, do).reshape(shape).sum(3)
    return o, lse, dq, dk, dv


def check(got, want, dtype, name=""):
    want = want.to(got.device)
    assert got.dtype == dtype and got.shape == want.shape
    assert torch.isfinite(got).all(), name
    err, norm = (got.double() - want).norm().item(), want.norm().item()
    assert err <= 4 * UNIT[dtype] / 2 * norm + 1e-30, (name, err / max(norm, 1e-300))


def make(cuda, b, s_q, s_kv, h, hkv, d, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    q = torch.randn(b, s_q, h, d, generator=g, device=cuda).to(dtype)
    kv = torch.randn(b, s_kv, 2, hkv, d, generator=g, device=cuda).to(dtype)
    do = torch.randn(b, s_q, h, d, generator=g, device=cuda).to(dtype)
    return q, kv[:, :, 0], kv[:, :, 1], do


def run(cuda, shape, dtype, kv_lens=None, key_mask=None, scale=None, seed=0):
    from minixmax_h3_b200 import _lib, ops

    b, s_q, s_kv, h, hkv, d = shape
    q, k, v, do = make(cuda, b, s_q, s_kv, h, hkv, d, dtype, seed)
    keep = torch.ones(b, s_kv, dtype=torch.bool, device=cuda) if key_mask is None else key_mask
    if kv_lens is not None:
        keep = keep & (torch.arange(s_kv, device=cuda)[None] < kv_lens[:, None])
    # what is left out may hold anything
    k, v = (torch.where(keep[:, :, None, None], t, torch.full_like(t, math.nan)) for t in (k, v))
    lse = torch.empty(b, h, s_q, device=cuda)
    o = ops.cross_attention(q, k, v, kv_lens=kv_lens, key_mask=key_mask, scale=scale, lse=lse)
    grads = ops.cross_attention_bwd(do, q, k, v, o, lse, kv_lens=kv_lens, key_mask=key_mask, scale=scale)
    want = formula(q, k, v, keep, scale, do)
    check(o, want[0], dtype, "o")
    # fp32 log-sum-exp: 2^-24 relative of scores of some tens, and __log2f's 2^-22
    assert torch.allclose(lse.double().cpu(), want[1], atol=2e-5, rtol=2e-6)
    if s_kv > 1:
        for g, w, n in zip(grads, want[2:], ("dq", "dk", "dv")):
            check(g, w, dtype, n)
    else:  # one key: dS = P (dP - delta) is 0, and what is left is fp32 rounding of the two
        check(grads[2], want[4], dtype, "dv")
        assert max(grads[0].float().abs().max().item(), grads[1].float().abs().max().item()) < 1e-3 * max(s_q, 1)
    assert _lib.device_status() == (0, 0, 0, 0)
    return grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [
    # b, s_q, s_kv, heads, key heads, head dim: few rows (one kernel), many (another), tiles cut and whole
    (1, 1, 1, 1, 1, 128), (1, 1, 77, 3, 3, 128), (2, 1, 513, 4, 2, 64), (3, 5, 16, 8, 1, 128), (1, 17, 130, 4, 4, 64),
    (2, 63, 200, 2, 1, 128), (1, 64, 128, 2, 2, 128), (2, 65, 127, 4, 2, 64), (1, 128, 129, 2, 1, 128),
    (1, 129, 256, 3, 3, 64), (2, 257, 77, 2, 2, 128), (1, 300, 385, 6, 3, 128), (3, 130, 1, 2, 1, 64),
    (1, 1025, 640, 2, 1, 64)])
def test_forward_and_gradients(cuda, shape, dtype):
    run(cuda, shape, dtype, seed=sum(shape))


@pytest.mark.parametrize("s_q", [3, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_lengths_and_masks(cuda, s_q, d):
    """Lengths of 0 and 1, beyond the tensor, at and inside tiles; masks with
    holes and with nothing left; both together."""
    lens = torch.tensor([0, 1, 128, 129, 300, 77, 100000, 255], dtype=torch.int32, device=cuda)
    run(cuda, (8, s_q, 300, 4, 2, d), torch.bfloat16, kv_lens=lens)
    g = torch.Generator(device=cuda).manual_seed(3)
    mask = torch.rand(4, 300, generator=g, device=cuda) < 0.5
    mask[1] = False
    mask[2, :290] = False
    run(cuda, (4, s_q, 300, 4, 2, d), torch.float16, key_mask=mask)
    run(cuda, (4, s_q, 300, 4, 2, d), torch.bfloat16, key_mask=mask,
        kv_lens=torch.tensor([300, 300, 295, 12], dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("s_q", [2, 150])
def test_rows_without_keys(cuda, s_q):
    from minixmax_h3_b200 import ops

    q, k, v, do = make(cuda, 2, s_q, 50, 2, 2, 128, torch.bfloat16)
    lse = torch.empty(2, 2, s_q, device=cuda)
    lens = torch.zeros(2, dtype=torch.int32, device=cuda)
    k.fill_(math.nan), v.fill_(math.inf)
    o = ops.cross_attention(q, k, v, kv_lens=lens, lse=lse)
    assert (o == 0).all() and (lse == -math.inf).all()
    for g in ops.cross_attention_bwd(do, q, k, v, o, lse, kv_lens=lens):
        assert (g == 0).all()
    # no keys at all, no queries at all, no samples at all
    o = ops.cross_attention(q, k[:, :0], v[:, :0], lse=lse)
    assert (o == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = ops.cross_attention_bwd(do, q, k[:, :0], v[:, :0], o, lse)
    assert (dq == 0).all() and dk.shape == dv.shape == (2, 0, 2, 128)
    e = q[:, :0]
    assert ops.cross_attention(e, k, v).shape == e.shape
    dq, dk, dv = ops.cross_attention_bwd(e, e, k, v, e, torch.empty(2, 2, 0, device=cuda))
    assert dq.shape == e.shape and (dk == 0).all() and (dv == 0).all()
    assert ops.cross_attention(q[:0], k[:0], v[:0]).shape == (0, s_q, 2, 128)


@pytest.mark.parametrize("s_q", [4, 140])
def test_strides_offsets_and_out(cuda, s_q):
    """Heads-major and packed storage, offsets that are not 32-byte aligned,
    and layouts that have to be copied."""
    from minixmax_h3_b200 import ops

    g = torch.Generator(device=cuda).manual_seed(1)
    packed = torch.randn(2, 3, s_q, 3 * 128 + 8, generator=g, device=cuda).to(torch.bfloat16)
    q = packed[..., 8:].unflatten(-1, (3, 128))[:, 1]                       # stride 392, 16-byte aligned
    k = torch.randn(2, 3, 90, 128, generator=g, device=cuda).to(torch.bfloat16).transpose(1, 2)  # heads first
    v = torch.randn(2, 3, 90, 128, generator=g, device=cuda).to(torch.bfloat16).transpose(1, 2)
    want = formula(q, k, v)[0]
    check(ops.cross_attention(q, k, v), want, torch.bfloat16)
    out = torch.zeros(2, s_q, 3 * 128 + 8, dtype=torch.bfloat16, device=cuda)
    view = out[..., 8:].unflatten(-1, (3, 128))
    assert ops.cross_attention(q, k, v, out=view) is view
    check(view, want, torch.bfloat16)
    assert (out[..., :8] == 0).all()
    odd = torch.randn(2, s_q, 3, 131, generator=g, device=cuda).to(torch.bfloat16)[..., 3:]  # copied
    check(ops.cross_attention(odd, k, v), formula(odd, k, v)[0], torch.bfloat16)
    shared = k[:1].expand(2, -1, -1, -1)                                    # one sample's states for the batch
    check(ops.cross_attention(q, shared, v), formula(q, shared, v)[0], torch.bfloat16)


@pytest.mark.parametrize("s_q", [7, 200])
def test_large_scores_and_scale(cuda, s_q):
    """Scores of several hundreds, growing along the keys: the running
    maximum moves, and most weights vanish."""
    from minixmax_h3_b200 import ops

    g = torch.Generator(device=cuda).manual_seed(2)
    q = (4 * torch.randn(1, s_q, 2, 128, generator=g, device=cuda)).to(torch.bfloat16)
    ramp = torch.linspace(0.1, 4, 700, device=cuda)[None, :, None, None]
    k = (ramp * torch.randn(1, 700, 2, 128, generator=g, device=cuda)).to(torch.bfloat16)
    v = torch.randn(1, 700, 2, 128, generator=g, device=cuda).to(torch.bfloat16)
    for scale in (0.5, 0.02):
        check(ops.cross_attention(q, k, v, scale=scale), formula(q, k, v, scale=scale)[0], torch.bfloat16)


def test_autograd_and_broadcast_states(cuda):
    """Gradients through autograd, of states shared by the batch (expand) and
    of heads that share a key head; the same bits each time."""
    from minixmax_h3_b200.attention import cross_attention

    q, k, v, do = make(cuda, 3, 140, 90, 4, 2, 64, torch.bfloat16, seed=9)
    q = q.requires_grad_()
    k1, v1 = k[:1].contiguous().requires_grad_(), v[:1].contiguous().requires_grad_()
    lens = torch.tensor([90, 33, 64], dtype=torch.int32, device=cuda)
    grads = []
    for _ in range(2):
        o = cross_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), kv_lens=lens)
        grads.append(torch.autograd.grad(o, (q, k1, v1), do))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    keep = torch.arange(90, device=cuda)[None] < lens[:, None]
    want = formula(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), keep, None, do)
    check(grads[0][0], want[2], torch.bfloat16, "dq")
    for got, w in zip(grads[0][1:], want[3:]):  # the batch's sum: three rounded gradients and their sum's rounding
        w = w.sum(0, keepdim=True).to(cuda)
        assert (got.double() - w).norm() <= 6 * UNIT[torch.bfloat16] / 2 * w.norm()


def test_gradients_against_differences(cuda):
    """<grad, direction> against (f(x + h u) - f(x - h u)) / 2h of the fp64
    formula, whose second-order error is below 1e-6 of it at h = 1e-4."""
    from minixmax_h3_b200 import ops

    q, k, v, do = make(cuda, 1, 70, 40, 2, 1, 64, torch.float16, seed=4)
    lse = torch.empty(1, 2, 70, device=cuda)
    o = ops.cross_attention(q, k, v, lse=lse)
    grads = ops.cross_attention_bwd(do, q, k, v, o, lse)
    f = lambda *x: (formula(*x)[0] * do.double().cpu()).sum().item()  # noqa: E731
    g = torch.Generator().manual_seed(0)
    base = [t.double().cpu() for t in (q, k, v)]
    for i in range(3):
        u = grads[i].double().cpu() / grads[i].double().norm().item() + 0.01 * torch.randn(base[i].shape, generator=g)
        h = 1e-4
        up, down = ([x + s * h * u if j == i else x for j, x in enumerate(base)] for s in (1, -1))
        slope = (f(*up) - f(*down)) / (2 * h)
        got = (grads[i].double().cpu() * u).sum().item()
        assert abs(got - slope) <= 4 * UNIT[torch.float16] / 2 * grads[i].double().norm().item() * u.norm().item()


def test_other_stream(cuda):
    from minixmax_h3_b200 import ops

    q, k, v, _ = make(cuda, 1, 300, 200, 2, 2, 128, torch.bfloat16)
    want = ops.cross_attention(q, k, v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.cross_attention(q, k, v) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, want) for g in got)


def test_many_units(cuda):
    """More work units than SMs, ragged, with empty samples between: every
    role of the persistent kernels passes from unit to unit."""
    lens = torch.tensor([200, 0, 513, 1, 0, 640], dtype=torch.int32, device=cuda)
    run(cuda, (6, 1300, 640, 8, 4, 64), torch.float16, kv_lens=lens)
    run(cuda, (6, 700, 640, 8, 8, 128), torch.bfloat16, kv_lens=lens)


def test_custom_operator(cuda):
    import minixmax_h3_b200.torch_ops  # noqa: F401
    from minixmax_h3_b200 import ops

    q, k, v, do = make(cuda, 2, 80, 60, 2, 2, 64, torch.bfloat16)
    q, k, v = (t.contiguous().requires_grad_() for t in (q, k, v))
    o, lse = torch.ops.h3b.cross_attention(q, k, v, None, None, None)
    got = torch.autograd.grad(o, (q, k, v), do)
    lse2 = torch.empty_like(lse)
    with torch.no_grad():
        o2 = ops.cross_attention(q, k, v, lse=lse2)
        want = ops.cross_attention_bwd(do, q, k, v, o2, lse2)
    assert torch.equal(o, o2) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_cross_attention_layer(cuda):
    """block.CrossAttention against its projections and the formula, dense and
    through the cache (whose values the formula is given)."""
    from minixmax_h3_b200 import ops
    from minixmax_h3_b200.block import CrossAttention, load_quant_linear

    g = torch.Generator(device=cuda).manual_seed(0)
    layer = CrossAttention(256, 4, 64, 512, kv_heads=2, device=cuda)
    for ql in (layer.q_proj, layer.kv_proj, layer.out_proj):
        load_quant_linear(ql, torch.randn(ql.out_features, ql.in_features, generator=g, device=cuda) * 0.05,
                          "int8_tensorwise")
    x = torch.randn(2, 70, 256, generator=g, device=cuda).to(torch.bfloat16)
    cond = torch.randn(2, 50, 512, generator=g, device=cuda).to(torch.bfloat16)
    lens = torch.tensor([50, 21], dtype=torch.int32, device=cuda)
    keep = torch.arange(50, device=cuda)[None] < lens[:, None]
    q = layer.q_proj(x.view(140, 256)).view(2, 70, 4, 64)
    k, v = layer.encode(cond)
    mid = formula(q, k, v, keep)[0].to(cuda, torch.bfloat16)
    want = layer.out_proj(mid.reshape(140, 256)).view(2, 70, 256)
    got = layer(x, cond, cond_lens=lens)
    # the attention's 4u, through an 8-bit quantiser (steps of 1/127 of a row's largest value) and a sum over 256
    assert (got - want).float().norm() <= 0.02 * want.float().norm()
    assert torch.equal(got, layer(x, kv=(k, v), cond_lens=lens))
    cache = ops.KV8Cache.empty(2, 2, 64, device=cuda)
    table = torch.tensor([[1], [0]], dtype=torch.int32, device=cuda)
    layer.fill(cache, cond, table, torch.zeros_like(lens), new_lens=lens)
    got = layer(x, cache=cache, block_table=table, cond_lens=lens)
    k8, v8 = ops.kv8_read(cache, table, lens, 50, dtype=torch.float32)
    mid = formula(q, k8, v8, keep)[0].to(cuda, torch.bfloat16)
    want = layer.out_proj(mid.reshape(140, 256)).view(2, 70, 256)
    assert (got - want).float().norm() <= 0.02 * want.float().norm()
    with pytest.raises(ValueError):
        layer(x)


def test_no_second_derivatives(cuda):
    """A gradient penalty must not silently lose this operator's part."""
    from minixmax_h3_b200.attention import cross_attention

    q, k, v, do = make(cuda, 1, 9, 12, 2, 2, 64, torch.bfloat16)
    q = q.requires_grad_()
    (dq,) = torch.autograd.grad(cross_attention(q, k, v), q, do, create_graph=True)
    with pytest.raises(RuntimeError):
        (dq.float().square().sum() + q.float().sum()).backward()
