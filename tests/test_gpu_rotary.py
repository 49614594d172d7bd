"""GPU: rotary positions against their definition in 64 bits.

Tolerance: a result is fp32 arithmetic rounded once.  Half a step of the type
(eps / 2 relative; 2^-25 absolute in fp16's subnormal range), and in fp32: sine
and cosine (2 ulp of sincospif, 2^-24 of its argument, 2^-24 of the factor's
product) and the product and sum (2^-24 each) - within 8 * 2^-24 of
factor * (|x1| + |x2|)."""
from __future__ import annotations

import math

import pytest
import torch

from minixmax_h3_b200 import _lib, attention, ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
PI = 3141592653589793238462643383279502884197169399375105820974945  # over 10^60


def angles(rope: ops.Rotary, w: list[float], positions: torch.Tensor) -> torch.Tensor:
    """[B, S, pairs] radians within a turn, whole turns taken off in integers."""
    p = positions.cpu()
    p = p[..., None] if len(rope.sections) == 1 else p
    axis = [a for a, n in enumerate(rope.sections) for _ in range(n)]
    two_pi = 2 * PI
    out = torch.empty(*p.shape[:-1], len(w), dtype=torch.float64)
    flat, src = out.flatten(0, -2), p.reshape(-1, p.shape[-1]).tolist()
    for r, row in enumerate(src):
        for i, f in enumerate(w):
            num, den = f.as_integer_ratio()
            # radians of the position, as a remainder by 2 pi over the common denominator
            rest = (row[axis[i]] * num * 10 ** 60) % (two_pi * den)
            flat[r, i] = rest / (10 ** 60 * den)
    return out


def turned(x: torch.Tensor, angle: torch.Tensor, rope: ops.Rotary, inverse: bool):
    """(result, sum of the pair's sizes) in 64 bits; angle [B or 1, S, pairs]."""
    x = x.double().cpu()
    n = angle.shape[-1]
    a = (-angle if inverse else angle)[:, :, None]
    one, two = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if rope.interleaved else (x[..., :n], x[..., n:2 * n])
    r1 = rope.factor * (one * a.cos() - two * a.sin())
    r2 = rope.factor * (two * a.cos() + one * a.sin())
    size = abs(rope.factor) * (one.abs() + two.abs())
    y, s = x.clone(), torch.zeros_like(x)
    for dst, v1, v2 in ((y, r1, r2), (s, size, size)):
        if rope.interleaved:
            dst[..., 0:2 * n:2], dst[..., 1:2 * n:2] = v1, v2
        else:
            dst[..., :n], dst[..., n:2 * n] = v1, v2
    return y, s


def close(got, want, size):
    eps = torch.finfo(got.dtype).eps
    bound = want.abs() * eps / 2 * 1.001 + 8 * 2.0 ** -24 * size
    if got.dtype == torch.float16:
        bound += 2.0 ** -25
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (off - bound).max().item()


def frequencies(dims, theta=10000.0):
    return [theta ** (-2 * i / d) for d in dims for i in range(d // 2)]


CASES = [  # b, s, h, hkv, d, dims, interleaved
    (1, 1, 24, 24, 128, (128,), False),
    (3, 37, 4, 2, 64, (32,), True),
    (2, 65, 3, 1, 80, (20,), False),       # ten pairs: vectors of two
    (2, 5, 2, 2, 96, (24,), True),
    (1, 130, 1, 1, 256, (256,), False),
    (2, 33, 5, 5, 128, (44, 42, 42), False),
    (1, 9, 2, 1, 10, (6,), True),          # nothing aligned
    (1, 9, 2, 1, 6, (2,), False),
    (2, 4, 2, 1, 64, (0,), False),         # nothing turned
    (1, 3, 40, 7, 64, (0, 16, 8), True),   # an empty section
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,h,hkv,d,dims,interleaved", CASES)
def test_rotary(cuda, dtype, b, s, h, hkv, d, dims, interleaved):
    g = torch.Generator(device=cuda).manual_seed(5)
    qkv = torch.randn(b, s, h + 2 * hkv, d, generator=g, device=cuda).to(dtype)
    q, k = qkv[:, :, :h], qkv[:, :, h:h + hkv]
    w = frequencies(dims)
    rope = ops.Rotary.from_frequencies(w, sections=[n // 2 for n in dims], interleaved=interleaved, factor=1.25)
    shape = (b, s) if len(dims) == 1 else (b, s, len(dims))
    p = torch.randint(-1000, 300000, shape, generator=g, device=cuda, dtype=torch.int32)
    angle = angles(rope, w, p)
    for inverse in (False, True):
        for got, x in zip(ops.rotary(q, k, p, rope, inverse=inverse), (q, k)):
            assert got.is_contiguous() and got.dtype == dtype
            close(got, *turned(x, angle, rope, inverse))
    # in place, and positions in 64 bits: the same bits
    want = ops.rotary(q, k, p, rope)
    ops.rotary(q, k, p.long(), rope, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    # k alone, as q
    assert ops.rotary(q, None, p, rope)[1] is None
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.parametrize("at", [0, 1, -1, 10 ** 6, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345])
def test_far_positions(cuda, at):
    """Exact whole turns at any position; a 32-bit angle would be noise there."""
    w = frequencies((64,)) + [3.0, -0.7, 1e-9, 6.5]
    rope = ops.Rotary.from_frequencies(w)
    x = torch.randn(1, 2, 1, 2 * len(w), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    p = torch.tensor([[at, at - 3]], dtype=torch.int64, device=cuda)
    y, size = turned(x, angles(rope, w, p), rope, False)
    got = ops.rotary(x, None, p, rope)[0]
    # a frequency is held to 2^-65 turns (the last bit of a turn's fraction): times the position, in radians
    off = (got.double().cpu() - y).abs()
    assert (off <= y.abs() * 2.0 ** -24 + size * (8 * 2.0 ** -24 + abs(at) * 2 * math.pi * 2.0 ** -64)).all()


def test_strides_and_shared_positions(cuda):
    g = torch.Generator(device=cuda).manual_seed(2)
    rope = ops.Rotary.build(64)
    w = frequencies((64,))
    p = torch.arange(50, device=cuda, dtype=torch.int32)
    angle = angles(rope, w, p[None])
    heads_first = torch.randn(2, 3, 50, 64, generator=g, device=cuda).bfloat16().transpose(1, 2)
    odd = torch.randn(2, 50, 3, 65, generator=g, device=cuda).bfloat16()[..., 1:]     # not aligned
    last = torch.randn(2, 50, 64, 3, generator=g, device=cuda).bfloat16().transpose(2, 3)  # no unit stride: copied
    spread = torch.randn(2, 1, 3, 64, generator=g, device=cuda).bfloat16().expand(2, 50, 3, 64)
    for x in (heads_first, odd, last, spread):
        close(ops.rotary(x, None, p, rope)[0], *turned(x, angle, rope, False))
        close(ops.rotary(heads_first, x, p, rope)[1], *turned(x, angle, rope, False))
    # positions with strides: every other one, and one column of a wider table
    table = torch.arange(4 * 100, device=cuda, dtype=torch.int64).view(2, 2, 100)
    sel = table[:, 1, ::2]
    close(ops.rotary(odd, None, sel, rope)[0], *turned(odd, angles(rope, w, sel), rope, False))
    # outputs inside a larger buffer: nothing beside them is written
    buf = torch.full((2, 50, 5, 96), 7.0, device=cuda, dtype=torch.bfloat16)
    out = buf[:, :, 1:4, 16:80]
    ops.rotary(odd, None, p, rope, q_out=out)
    assert torch.equal(out, ops.rotary(odd, None, p, rope)[0])
    buf[:, :, 1:4, 16:80] = 7.0
    assert (buf == 7.0).all()


def test_empty_and_non_finite(cuda):
    rope = ops.Rotary.build(64)
    e = torch.empty(2, 0, 4, 64, device=cuda)
    assert ops.rotary(e, e[:, :, :1], torch.empty(0, dtype=torch.int32, device=cuda), rope)[1].shape == (2, 0, 1, 64)
    none = torch.empty(1, 3, 0, 64, device=cuda)
    p = torch.arange(3, device=cuda)
    x = torch.randn(1, 3, 2, 64, device=cuda)
    got = ops.rotary(none, x, p, rope)
    assert got[0].shape == none.shape and torch.equal(got[1], ops.rotary(x, None, p, rope)[0])
    x[0, 1, 0, 3] = float("nan")
    y = ops.rotary(x, None, p, rope)[0]
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 1, 0, [3, 35]] = True  # the pair, and nothing else
    assert torch.equal(y.isnan(), bad)


def test_gradients(cuda):
    g = torch.Generator(device=cuda).manual_seed(3)
    rope = ops.Rotary.build((24, 20, 20), factor=1.5)
    p = torch.randint(0, 500, (2, 11, 3), generator=g, device=cuda)
    q = torch.randn(2, 11, 4, 96, generator=g, device=cuda).requires_grad_()
    k = torch.randn(2, 11, 2, 96, generator=g, device=cuda).requires_grad_()
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    oq, ok = attention.rotary(q, k, p, rope)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk), create_graph=True)
    # <R q, gq> = <q, R^T gq>, to the rounding of both sides
    for x, o, do, dx in ((q, oq, gq, dq), (k, ok, gk, dk)):
        a, b = (o.double() * do).sum(), (x.double() * dx).sum()
        assert (a - b).abs() <= 20 * 2.0 ** -24 * (x.abs().double() * do.abs().double()).sum() * 3
    # differences: the map is linear, so a step of any size gives the derivative
    step = torch.randn_like(q)
    with torch.no_grad():
        moved = attention.rotary(q + step, None, p, rope)[0]
    lhs, rhs = ((moved.double() - oq) * gq).sum(), (step.double() * dq).sum()
    assert (lhs - rhs).abs() <= 40 * 2.0 ** -24 * ((q.abs() + step.abs()).double() * gq.abs()).sum() * 3
    # the gradient's gradient is the rotation again
    v = gq.clone().requires_grad_()
    first, = torch.autograd.grad(attention.rotary(q, None, p, rope)[0], q, v, create_graph=True)
    u = torch.randn_like(q)
    second, = torch.autograd.grad(first, v, u)
    assert torch.equal(second, ops.rotary(u, None, p, rope)[0])
    # one of the results used, q without a gradient
    only, = torch.autograd.grad(attention.rotary(q.detach(), k, p, rope)[1].sum(), k)
    assert torch.equal(only, ops.rotary(torch.ones_like(k), None, p, rope, inverse=True)[0])


def test_graph_and_streams(cuda):
    """Captured and replayed with other positions; two streams at once."""
    rope = ops.Rotary.build(128)
    x = torch.randn(4, 1, 24, 128, device=cuda).bfloat16()
    p = torch.tensor([[3], [70], [0], [9000]], dtype=torch.int32, device=cuda)
    ops.rotary(x, x, p, rope)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rotary(x, x, p, rope)
    for _ in range(3):
        p += 1
        graph.replay()
        assert torch.equal(got[0], ops.rotary(x, None, p, rope)[0]) and torch.equal(got[0], got[1])
    want = ops.rotary(x, None, p, rope)[0]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append(ops.rotary(x, None, p, rope)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_offsets_past_32_bits(cuda):
    """A tensor of more than 2^31 elements: its last tokens."""
    s, h, d = 2 ** 31 // (32 * 128) + 5, 32, 128
    x = torch.zeros(1, s, h, d, dtype=torch.bfloat16, device=cuda)
    tail = torch.randn(1, 3, h, d, device=cuda).bfloat16()
    x[:, -3:] = tail
    rope = ops.Rotary.build(d)
    p = torch.arange(s, device=cuda, dtype=torch.int32)
    ops.rotary(x, None, p, rope, q_out=x)
    assert torch.equal(x[:, -3:], ops.rotary(tail, None, p[-3:], rope)[0])
    assert not x[:, :-3].any()


def test_refusals(cuda):
    rope = ops.Rotary.build(64)
    x = torch.zeros(2, 3, 4, 64, device=cuda)
    p = torch.zeros(3, dtype=torch.int32, device=cuda)
    ops.rotary(x, x, p, rope)
    for error, args, kw in (
            (RuntimeError, (x.cpu(), None, p, rope), {}),
            (RuntimeError, (x, None, p.cpu(), rope), {}),
            (TypeError, (x.double(), None, p, rope), {}),
            (TypeError, (x, x.half(), p, rope), {}),
            (ValueError, (x, x[:, :2], p, rope), {}),
            (ValueError, (x[0], None, p, rope), {}),
            (TypeError, (x, None, p.float(), rope), {}),
            (ValueError, (x, None, p[:2], rope), {}),
            (ValueError, (x, None, torch.zeros(2, 3, 1, dtype=torch.int32, device=cuda), rope), {}),
            (ValueError, (x[..., :32], None, p, rope), {}),
            (ValueError, (torch.zeros(2, 3, 4, 65, device=cuda), None, p, rope), {}),
            (ValueError, (x, None, p, rope), {"q_out": x[..., :32]}),
            (ValueError, (x, None, p, rope), {"q_out": torch.zeros(2, 3, 64, 4, device=cuda).transpose(2, 3)}),
            (ValueError, (x, x, p, rope), {"k_out": x.half()}),
            (ValueError, (x, None, p, rope), {"q_out": x[:, :, :1].expand(2, 3, 4, 64)})):
        with pytest.raises(error):
            ops.rotary(*args, **kw)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises(NotImplementedError):
            attention.rotary(dual, None, p, rope)
