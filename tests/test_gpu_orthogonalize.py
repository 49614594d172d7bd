"""GPU: orthogonalised updates against the formula in 64 bits.

Tolerance, in Frobenius norms (|.|) and spectral ones (s).  With u the relative
rounding of an operand (2^-22 in pairs of planes, 2^-12 in one), v = 2^-24 (40 +
K / 32) that of a sum over K (24 additions of 16 elements within an accumulator,
cut, not rounded; one addition for each 128 after), t = 1.2 at most what is
added to G's diagonal (r rows), a step is off by

  dG = (2 u + v) s |X| + u (|G| + t sqrt(r))
  dB = (|b| + 2 |c| (s^2 + t)) dG + |c| (2 u + v) (s^2 + t) (|G| + t sqrt(r)) + (u + v) (|B| + 8 sqrt(r))
  dX = s dB + (2 u + v) s(B) |X| + u |X'|

(8: the constants that the completed square takes off again), and what a step
starts with grows by max |p'| over the singular values, p(x) = a x + b x^3 +
c x^5, at most.  The result is rounded once more: half a step of its type."""
from __future__ import annotations

import math

import pytest
import torch

from minixmax_h3_b200 import _lib, ops

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEFAULT = (3.4445, -4.7750, 2.0315)


def formula(x, steps, co, eps, dtype):
    """The result of one matrix in 64 bits, and the tolerance."""
    a, b, c = co
    x = x.double()
    if x.shape[0] > x.shape[1]:
        y, off = formula(x.T, steps, co, eps, dtype)
        return y.T, off
    x = x / (torch.linalg.matrix_norm(x) + eps)
    r, off, t = x.shape[0], 2.0 ** -22 * float(torch.linalg.matrix_norm(x)), 1.2
    if b * b > 64 * c * c or dtype == F32:
        t = 1.0
    for step in range(steps):
        left = steps - step
        ux = 2.0 ** -12 if dtype == BF16 and left == 1 else 2.0 ** -22
        ub = 2.0 ** -12 if dtype == BF16 and left <= 2 else 2.0 ** -22
        vx, vb = (2.0 ** -24 * (40 + k / 32) for k in (x.shape[1], r))
        s = float(torch.linalg.matrix_norm(x, 2))
        g = x @ x.T
        p = b * g + c * (g @ g)
        y = a * x + p @ x
        n = lambda z: float(torch.linalg.matrix_norm(z))  # noqa: E731
        h = n(g) + t * math.sqrt(r)
        dg = (2 * ub + vx) * s * n(x) + ub * h
        db = ((abs(b) + 2 * abs(c) * (s * s + t)) * dg + abs(c) * (2 * ub + vb) * (s * s + t) * h
              + (ux + vb) * (n(p) + 8 * math.sqrt(r)))
        sb = float(torch.linalg.matrix_norm(p, 2)) + abs(a)
        grid = torch.linspace(0, s, 200, dtype=torch.float64)
        grow = float((a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs().max())
        off = grow * off + s * db + (2 * ux + vb) * sb * n(x) + ux * n(y)
        x = y
    return x, off


def check(x, steps=5, co=DEFAULT, eps=1e-7, **kw):
    y = ops.orthogonalize(x, steps=steps, coefficients=co, eps=eps, **kw)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    half = torch.finfo(x.dtype).eps / 2
    for got, m in zip(y.reshape(-1, *x.shape[-2:]), x.reshape(-1, *x.shape[-2:])):
        want, off = formula(m, steps, co, eps, x.dtype)
        d = (got.double() - want).abs()
        small = 2.0 ** -25 * math.sqrt(want.numel()) if x.dtype == F16 else 0.0
        assert float(torch.linalg.matrix_norm(d)) <= 1.01 * (off + half * float(torch.linalg.matrix_norm(want)) + small)
        assert (d <= 1.01 * (off + half * want.abs() + small)).all()
    assert _lib.device_status() == (0, 0, 0, 0)
    return y


def gradient(cuda, *shape, dtype=F32, noise=0.5, size=1e-3, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    rank = min(4, *shape[-2:])
    x = torch.randn(*shape[:-1], rank, generator=g, device=cuda) @ torch.randn(*shape[:-2], rank, shape[-1], generator=g,
                                                                             device=cuda)
    return (size * (x + noise * torch.randn(*shape, generator=g, device=cuda))).to(dtype)


SHAPES = [  # in one launch: one CTA, clusters of two, four and eight; a launch a product: both sides odd, large
    (1, 1, 1), (2, 1, 37), (1, 300, 3), (3, 17, 33), (5, 16, 16), (2, 96, 250), (1, 128, 256), (1, 300, 31), (2, 100, 400),
    (1, 128, 513), (2, 1000, 128), (1, 40, 2047), (1, 128, 2048), (1, 128, 2049), (1, 129, 129), (3, 130, 257),
    (1, 700, 301), (2, 512, 512), (1, 1023, 1100),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,m,n", SHAPES)
def test_shapes(cuda, b, m, n, dtype):
    for steps in (1, 2, 5):
        check(gradient(cuda, b, m, n, dtype=dtype, seed=m), steps)


@pytest.mark.parametrize("m,n,dtype", [(2304, 2304, BF16), (1024, 4096, F32), (4100, 600, F16), (200, 9000, BF16)])
def test_large(cuda, m, n, dtype):
    """Pairs of CTAs, parts of K, several rounds of tiles."""
    check(gradient(cuda, 1, m, n, dtype=dtype), 5)


@pytest.mark.parametrize("co", [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.1), (1.0, 0.0, 0.0), (0.5, 0.0, 0.25)])
def test_coefficients(cuda, co):
    """With and without a square to complete; steps 0 and many."""
    for dtype in (BF16, F32):
        for m, n in ((60, 100), (201, 333)):
            check(gradient(cuda, 2, m, n, dtype=dtype), 3, co)
    for dtype in (BF16, F16, F32):
        x = gradient(cuda, 2, 33, 70, dtype=dtype)
        y = ops.orthogonalize(x, steps=0)
        want = x.double() / (torch.linalg.matrix_norm(x.double())[:, None, None] + 1e-7)
        assert ((y.double() - want).abs() <= want.abs() * torch.finfo(dtype).eps * 0.51 + 2.0 ** -25).all()
    x = gradient(cuda, 1, 150, 150)
    check(x, 12, (1.5, -0.5, 0.0))


def test_sizes_of_values(cuda):
    """The norm leaves nothing of the scale: tiny and huge gradients, zeros, an eps that counts."""
    for dtype, sizes in ((F32, (1e-30, 1e-20, 1e15, 1e30)), (BF16, (1e-30, 1e30)), (F16, (1e-4, 1e3))):
        for shape in ((2, 50, 90), (1, 150, 190)):
            for size in sizes:
                check(gradient(cuda, *shape, dtype=dtype, size=size), 5, eps=1e-38 if dtype != F16 else 1e-7)
    for shape in ((2, 50, 90), (1, 150, 190)):
        x = gradient(cuda, *shape)
        check(x, 3, eps=0.3)
        z = torch.zeros(*shape, device=cuda)
        assert not ops.orthogonalize(z).any()
        # one element much larger than the rest, and a matrix of rank one
        x[:, 3, 5] = 100.0
        check(x, 5)
        check(torch.outer(torch.randn(shape[1], device=cuda), torch.randn(shape[2], device=cuda))[None], 5)


def test_non_finite(cuda):
    """NaN or an infinity makes its matrix NaN, and no other of the batch."""
    for shape in ((3, 50, 90), (3, 90, 50), (3, 150, 190)):
        x = gradient(cuda, *shape)
        want = ops.orthogonalize(x)
        x[0, 7, 11], x[2, 4, 4] = float("nan"), float("inf")
        y = ops.orthogonalize(x)
        assert y[0].isnan().all() and y[2].isnan().all() and torch.equal(y[1], want[1])


def test_layouts(cuda):
    """Strided rows, transposed views, leading axes, in place, unaligned results."""
    for m, n in ((60, 72), (150, 200)):
        wide = gradient(cuda, 2, m, 3 * n + 1)
        for x in (wide[..., n:2 * n], wide[..., 1:n + 1], wide[:, :, ::2][..., :n], wide[0, :, :n].T, wide[1:, :, :n].mT,
                  wide[:, None, :, :n].expand(2, 3, m, n)):
            y = check(x)
            assert torch.equal(y, ops.orthogonalize(x.contiguous()))
        x = gradient(cuda, 2, m, n, dtype=BF16)
        want = ops.orthogonalize(x)
        flat = torch.full((2 * m * n + 2,), 7.0, device=cuda, dtype=BF16)
        out = flat[1:-1].view(2, m, n)  # not on a 16-byte border
        assert ops.orthogonalize(x, out=out) is out and torch.equal(out, want) and flat[0] == 7 and flat[-1] == 7
        tall = ops.orthogonalize(x.mT.contiguous())
        assert torch.equal(ops.orthogonalize(x.mT.contiguous(), out=flat[1:-1].view(2, n, m)), tall)
        assert ops.orthogonalize(x, out=x) is x and torch.equal(x, want)
    assert ops.orthogonalize(torch.empty(0, 8, 9, device=cuda)).shape == (0, 8, 9)


def test_batches_stay_apart(cuda):
    """Each matrix of a batch alone gives the same bits; many small ones."""
    for shape, dtype in (((7, 130, 70), BF16), ((40, 20, 31), F32), ((24, 128, 700), BF16)):
        x = gradient(cuda, *shape, dtype=dtype)
        y = ops.orthogonalize(x)
        for i in (0, 3, shape[0] - 1):
            assert torch.equal(ops.orthogonalize(x[i]), y[i])
    x = gradient(cuda, 700, 24, 24)
    check(x[:3])
    assert torch.equal(ops.orthogonalize(x)[699], ops.orthogonalize(x[699]))


def test_graph_and_streams(cuda):
    """Captured twice and replayed on other values; two streams at once."""
    for shape, dtype in (((2, 90, 100), F32), ((1, 300, 260), BF16)):
        x = gradient(cuda, *shape, dtype=dtype)
        ops.orthogonalize(x)
        graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
        for graph in graphs:
            with torch.cuda.graph(graph):
                outs.append(ops.orthogonalize(x))
        x.copy_(gradient(cuda, *shape, dtype=dtype, seed=9))
        for graph in graphs:
            graph.replay()
        want = ops.orthogonalize(x)
        assert all(torch.equal(o, want) for o in outs)
        torch.cuda.synchronize()
        outs = []
        for _ in range(3):
            with torch.cuda.stream(torch.cuda.Stream()):
                outs.append([ops.orthogonalize(x) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for some in outs for o in some)
        # work before it on the stream is waited for
        y = x.clone()
        for _ in range(4):
            y.zero_()
            y.add_(x)
            assert torch.equal(ops.orthogonalize(y), want)


def test_refusals(cuda):
    x = gradient(cuda, 8, 9)
    for error, args, kw in (
            (RuntimeError, (x.cpu(),), {}), (TypeError, (x.double(),), {}), (TypeError, (x.to(torch.int32),), {}),
            (ValueError, (x[0],), {}), (ValueError, (x[:, :0],), {}), (ValueError, (x,), {"steps": -1}),
            (ValueError, (x,), {"steps": 2.0}), (ValueError, (x,), {"steps": 1001}),
            (ValueError, (x,), {"coefficients": (1.0, float("nan"), 0.0)}), (ValueError, (x,), {"coefficients": (1.0, 2.0)}),
            (ValueError, (x,), {"eps": -1e-7}), (ValueError, (x,), {"out": x.half()}),
            (ValueError, (x,), {"out": torch.empty(9, 8, device=cuda).T})):
        with pytest.raises(error):
            ops.orthogonalize(*args, **kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,m,n", [(4, 512, 520), (20, 130, 200), (1, 161, 161), (1, 225, 1000), (2, 350, 290), (1, 900, 1100)])
def test_narrow_tiles(cuda, b, m, n, dtype):
    """Tiles of 64 and 32 columns, some of them wholly beyond the matrix."""
    check(gradient(cuda, b, m, n, dtype=dtype, seed=n), 5)
