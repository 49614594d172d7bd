"""Orthogonalised updates have the accuracy of 32-bit arithmetic, element by
element, for every type: what a lost plane, a left-out product or a block out
of its place would do to a result is far outside the bounds here.

Bounds.  ``modelled`` takes the steps in 64 bits with the roundings of a
product of f16 pairs where they happen, made of random numbers where their
size alone is known:

* an operand is the sum of two f16 numbers of 1024 times its value (22 bits,
  no finer than 2^-35);
* a product leaves out lo x lo;
* a sum over K is cut, not rounded, at each of its additions of 16 products:
  half a last place of what is there by then, 2^-24.5 of it on average, half
  of the whole on average, for 8 to 16 additions in a row 2^-21 of the whole
  at most; and rounded where parts are added, 2^-22 of its random size (the
  root of the sum of the squared products) with either sign;
* 16-bit results complete the square: G's diagonal is rounded with b / 2c
  beside it.

What these come to in the result follows from the steps themselves, which
multiply small singular values by 480.  A result is the nearest number of its
type to a value whose elements are off by at most 4 times the largest element
of two such errors (4: the numbers are random, and a kernel may cut in another
order), and in Frobenius norm by 4 times theirs; half a step of its type comes
on top."""
from __future__ import annotations

import math

import pytest
import torch

from minixmax_h3_b200 import _lib, ops

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEFAULT = (3.4445, -4.7750, 2.0315)
SCALE = 1024.0


def exact(x, steps, co, eps):
    """The formula in 64 bits, for one matrix."""
    a, b, c = co
    x = x.double()
    if x.shape[0] > x.shape[1]:
        return exact(x.T, steps, co, eps).T
    x = x / (torch.linalg.matrix_norm(x) + eps)
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def planes(v, count=2):
    """The f16 planes of SCALE v, as 64-bit numbers of v's size."""
    hi = (v * SCALE).half().double() / SCALE
    return hi, ((v - hi) * SCALE).half().double() / SCALE * (count > 1)


def product(x, y, gen, lo=(True, True)):
    """x y^T of planes, with the errors of its sums; lo: which of lo hi and hi lo are there."""
    s = x[0] @ y[0].T
    if lo[0]:
        s = s + x[1] @ y[0].T
    if lo[1]:
        s = s + x[0] @ y[1].T
    size = ((x[0] * x[0]) @ (y[0] * y[0]).T).sqrt()
    noise = torch.rand(s.shape, generator=gen, dtype=torch.float64).to(s.device) * 2 - 1
    return s * (1 - 2.0 ** -21) + 2.0 ** -22 * size * noise


def modelled(x, steps, co, eps, dtype, seed=0, wrong=None):
    """The value that is rounded to the result; ``wrong``(step, name) changes the planes that an operand has (an int)
    or the products that are made of it (a pair)."""
    a, b, c = co
    if x.shape[0] > x.shape[1]:
        return modelled(x.T, steps, co, eps, dtype, seed, wrong).T
    gen = torch.Generator().manual_seed(seed)
    wrong = wrong or (lambda step, name: None)

    def take(v, step, name):
        return planes(v, wrong(step, name) or 2)

    x = x.double()
    x = x / (torch.linalg.matrix_norm(x) + eps)
    square = dtype != F32 and c != 0 and b * b <= 64 * c * c
    one = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for step in range(steps):
        xs = take(x, step, "x")
        g = product(xs, xs, gen, wrong(step, "gram") or (True, True))
        if square:
            h = take(g + b / (2 * c) * one, step, "g")
            p = c * product(h, h, gen, wrong(step, "poly") or (True, True)) + (a - b * b / (4 * c)) * one
        else:
            h = take(g, step, "g")
            k = planes(c * g + b * one)
            p = product(h, k, gen, wrong(step, "poly") or (True, True)) + a * one
        p = take(p, step, "b")
        x = product(p, (xs[0].T, xs[1].T), gen, wrong(step, "mul") or (True, True))
    hi, lo = planes(x)
    return hi + lo


def outside(got, x, steps=5, co=DEFAULT, eps=1e-7):
    """What of ``got`` is out of its bounds, or None: (share of elements, Frobenius norm of the error over its bound)."""
    want = exact(x, steps, co, eps)
    errors = [modelled(x, steps, co, eps, got.dtype, seed) - want for seed in (1, 2)]
    most, norm = (4 * max(float(f(e)) for e in errors) for f in (lambda e: e.abs().max(), torch.linalg.matrix_norm))
    half, small = torch.finfo(got.dtype).eps / 2, 2.0 ** -25 if got.dtype == F16 else 0.0
    d = (got.double() - want).abs()
    out = ~(d <= most + half * (want.abs() + most) + small)
    over = float(torch.linalg.matrix_norm(d)) / (norm + half * float(torch.linalg.matrix_norm(want))
                                                 + small * math.sqrt(want.numel()))
    return (float(out.double().mean()), over) if bool(out.any()) or not over <= 1.0 else None


def gradient(m, n, dtype, noise, seed=0, batch=None):
    """A few directions and noise beside them."""
    g = torch.Generator().manual_seed(seed)
    lead = () if batch is None else (batch,)
    rank = min(4, m, n)
    x = torch.randn(*lead, m, rank, generator=g) @ torch.randn(*lead, rank, n, generator=g)
    return (1e-3 * (x + noise * torch.randn(*lead, m, n, generator=g))).to(dtype)


# ----------------------------------------------------------------------------- the bounds, on the CPU


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_bounds_take_what_is_modelled(dtype):
    for m, n, noise, steps in ((60, 130, 0.5, 5), (130, 100, 0.02, 5), (96, 97, 0.002, 5), (64, 200, 0.02, 2)):
        x = gradient(m, n, dtype, noise)
        for seed in (3, 4):
            assert outside(modelled(x, steps, DEFAULT, 1e-7, dtype, seed).to(dtype), x, steps) is None


def one_plane(names, steps):
    return lambda step, name: 1 if name in names and step in steps else None


def no_product(name, which, at):
    return lambda step, n: tuple(i != which for i in (0, 1)) if n == name and step == at else None


WRONG = {
    "x, g and b in one plane in the last steps": one_plane(("x", "g", "b"), (3, 4)),
    "x in one plane in the last step": one_plane(("x",), (4,)),
    "g and b in one plane in the last step": one_plane(("g", "b"), (4,)),
    "x in one plane once": one_plane(("x",), (2,)),
    "b in one plane once": one_plane(("b",), (1,)),
    "gram without lo hi once": no_product("gram", 0, 3),
    "gram without hi lo at last": no_product("gram", 1, 4),
    "polynomial without lo hi at last": no_product("poly", 0, 4),
    "polynomial without hi lo once": no_product("poly", 1, 2),
    "X' without lo hi at last": no_product("mul", 0, 4),
    "X' without hi lo once": no_product("mul", 1, 3),
}


@pytest.mark.parametrize("dtype,name", [(F32, n) for n in WRONG]
                         + [(t, n) for t in (BF16, F16) for n in WRONG if "plane" in n])
def test_bounds_refuse_what_is_left_out(dtype, name):
    """(A product left out of one sum can be less than half a step of 16 bits; the code of the sums is one for all types.)"""
    x = gradient(120, 190, dtype, 0.1)
    y = modelled(x, 5, DEFAULT, 1e-7, dtype, 3, WRONG[name])
    assert outside(y.to(dtype), x) is not None


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_bounds_refuse_blocks_out_of_place(dtype):
    x = gradient(150, 210, dtype, 0.5)
    y = modelled(x, 5, DEFAULT, 1e-7, dtype, 3).to(dtype)
    assert outside(y, x) is None

    def changed(f):
        z = y.clone()
        f(z)
        return outside(z, x)

    assert changed(lambda z: z[-1, -8:].zero_()) is not None  # the last row's last 16-byte words
    assert changed(lambda z: z[-1:].zero_()) is not None
    assert changed(lambda z: z[128:, 192:].zero_()) is not None  # a corner's block
    assert changed(lambda z: z[:32, 32:64].copy_(y[32:64, :32])) is not None  # another block's place
    assert changed(lambda z: z[:32, 32:64].copy_(y[:32, 32:64].T.clone())) is not None
    assert changed(lambda z: z[:, -1].copy_(y[:, -2])) is not None
    assert changed(lambda z: z[77, 33].fill_(float("nan"))) is not None


# ----------------------------------------------------------------------------- the kernels


def check(cuda, x, steps=5, co=DEFAULT, eps=1e-7):
    x = x.to(cuda)
    y = ops.orthogonalize(x, steps=steps, coefficients=co, eps=eps)
    for got, m in zip(y.reshape(-1, *x.shape[-2:]), x.reshape(-1, *x.shape[-2:])):
        assert outside(got, m, steps, co, eps) is None, (x.shape, x.dtype, steps, outside(got, m, steps, co, eps))
    assert _lib.device_status() == (0, 0, 0, 0)


SHAPES = [  # one CTA, clusters of two to eight, a launch a product: narrow tiles, shared K, single CTAs, pairs
    (17, 33), (96, 250), (300, 31), (128, 513), (1000, 128), (40, 2047), (128, 2048), (128, 2049), (129, 129), (130, 257),
    (225, 1000), (700, 301), (512, 512), (900, 1100), (600, 4100), (1300, 1200), (2304, 2304),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes(cuda, m, n, dtype):
    for steps, noise in ((1, 0.5), (2, 0.02), (5, 0.5)):
        check(cuda, gradient(m, n, dtype, noise, seed=m), steps)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("noise", [0.02, 0.002])
def test_few_directions(cuda, dtype, noise):
    """Updates of which a few directions are nearly all, which the steps do not bring near an orthogonal factor."""
    for m, n in ((96, 250), (512, 500), (1023, 1100)):
        for steps in (2, 3, 4, 5):
            check(cuda, gradient(m, n, dtype, noise, seed=n), steps)


@pytest.mark.gpu
@pytest.mark.parametrize("co", [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.1)])
def test_coefficients(cuda, co):
    for dtype in (BF16, F16, F32):
        for m, n in ((60, 100), (201, 333), (640, 600)):
            check(cuda, gradient(m, n, dtype, 0.5), 4, co)


@pytest.mark.gpu
def test_batches(cuda):
    for dtype in (BF16, F32):
        check(cuda, gradient(96, 700, dtype, 0.5, batch=3))
        check(cuda, gradient(200, 150, dtype, 0.5, batch=5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_zeros(cuda, dtype):
    """Zeros for any eps above zero, beside a matrix that has values; 0 / 0 without one."""
    for shape in ((3, 50, 90), (3, 150, 190), (3, 190, 150), (3, 700, 600)):
        x = gradient(*shape[1:], dtype, 0.5, batch=3).to(cuda)
        x[1] = 0
        for eps in (1.0, 1e-7, 1e-19, 1e-30, 1e-38, 1e-44):
            y = ops.orthogonalize(x, eps=eps)
            assert not y[1].any() and y[0].isfinite().all() and outside(y[2], x[2], eps=eps) is None
            assert not ops.orthogonalize(x, eps=eps, steps=0)[1].any()
        y = ops.orthogonalize(x, eps=0.0)
        assert y[1].isnan().all() and y[0].isfinite().all()
