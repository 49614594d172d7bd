"""GPU: layer norm and its gradients against the formulas in 64 bits.

Tolerances count roundings (u = 2^-24).  A row's sums run over at most 64 terms
a thread (long rows: n / 1024), 5 shuffles and 32 partial sums, so a mean of
values a is off by K u mean|a| at most, K = 110 + n / 1024; the first mean's own
error is taken off again by the second pass.

* forward: (K + 4) u |w| (1 + |xhat|) + 2 u |b|, and eps / 2 of the type;
* dx: rstd u (4 |g| + (2 K + 8) (mean|g| + |xhat| mean|g xhat|)), and what the
  stored mean's rounding (u |mean|, in units of the row's deviation) moves,
  rstd u |mean| rstd 2 (|c2| + mean|g| |xhat|);
* dw, db: sums over m rows: (m / ctas + ctas + 40) u sum|terms| - counted as
  (m + 200) u at most - and the same shift of xhat in each row.

The backward pass takes xhat from the stored mean and 1 / std, which are off as
in the forward pass, so xhat is off by e = K u (1 + |xhat|) before anything
else: where xhat itself is next to nothing that is more than its own rounding.
A term dy xhat moves by |dy| e, and dx by rstd (e |c2| + |xhat| mean(|g| e))."""
from __future__ import annotations

import pytest
import torch

from minixmax_h3_b200 import _lib, modules, ops

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def formulas(x, w, b, eps, dy=None):
    x = x.double()
    n = x.shape[-1]
    w = torch.ones(n, device=x.device, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = (x - mean) * rstd
    k = 110 + n / 1024
    out = {"y": (xhat * w + b, (k + 4) * U * w.abs() * (1 + xhat.abs()) + 2 * U * b.abs())}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w
    c1, c2 = g.mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True)
    a1, a2 = g.abs().mean(-1, keepdim=True), (g * xhat).abs().mean(-1, keepdim=True)
    shift = U * mean.abs() * rstd
    e = k * U * (1 + xhat.abs())
    out["dx"] = (rstd * (g - c1 - xhat * c2),
                 rstd * (U * (4 * g.abs() + (2 * k + 8) * (a1 + xhat.abs() * a2))
                         + 2 * shift * (c2.abs() + a1 * xhat.abs())
                         + e * c2.abs() + xhat.abs() * (g.abs() * e).mean(-1, keepdim=True)))
    m = x.shape[0]
    out["dw"] = ((dy * xhat).sum(0), (m + 200) * U * (dy * xhat).abs().sum(0) + (shift * dy.abs()).sum(0) * 2
                 + (dy.abs() * e).sum(0))
    out["db"] = (dy.sum(0), (m + 200) * U * dy.abs().sum(0))
    return out


def close(got, want, bound, name=""):
    eps = torch.finfo(got.dtype).eps
    bound = bound * 1.01 + want.abs() * eps / 2 * 1.01 + (2.0 ** -25 if got.dtype == F16 else 0)
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (name, (off - bound).max().item(), off.max().item())


def check(x, w, b, eps=1e-5, seed=7):
    m, n = x.shape
    stats = torch.empty(2, m, device=x.device)
    y = ops.layer_norm(x, w, b, eps, stats=stats)
    assert torch.equal(y, ops.layer_norm(x, w, b, eps))
    g = torch.Generator(device=x.device).manual_seed(seed)
    dy = torch.randn(m, n, generator=g, device=x.device).to(x.dtype)
    want = formulas(x, w, b, eps, dy)
    close(y, *want["y"], "y")
    dx, dw, db = ops.layer_norm_bwd(dy, x, stats, w)
    close(dx, *want["dx"], "dx")
    if w is None:
        assert dw is None and db is None
    else:
        close(dw, *want["dw"], "dw")
        close(db, *want["db"], "db")
        again = ops.layer_norm_bwd(dy, x, stats, w)
        assert all(torch.equal(s, t) for s, t in zip((dx, dw, db), again))
    assert _lib.device_status() == (0, 0, 0, 0)


TYPES = [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)]
# every group size (8 to 1024 threads, both passes), one element, odd widths, rows longer than the registers hold
WIDTHS = [1, 2, 7, 64, 128, 129, 250, 512, 1000, 1024, 1111, 2048, 3000, 4096, 8192, 8200, 12345, 16384, 20000, 40000]


@pytest.mark.parametrize("n", WIDTHS)
def test_widths(cuda, n):
    for i, (dtype, wtype) in enumerate(TYPES):
        g = torch.Generator(device=cuda).manual_seed(n + i)
        m = (1, 5, 37, 300)[(n + i) % 4]
        x = (torch.randn(m, n, generator=g, device=cuda) * 3 + torch.randn(m, 1, generator=g, device=cuda)).to(dtype)
        w = (1 + 0.2 * torch.randn(n, generator=g, device=cuda)).to(wtype)
        b = (0.3 * torch.randn(n, generator=g, device=cuda)).to(wtype)
        check(x, w, b)


@pytest.mark.parametrize("m", [1, 2, 3, 147, 149, 1000, 4099])
def test_rows(cuda, m):
    for n, dtype in ((96, BF16), (600, F32), (4096, BF16)):
        g = torch.Generator(device=cuda).manual_seed(m)
        x = torch.randn(m, n, generator=g, device=cuda).to(dtype)
        check(x, torch.randn(n, generator=g, device=cuda), torch.randn(n, generator=g, device=cuda))


def test_without_weights(cuda):
    x = torch.randn(33, 768, device=cuda).bfloat16()
    check(x, None, None)
    w = torch.randn(768, device=cuda)
    stats = torch.empty(2, 33, device=cuda)
    assert torch.equal(ops.layer_norm(x, w), ops.layer_norm(x, w, torch.zeros_like(w)))
    ops.layer_norm(x, w, stats=stats)
    dx, dw, db = ops.layer_norm_bwd(x, x, stats, w)
    for kw, want in (({"bias_grad": False}, (dw, None)), ({"weight_grad": False}, (None, db)),
                     ({"weight_grad": False, "bias_grad": False}, (None, None))):
        got = ops.layer_norm_bwd(x, x, stats, w, **kw)
        assert torch.equal(got[0], dx)
        for s, t in zip(got[1:], want):
            assert (s is None) == (t is None) and (t is None or torch.equal(s, t))


def test_large_mean_and_constant_rows(cuda):
    """A mean 10^4 deviations away, constant rows, eps 0, tiny and large values."""
    g = torch.Generator(device=cuda).manual_seed(1)
    base = torch.randn(8, 1024, generator=g, device=cuda)
    check(base + 10000.0, torch.ones(1024, device=cuda), torch.zeros(1024, device=cuda))
    check(base * 1e-3, torch.ones(1024, device=cuda), torch.zeros(1024, device=cuda))
    check(base * 1e4, torch.ones(1024, device=cuda), torch.zeros(1024, device=cuda), eps=0.0)
    for value in (0.0, 0.1, -77.7, 1e6):
        x = torch.full((3, 700), value, device=cuda)
        # sum and mean of equal values are off by K u |value|; what the second pass finds is taken off, the rest is
        # below u |value|: against the deviation sqrt(eps)
        y = ops.layer_norm(x, eps=1e-5)
        assert y.abs().max().item() <= 2 * U * abs(value) / 1e-5 ** 0.5 * 110


def test_non_finite_rows(cuda):
    """A row with NaN or an infinity gives NaN, its neighbours keep their bits."""
    for n, dtype in ((64, BF16), (4096, F32), (1111, F16)):
        x = torch.randn(6, n, device=cuda).to(dtype)
        w, b = torch.randn(n, device=cuda), torch.randn(n, device=cuda)
        want = ops.layer_norm(x, w, b)
        x[1, n // 2], x[4, 0] = float("nan"), float("inf")
        y = ops.layer_norm(x, w, b)
        bad = torch.tensor([1, 4], device=cuda)
        good = torch.tensor([0, 2, 3, 5], device=cuda)
        assert y[bad].isnan().all() and torch.equal(y[good], want[good])


def test_strides_and_shapes(cuda):
    g = torch.Generator(device=cuda).manual_seed(4)
    wide = torch.randn(20, 3, 776, generator=g, device=cuda).bfloat16()
    w, b = (torch.randn(768 + 1, generator=g, device=cuda)[1:] for _ in range(2))  # not aligned
    for x in (wide[:, 1, 8:], wide[:, 1, :768], wide[:, 2, 3:771], wide[:, 0].t()[:768].t().contiguous().t().t()):
        check(x, w, b)
    check(torch.randn(768, 20, generator=g, device=cuda).t(), w, b)          # columns apart: copied
    check(torch.randn(1, 768, generator=g, device=cuda).expand(9, 768), w, b)  # one row, read nine times
    strided = torch.randn(768, 2, generator=g, device=cuda)[:, 0]
    x = wide[:, 1, :768]
    assert torch.equal(ops.layer_norm(x, strided, strided), ops.layer_norm(x, strided.contiguous(), strided.contiguous()))
    x4 = torch.randn(2, 3, 5, 768, generator=g, device=cuda)
    y = ops.layer_norm(x4, w, b)
    assert y.shape == x4.shape and torch.equal(y.view(30, 768), ops.layer_norm(x4.view(30, 768), w, b))
    assert torch.equal(ops.layer_norm(x4[0, 0, 0], w, b), y[0, 0, 0])
    out = torch.empty_like(x4)
    assert ops.layer_norm(x4, w, b, out=out) is out and torch.equal(out, y)
    ops.layer_norm(x4, w, b, out=x4)  # in place
    assert torch.equal(x4, y)


def test_empty(cuda):
    x = torch.empty(2, 0, 96, device=cuda)
    w = torch.ones(96, device=cuda)
    assert ops.layer_norm(x, w).shape == x.shape
    dx, dw, db = ops.layer_norm_bwd(x, x, torch.empty(2, 0, device=cuda), w)
    assert dx.shape == x.shape and not dw.any() and not db.any()


def test_autograd(cuda):
    """modules.LayerNorm against the formulas, through a strided gradient, and
    against differences in the direction of the gradient."""
    g = torch.Generator(device=cuda).manual_seed(6)
    layer = modules.Ops.LayerNorm(320, eps=1e-6, device=cuda)
    assert layer.weight.dtype == F32 and set(dict(layer.named_parameters())) == {"weight", "bias"}
    with torch.no_grad():
        layer.weight.copy_(1 + 0.1 * torch.randn(320, generator=g, device=cuda))
        layer.bias.copy_(0.1 * torch.randn(320, generator=g, device=cuda))
    x = torch.randn(3, 17, 320, generator=g, device=cuda).requires_grad_()
    dy = torch.randn(320, 17, 3, generator=g, device=cuda).permute(2, 1, 0)
    y = layer(x)
    grads = torch.autograd.grad(y, (x, layer.weight, layer.bias), dy)
    want = formulas(x.detach().view(51, 320), layer.weight.detach(), layer.bias.detach(), 1e-6, dy.reshape(51, 320))
    for got, name in zip(grads, ("dx", "dw", "db")):
        close(got.view(want[name][0].shape), *want[name], name)
    # (f(x + h v) - f(x - h v)) / 2h = <dx, v> + O(h^2): fp32 results of size 1 give 51 * 320 u / h of noise at most
    v = torch.randn(3, 17, 320, generator=g, device=cuda)
    h = 2.0 ** -6
    with torch.no_grad():
        f = [(layer(x + s * h * v).double() * dy).sum() for s in (1, -1)]
    slope = (grads[0].double() * v).sum()
    size = (grads[0].double().square().sum() * v.double().square().sum()).sqrt()
    assert ((f[0] - f[1]) / (2 * h) - slope).abs() <= 0.02 * size
    # only what is asked for
    bare = modules.LayerNorm(320, elementwise_affine=False, device=cuda)
    assert not list(bare.parameters())
    gx, = torch.autograd.grad(bare(x), x, dy)
    close(gx.view(51, 320), *formulas(x.detach().view(51, 320), None, None, 1e-5, dy.reshape(51, 320))["dx"])
    fixed = x.detach()
    gw, = torch.autograd.grad(layer(fixed), layer.weight, dy)
    assert torch.equal(gw, grads[1])
    assert not layer(fixed.clone()).detach().requires_grad
    # a second derivative raises where it reaches the gradients
    first, = torch.autograd.grad(layer(x), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(first.sum(), x)
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        dual = torch.autograd.forward_ad.make_dual(fixed, v)
        with pytest.raises(NotImplementedError):
            layer(dual)


def test_graph_and_streams(cuda):
    w = torch.randn(1024, device=cuda)
    x, dy = (torch.randn(500, 1024, device=cuda).bfloat16() for _ in range(2))
    stats = torch.empty(2, 500, device=cuda)

    def step():
        y = ops.layer_norm(x, w, w, stats=stats)
        return (y, *ops.layer_norm_bwd(dy, x, stats, w))

    step()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    got = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            got.append(step())
    x.copy_(torch.randn_like(x))
    for graph in graphs:
        graph.replay()
    want = step()
    for outs in got:
        assert all(torch.equal(s, t) for s, t in zip(outs, want))
    # two streams at once, each with its own statistics and workspace
    torch.cuda.synchronize()
    results = []
    for _ in range(2):
        with torch.cuda.stream(torch.cuda.Stream()):
            own = torch.empty(2, 500, device=cuda)
            y = ops.layer_norm(x, w, w, stats=own)
            results.append((y, *ops.layer_norm_bwd(dy, x, own, w)))
    torch.cuda.synchronize()
    for outs in results:
        assert all(torch.equal(s, t) for s, t in zip(outs, want))


def test_offsets_past_32_bits(cuda):
    n = 4096
    m = 2 ** 31 // n + 3
    x = torch.zeros(m, n, dtype=BF16, device=cuda)
    tail = torch.randn(3, n, device=cuda).bfloat16()
    x[-3:] = tail
    w = torch.randn(n, device=cuda)
    stats = torch.empty(2, m, device=cuda)
    y = ops.layer_norm(x, w, w, stats=stats)
    assert torch.equal(y[-3:], ops.layer_norm(tail, w, w))
    dx, _, _ = ops.layer_norm_bwd(x, x, stats, w)
    own = torch.empty(2, 3, device=cuda)
    ops.layer_norm(tail, w, w, stats=own)
    assert torch.equal(dx[-3:], ops.layer_norm_bwd(tail, tail, own, w)[0])


def test_refusals(cuda):
    x, w = torch.zeros(4, 64, device=cuda), torch.ones(64, device=cuda)
    stats = torch.zeros(2, 4, device=cuda)
    for error, args, kw in (
            (RuntimeError, (x.cpu(),), {}), (RuntimeError, (x, w.cpu()), {}), (TypeError, (x.double(),), {}),
            (ValueError, (x, w[:32]), {}), (ValueError, (x, w.half()), {}), (ValueError, (x, None, w), {}),
            (ValueError, (x.bfloat16(), w, w.bfloat16()), {}), (ValueError, (x, w, w, -1.0), {}),
            (ValueError, (x, w, w, float("nan")), {}), (ValueError, (x[:, :0],), {}),
            (ValueError, (x[0, 0],), {}), (ValueError, (x, w), {"stats": stats[:, :3]}),
            (ValueError, (x, w), {"stats": stats.half()}), (ValueError, (x, w), {"out": x.half()}),
            (ValueError, (x, w), {"out": torch.empty(64, 4, device=cuda).t()})):
        with pytest.raises(error):
            ops.layer_norm(*args, **kw)
    for error, args in ((ValueError, (x[:2], x, stats, w)), (ValueError, (x.half(), x, stats, w)),
                        (ValueError, (x, x, stats[:1], w)), (RuntimeError, (x.cpu(), x, stats, w)),
                        (ValueError, (x, x, stats, w.half()))):
        with pytest.raises(error):
            ops.layer_norm_bwd(*args)


@pytest.mark.parametrize("n", [256, 100, 40000])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_c_entries_arguments(cuda, n, dt):
    """A bias without a weight (the Python call refuses it); a workspace off its alignment."""
    x, b = torch.randn(5, n, device=cuda).to(dt), torch.randn(n, device=cuda).to(dt)
    y, stats = torch.empty_like(x), torch.empty(2, 5, device=cuda)
    code, stream = {BF16: 0, F32: 2}[dt], torch.cuda.current_stream().cuda_stream
    assert code == ops._FLOATS[dt]
    at = stats.data_ptr()
    _lib.call("h3b_layer_norm_fwd", ops._NORM_ARGS.pack(x.data_ptr(), 0, b.data_ptr(), y.data_ptr(), at, at + 20, 5, n, n, n,
                                                        1e-5, code, code), stream)
    close(y, *formulas(x, None, b, 1e-5)["y"], "y")
    ws = torch.empty(1 << 24, dtype=torch.uint8, device=cuda)
    with pytest.raises(RuntimeError):
        _lib.call("h3b_layer_norm_bwd", ops._NORM_BWD_ARGS.pack(
            x.data_ptr(), x.data_ptr(), 0, at, at + 20, y.data_ptr(), b.data_ptr(), 0, ws.data_ptr() + 2, 5, n, n, n, n,
            ws.numel() - 2, code, code), stream)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("n", [264, 600, 768, 1152, 1536, 2056, 2560, 4104, 5120, 5128, 6144, 7000, 12288, 12296])
def test_rows_share_warps(cuda, n, dt):
    """Rows by fours and twos, and what is left of them: the same bits in any company."""
    g = torch.Generator(device=cuda).manual_seed(n)
    x = (torch.randn(11, n, generator=g, device=cuda) * 3 - 1).to(dt)
    w, b = torch.randn(n, generator=g, device=cuda), torch.randn(n, generator=g, device=cuda)
    want, stats = ops.layer_norm(x, w, b), torch.empty(2, 11, device=cuda)
    ops.layer_norm(x, w, b, stats=stats)
    for rows in (1, 2, 3, 5):
        wide, own = torch.full((rows + 1, n), 7.0, dtype=dt, device=cuda), torch.full((2, rows), 7.0, device=cuda)
        ops.layer_norm(x[4:4 + rows], w, b, out=wide[:rows], stats=own)
        assert torch.equal(wide[:rows], want[4:4 + rows]) and torch.equal(own, stats[:, 4:4 + rows])
        assert (wide[rows] == 7).all()
        check(x[:rows], w, b)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("m,n", [(9001, 520), (5003, 1048), (2777, 2056), (1201, 4104), (1999, 8192)])
def test_many_rounds(cuda, m, n, dt):
    """Several turns of the backward pass's ring, groups that end within a round, rows apart in memory."""
    g = torch.Generator(device=cuda).manual_seed(m)
    x = torch.randn(m, n + 24, generator=g, device=cuda).to(dt)[:, 8:n + 8]
    w, b = torch.randn(n, generator=g, device=cuda), torch.randn(n, generator=g, device=cuda)
    check(x, w, b)
    stats = torch.empty(2, m, device=cuda)
    ops.layer_norm(x, w, b, stats=stats)
    one = torch.randn(1, n, generator=g, device=cuda).to(dt)  # a gradient that is one row for all
    got, want = (ops.layer_norm_bwd(dy, x, stats, w) for dy in (one.expand(m, n), one.expand(m, n).contiguous()))
    assert all(torch.equal(s, t) for s, t in zip(got, want))
