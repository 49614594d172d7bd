"""CPU: the host side of what conditioned layers are trained with - rotations'
frequencies, Muon around a plain orthogonalisation, the modules' arguments, the
custom operators' shapes, derivatives that are not there.  No kernel runs."""
from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from minixmax_h3_b200 import attention, block, modules, ops, optim
from minixmax_h3_b200 import torch_ops as T

PI = Fraction(3141592653589793238462643383279502884197169399375105820974945, 10 ** 60)


# ----------------------------------------------------------------------------- Rotary


@pytest.mark.parametrize("f", [0.0, 1.0, -1.0, 1e-4, 0.3, 6.5, -7.25, 1e-12, 123456.789, 5e-324])
def test_turns(f):
    """The nearest multiple of 2^-64 turns, modulo one, as a signed number."""
    got = ops._turns(f)
    assert -2 ** 63 <= got < 2 ** 63
    off = (Fraction(got) - Fraction(f) / (2 * PI) * 2 ** 64) % 2 ** 64
    assert min(off, 2 ** 64 - off) <= Fraction(51, 100) + abs(Fraction(f)) / 2 ** 100


def test_build():
    r = ops.Rotary.build(128, device="cpu")
    assert r.sections == (64,) and r.factor == 1.0 and not r.interleaved and r.turns.dtype == torch.int64
    assert r.turns.tolist() == [ops._turns(10000.0 ** (-2 * i / 128)) for i in range(64)]
    r = ops.Rotary.build((44, 42, 42), interleaved=True, device="cpu")
    assert r.sections == (22, 21, 21) and r.turns[22] == ops._turns(1.0) and r.interleaved
    # scaled: all, by the base (the fastest pair stays, the slowest is divided), by parts
    plain = [10000.0 ** (-2 * i / 64) for i in range(32)]
    by = {s: ops.Rotary.build(64, scaling=s, scale=4.0, trained_len=2048, device="cpu") for s in ("linear", "base", "by_parts")}
    assert by["linear"].turns.tolist() == [ops._turns(f / 4) for f in plain]
    base = by["base"].turns.tolist()
    assert base[0] == ops._turns(1.0) and abs(base[31] / ops._turns(plain[31] / 4) - 1) < 1e-12
    parts = by["by_parts"]
    assert parts.factor == 0.1 * math.log(4.0) + 1 and by["linear"].factor == by["base"].factor == 1.0
    for i, f in enumerate(plain):
        turns = 2048 * f / (2 * math.pi)
        low, high = sorted((ops._turns(f / 4), ops._turns(f)))
        assert low <= parts.turns[i] <= high
        if turns >= 32:
            assert parts.turns[i] == ops._turns(f)
        if turns <= 1:
            assert parts.turns[i] == ops._turns(f / 4)
    assert ops.Rotary.build(64, scaling="by_parts", scale=4.0, trained_len=2048, factor=1.0, device="cpu").factor == 1.0
    assert ops.Rotary.build((0, 2), scaling="base", scale=3.0, device="cpu").turns.tolist() == [ops._turns(1.0)]
    w = torch.tensor([0.5, 0.25], dtype=torch.float32)
    assert ops.Rotary.from_frequencies(w, device="cpu").turns.tolist() == [ops._turns(0.5), ops._turns(0.25)]


@pytest.mark.parametrize("kw", [
    {"dims": 63}, {"dims": (2, -2)}, {"dims": ()}, {"dims": 64, "scaling": "other"}, {"dims": 64, "theta": 0.0},
    {"dims": 64, "scale": -1.0}, {"dims": 64, "scaling": "by_parts", "scale": 2.0}, {"dims": (2, 2, 2, 2)},
    {"dims": 64, "scaling": "by_parts", "scale": 2.0, "trained_len": 100, "fast": 1.0, "slow": 2.0},
    {"dims": 64, "theta": float("nan")}, {"dims": 64, "factor": float("inf")},
])
def test_build_refusals(kw):
    with pytest.raises(ValueError):
        ops.Rotary.build(device="cpu", **kw)


def test_from_frequencies_refusals():
    for w, kw in (([1.0, float("nan")], {}), ([1.0], {"sections": (2,)}), ([1.0], {"sections": ()}), ([], {"sections": (1, -1)})):
        with pytest.raises(ValueError):
            ops.Rotary.from_frequencies(w, device="cpu", **kw)


def test_fields_are_checked():
    """Sections that are not the pairs would read positions that are not there."""
    turns = torch.zeros(4, dtype=torch.int64)
    for error, args in ((TypeError, (turns.int(), (4,))), (TypeError, (turns.view(2, 2), (2,))), (ValueError, (turns, (1, 1))),
                        (ValueError, (turns, ())), (ValueError, (turns, (5, -1))), (ValueError, (turns, (1, 1, 1, 1)))):
        with pytest.raises(error):
            ops.Rotary(*args)


def test_fields_stay_as_checked():
    sections = [2, 2]
    rope = ops.Rotary(torch.zeros(4, dtype=torch.int64), sections)
    sections[1] = 1
    assert rope.sections == (2, 2)
    for name, value in (("sections", (1, 1)), ("turns", torch.zeros(2, dtype=torch.int64)), ("factor", 2.0)):
        with pytest.raises(AttributeError):
            setattr(rope, name, value)


# ----------------------------------------------------------------------------- Muon


def plain(x, *, steps, coefficients, eps, out=None):
    a, b, c = coefficients
    y = x.double()
    y = y / (torch.linalg.matrix_norm(y)[..., None, None] + eps)
    for _ in range(steps):
        g = y @ y.mT
        y = a * y + (b * g + c * (g @ g)) @ y
    y = y.to(x.dtype)
    return y if out is None else out.copy_(y)


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def record(x, **kw):
        seen.append((tuple(x.shape), x.dtype))
        return plain(x, **kw)

    monkeypatch.setattr(ops, "orthogonalize", record)
    return seen


def test_muon_step(calls):
    """Two steps against the formula; one call for parameters of one shape; those without a gradient stay."""
    g = torch.Generator().manual_seed(0)
    params = [torch.randn(*s, generator=g).requires_grad_() for s in ((6, 4), (6, 4), (3, 5), (2, 4, 7), (6, 4))]
    grads = [[torch.randn(p.shape, generator=g) for p in params] for _ in range(2)]
    for nesterov in (True, False):
        want = [p.detach().clone().double() for p in params]
        mine = [p.detach().clone().requires_grad_() for p in params]
        opt = optim.Muon(mine, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.01, dtype=torch.float32)
        avg = [torch.zeros_like(w) for w in want]
        for step in range(2):
            calls.clear()
            for i, p in enumerate(mine):
                p.grad = None if i == 4 else grads[step][i].clone()
            opt.step()
            assert sorted(calls) == [((1, 2, 4, 7), torch.float32), ((1, 3, 5), torch.float32), ((2, 6, 4), torch.float32)]
            for i in range(4):
                gr = grads[step][i].double()
                avg[i] = 0.9 * avg[i] + 0.1 * gr
                u = 0.9 * avg[i] + 0.1 * gr if nesterov else avg[i]
                u = plain(u, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7)
                m, n = u.shape[-2:]
                want[i] = (1 - 0.1 * 0.01) * want[i] - 0.1 * max(1.0, m / n) ** 0.5 * u
        # fp32 states and updates, a few roundings each; the steps multiply an update's by 500 at most
        for p, w in zip(mine, want):
            assert (p.detach().double() - w).abs().max() <= 4000 * 2.0 ** -24
        assert torch.equal(mine[4].detach(), params[4].detach()) and mine[4] not in opt.state


def test_muon_state_and_types(calls):
    p = torch.randn(4, 6, dtype=torch.bfloat16).requires_grad_()
    opt = optim.Muon([p])
    p.grad = torch.randn(4, 6).bfloat16()
    opt.step()
    assert calls == [((1, 4, 6), torch.bfloat16)] and opt.state[p]["average"].dtype == torch.float32
    opt.state[p]["average"].fill_(1.0 + 2.0 ** -20)
    q = p.detach().clone().requires_grad_()
    other = optim.Muon([q], lr=0.5)
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["lr"] == 0.02
    assert torch.equal(other.state[q]["average"], opt.state[p]["average"])  # still fp32
    assert other.state[q]["average"].data_ptr() != opt.state[p]["average"].data_ptr()
    assert opt.step(lambda: torch.tensor(3.0)) == 3.0


def test_muon_refusals():
    m = torch.zeros(2, 2, requires_grad=True)
    for kw in ({"lr": -1.0}, {"momentum": 1.0}, {"weight_decay": -0.1}, {"dtype": torch.float64}, {"lr": float("nan")}):
        with pytest.raises(ValueError):
            optim.Muon([m], **kw)
    with pytest.raises(ValueError):
        optim.Muon([torch.zeros(3, requires_grad=True)])
    opt = optim.Muon([m])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.zeros(3, requires_grad=True)]})
    assert len(opt.param_groups) == 1


# ----------------------------------------------------------------------------- modules


def test_layers_arguments():
    rope = ops.Rotary.build(128, device="cpu")
    layer = block.CrossAttention(256, 4, 128, 64, kv_heads=2, norm=True, rope=rope)
    assert isinstance(layer.norm, modules.LayerNorm) and not any(p.requires_grad for p in layer.norm.parameters())
    assert block.CrossAttention(256, 4, 128, 64).norm is None
    x, cond = torch.zeros(1, 2, 256), torch.zeros(1, 3, 64)
    with pytest.raises(ValueError):
        layer._turned(x, None, "positions", False)
    with pytest.raises(ValueError):
        block.CrossAttention(256, 4, 128, 64)._turned(x, torch.zeros(2), "positions", False)
    with pytest.raises(ValueError):
        layer(x, kv=(x, x), cond_positions=torch.zeros(3))
    trained = block.TrainableCrossAttention(256, 4, 64, 96, kv_heads=2, rope=rope)
    assert [tuple(m.shape) for m in trained.matrices()] == [(256, 256), (128, 96), (128, 96), (256, 256)]
    assert set(trained.matrices()) | set(trained.norm.parameters()) == set(trained.parameters())
    with pytest.raises(ValueError):
        trained(x, cond)
    for kw in ({"head_dim": 96}, {"kv_heads": 3}, {"compute_dtype": torch.float32}):
        with pytest.raises(ValueError):
            block.TrainableCrossAttention(**{"hidden": 256, "heads": 4, "head_dim": 64, "cond_dim": 96, **kw})


def test_no_cpu_path():
    x, w = torch.zeros(1, 2, 2, 64), torch.ones(64)
    rope = ops.Rotary.build(64, device="cpu")
    for f in (lambda: ops.rotary(x, None, torch.zeros(2, dtype=torch.int32), rope), lambda: ops.layer_norm(x, w, w),
              lambda: ops.layer_norm_bwd(x, x, torch.zeros(2, 4), w), lambda: ops.orthogonalize(x)):
        with pytest.raises(RuntimeError):
            f()
    with pytest.raises(NotImplementedError):
        torch.ops.h3b.layer_norm(x, w, w, 1e-5)


# ----------------------------------------------------------------------------- custom operators


def test_fake_shapes():
    with FakeTensorMode():
        x = torch.empty(2, 5, 3, 64, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(64, device="cuda")
        y = torch.ops.h3b.rotary(x, torch.empty(2, 5, dtype=torch.int32, device="cuda"),
                                 torch.empty(32, dtype=torch.int64, device="cuda"), [32], False, 1.0, False)
        assert (y.shape, y.dtype) == (x.shape, x.dtype)
        y, stats = torch.ops.h3b.layer_norm(x, w, w, 1e-5)
        assert (y.shape, y.dtype, stats.shape, stats.dtype) == (x.shape, x.dtype, (2, 30), torch.float32)
        dx, dw, db = torch.ops.h3b.layer_norm_bwd(y, x, stats, w)
        assert dx.shape == x.shape and dw.shape == db.shape == (64,) and dw.dtype == torch.float32
        assert torch.ops.h3b.layer_norm_bwd(y, x, stats)[1].shape == (0,)
        assert torch.ops.h3b.orthogonalize(x, 5, 3.4445, -4.7750, 2.0315, 1e-7).shape == x.shape


# ----------------------------------------------------------------------------- derivatives


@pytest.fixture
def stub(monkeypatch):
    """The entry points' results without their work."""
    monkeypatch.setattr(ops, "_one_device", lambda *a: None)
    monkeypatch.setattr(ops, "_call_on", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda t: 0)
    monkeypatch.setattr(ops, "_workspace_on", lambda *a: torch.empty(0, dtype=torch.uint8))


def test_derivatives_that_are_not_there_raise(stub):
    x, w = torch.randn(3, 8, requires_grad=True), torch.ones(8, requires_grad=True)
    for p in (x, w):
        first, = torch.autograd.grad(modules.layer_norm(x, w, w).sum(), p, create_graph=True)
        with pytest.raises(RuntimeError, match="second"):
            torch.autograd.grad(first.sum(), x)
    rope = ops.Rotary.build(4, device="cpu")
    q, p = torch.randn(1, 2, 3, 8), torch.zeros(2, dtype=torch.int32)
    with torch.autograd.forward_ad.dual_level():
        for f in (lambda t: modules.layer_norm(t, w.detach()), lambda t: attention.rotary(t, None, p, rope),
                  lambda t: T._layer_norm(t, w.detach()), lambda t: T._rotary(t, p, rope.turns, [2])):
            with pytest.raises(NotImplementedError):
                f(torch.autograd.forward_ad.make_dual(q, q))


def test_gradients_asked_for(stub, monkeypatch):
    """Only what needs a gradient is computed, and rotary's gradient is the other rotation."""
    seen = []
    real = ops.layer_norm_bwd
    monkeypatch.setattr(ops, "layer_norm_bwd", lambda *a, **kw: seen.append(kw) or real(*a, **kw))
    x, w, b = torch.randn(3, 8), torch.ones(8, requires_grad=True), torch.zeros(8)
    modules.layer_norm(x, w, b).sum().backward()
    assert seen == [{"weight_grad": True, "bias_grad": False}] and w.grad.shape == (8,)
    assert not modules.layer_norm(x, w.detach(), b).requires_grad
    turned = []
    monkeypatch.setattr(ops, "rotary", lambda q, k, p, r, *, inverse=False: turned.append(inverse) or
                        (q.clone(), None if k is None else k.clone()))
    rope = ops.Rotary.build(4, device="cpu")
    q, p = torch.randn(1, 2, 3, 8, requires_grad=True), torch.zeros(2, dtype=torch.int32)
    k = torch.randn(1, 2, 1, 8)
    out = attention.rotary(q, k, p, rope)
    out[0].sum().backward()
    assert turned == [False, True]
    assert attention.rotary(q.detach(), k, p, rope, inverse=True)[1] is not None and turned[-1]
