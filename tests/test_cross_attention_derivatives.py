"""CPU: derivatives that cross attention does not have raise, none is silently
left out (the library is replaced by a stub; no kernel runs)."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from minixmax_h3_b200 import attention, ops
from minixmax_h3_b200 import torch_ops as T

BF16 = torch.bfloat16


def qkv(**kw):
    return [torch.randn(1, n, 2, 64, **kw).to(BF16) for n in (4, 5, 5)]


@pytest.fixture
def stub(monkeypatch):
    """The entry points' results without their work."""
    monkeypatch.setattr(ops, "_cuda", lambda *a: None)
    monkeypatch.setattr(ops, "call", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda t: 0)
    monkeypatch.setattr(ops, "_workspace", lambda *a: None)


@pytest.fixture
def cpu_operator(stub):
    """h3b::cross_attention with its own formula for gradients, for CPU
    tensors under another name."""
    lib = torch.library.custom_op("h3b_test::cross_attention", mutates_args=())(T._cross_attention)
    lib.register_autograd(T._cross_attention_grad, setup_context=T._cross_attention_setup)
    return lib


def test_gradient_through_the_log_sum_exps_raises(cpu_operator, monkeypatch):
    """lse is for the backward pass: a loss that uses it has no gradient here,
    alone or beside one that uses o."""
    def no_bwd(*a):
        pytest.fail("gradients without the part of lse")

    q, k, v = (t.requires_grad_() for t in qkv())
    for loss in (lambda o, lse: lse.sum(), lambda o, lse: lse.sum() + o.float().sum()):
        out = cpu_operator(q, k, v, None, None, None)
        with monkeypatch.context() as m:
            m.setattr(T.torch.ops.h3b, "cross_attention_bwd", no_bwd, raising=False)
            with pytest.raises(RuntimeError, match="lse"):
                loss(*out).backward()


def test_gradient_of_the_result_alone(cpu_operator, monkeypatch):
    q, k, v = (t.requires_grad_() for t in qkv())
    o, _ = cpu_operator(q, k, v, None, None, None)
    do = torch.randn_like(o)
    seen = []

    def bwd(dout, q, k, v, *rest):
        seen.append(dout)
        return torch.ones_like(q), 2 * torch.ones_like(k), 3 * torch.ones_like(v)

    monkeypatch.setattr(T.torch.ops.h3b, "cross_attention_bwd", bwd, raising=False)
    got = torch.autograd.grad(o, (q, k, v), do)
    assert len(seen) == 1 and torch.equal(seen[0], do)
    assert [g.flatten()[0].item() for g in got] == [1, 2, 3]


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_raises(stub, which, grad):
    """A tangent of q, k or v must not be dropped."""
    with fwd.dual_level():
        args = qkv()
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        if grad:
            args[(which + 1) % 3].requires_grad_()
        with pytest.raises(NotImplementedError):
            attention.cross_attention(*args)
        attention.cross_attention(*qkv())
    attention.cross_attention(*qkv())


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_of_the_operator_raises(cpu_operator, which):
    with fwd.dual_level():
        args = qkv()
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            cpu_operator(*args, None, None, None)
        cpu_operator(*qkv(), None, None, None)


def test_layer_refuses_what_needs_a_gradient(stub, monkeypatch):
    """The layer's projections are quantised and have no gradients: inputs
    that need one raise, and do not come back detached."""
    from minixmax_h3_b200.block import CrossAttention

    layer = CrossAttention(128, 2, 64, 256)
    for name in ("q_proj", "kv_proj", "out_proj"):
        p = getattr(layer, name)
        monkeypatch.setattr(p, "forward", lambda x, n=p.out_features: x.new_zeros(x.shape[0], n))
    x, cond = torch.randn(1, 4, 128).to(BF16), torch.randn(1, 5, 256).to(BF16)
    kv = layer.encode(cond)
    layer(x, cond), layer(x, kv=kv)
    need = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    for call in (lambda: layer(need(x), cond), lambda: layer(x, need(cond)), lambda: layer.encode(need(cond)),
                 lambda: layer(x, kv=(kv[0], need(kv[1]))), lambda: layer(need(x), kv=kv)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()
