"""CPU: host-side checks of cross attention and the 8-bit cache (no kernel
runs): argument refusals of the C ABI and of ops, workspace sizes, the custom
operators' shapes."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from minixmax_h3_b200 import _lib, ops
from minixmax_h3_b200 import torch_ops as T  # noqa: F401

BF16 = torch.bfloat16


def fwd(**kw):
    a = dict(q=32, k=32, v=32, o=32, lse=None, dtype=0, b=1, h=2, hkv=2, d=128, sq=4, skv=8, qs=(1024, 256, 128),
             ks=(2048, 256, 128), os=(1024, 256, 128), lens=None, mask=None, ms=0, scale=0.1, ws=None, wsb=0)
    a.update(kw)
    return _lib.lib().h3b_cross_attention_fwd(
        a["q"], a["k"], a["v"], a["o"], a["lse"], a["dtype"], a["b"], a["h"], a["hkv"], a["d"], a["sq"], a["skv"],
        *a["qs"], *a["ks"], *a["os"], a["lens"], a["mask"], a["ms"], a["scale"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 8), (dict(o=None), 8), (dict(scale=0.0), 8), (dict(scale=float("nan")), 8), (dict(ms=-1), 8),
    (dict(dtype=2), 3), (dict(d=96), 1), (dict(h=3), 1), (dict(hkv=0), 1), (dict(sq=-1), 1),
    (dict(q=40), 2), (dict(qs=(1024, 250, 128)), 2), (dict(ks=(2048, -256, 128)), 2), (dict(os=(1024, 0, 128)), 2),
    (dict(sq=0), 0), (dict(b=0), 0)])
def test_forward_refusals(kw, code):
    assert fwd(**kw) == code


def bwd(**kw):
    a = dict(do=32, q=32, k=32, v=32, o=32, lse=32, dq=32, dk=32, dv=32, dtype=0, b=1, h=2, hkv=2, d=128, sq=4, skv=8,
             s=(1024, 256, 128), ks=(2048, 256, 128), ws=32, wsb=1 << 20, scale=0.1)
    a.update(kw)
    return _lib.lib().h3b_cross_attention_bwd(
        a["do"], a["q"], a["k"], a["v"], a["o"], a["lse"], a["dq"], a["dk"], a["dv"], a["dtype"], a["b"], a["h"],
        a["hkv"], a["d"], a["sq"], a["skv"], *a["s"], *a["s"], *a["ks"], *a["s"], None, None, 0, a["scale"], a["ws"],
        a["wsb"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(do=None), 8), (dict(lse=None), 8), (dict(dk=None), 8), (dict(ws=None), 8), (dict(wsb=0), 1),
    (dict(dq=48), 2), (dict(do=40), 2), (dict(s=(1024, 250, 128)), 2), (dict(dtype=7), 3), (dict(d=32), 1),
    (dict(b=0), 0)])
def test_backward_refusals(kw, code):
    assert bwd(**kw) == code


def kv8(**kw):
    a = dict(q=32, o=32, dtype=0, b=1, h=4, hkv=2, d=64, sq=2, qs=(512, 256, 64), k=32, v=32, ks=32, vs=32, ct=0, nb=4,
             bt=64, table=32, mb=2, lens=32, scale=0.1, ws=None, wsb=0)
    a.update(kw)
    return _lib.lib().h3b_kv8_attention(
        a["q"], a["o"], None, a["dtype"], a["b"], a["h"], a["hkv"], a["d"], a["sq"], *a["qs"], *a["qs"], a["k"], a["v"],
        a["ks"], a["vs"], a["ct"], a["nb"], a["bt"], a["table"], a["mb"], a["lens"], 0, a["scale"], a["ws"], a["wsb"],
        None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 8), (dict(table=None), 8), (dict(lens=None), 8), (dict(scale=-1.0), 8), (dict(ct=2), 3),
    (dict(dtype=3), 3), (dict(bt=48), 1), (dict(nb=0), 1), (dict(mb=0), 1), (dict(nb=1 << 31), 1), (dict(d=80), 1),
    (dict(k=24), 2), (dict(qs=(512, 257, 64)), 2), (dict(b=0), 0), (dict(sq=0), 0)])
def test_cache_attention_refusals(kw, code):
    assert kv8(**kw) == code


def test_cache_write_and_read_refusals():
    lib = _lib.lib()
    ok = [32, 32, 0, 1, 4, 2, 64, 512, 128, 64, 32, 32, 32, 32, 0, 4, 64, 32, 2, 32, None, None]
    for at, value, code in ((0, None, 8), (17, None, 8), (2, 2, 3), (14, 5, 3), (6, 100, 1), (16, 16, 1), (15, 0, 1),
                            (8, 130, 2), (0, 40, 2), (3, 0, 0), (4, 0, 0)):
        args = list(ok)
        args[at] = value
        assert lib.h3b_kv8_append(*args) == code, at
    ok = [32, 32, 32, 32, 0, 4, 2, 64, 64, 32, 2, 32, 1, 10, 32, 32, 0, None]
    for at, value, code in ((0, None, 8), (14, None, 8), (4, 9, 3), (16, 3, 3), (7, 65, 1), (8, 32, 1), (0, 8, 2),
                            (13, 0, 0), (12, 0, 0)):
        args = list(ok)
        args[at] = value
        assert lib.h3b_kv8_read(*args) == code, at


def test_workspace_sizes():
    lib, n = _lib.lib(), ctypes.c_int64(-1)
    at = ctypes.addressof(n)
    assert lib.h3b_cross_attention_workspace(1, 24, 24, 128, 32768, 512, at) == 0 and n.value == 0
    assert lib.h3b_kv8_attention_workspace(1, 24, 24, 128, 1, 64, 2048, at) == 0 and n.value > 0
    # a multiple of whole partial rows: 128 values and two statistics
    assert n.value % (24 * 130 * 4) == 0
    assert lib.h3b_cross_attention_bwd_workspace(2, 4, 2, 64, 100, 77, at) == 0
    assert n.value >= 2 * 4 * 100 * 4
    assert lib.h3b_cross_attention_workspace(1, 3, 2, 128, 1, 1, at) == 1
    assert lib.h3b_kv8_attention_workspace(1, 4, 2, 128, 1, 64, 0, at) == 1
    assert lib.h3b_cross_attention_workspace(1, 1, 1, 128, 1, 1, None) == 8


def t(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype)


def test_ops_refuse_cpu_tensors():
    q, k = t(1, 4, 2, 64), t(1, 5, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.cross_attention(q, k, k)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.cross_attention_bwd(q, q, k, k, q, t(1, 2, 4, dtype=torch.float32))
    c = ops.KV8Cache.empty(2, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.kv8_attention(q, c, t(1, 2, dtype=torch.int32), t(1, dtype=torch.int32))


def test_ops_refuse_bad_arguments(monkeypatch):
    """The checks behind the device test, which is switched off here; the
    library is never reached."""
    monkeypatch.setattr(ops, "_cuda", lambda *a: None)
    monkeypatch.setattr(ops, "call", lambda *a: pytest.fail("reached the library"))
    q, k = t(2, 4, 4, 64), t(2, 5, 2, 64)
    bad = [
        (TypeError, (q, k, k.half()), {}), (TypeError, (q.float(), k.float(), k.float()), {}),
        (ValueError, (q[0], k, k), {}), (ValueError, (q, k[:1], k[:1]), {}), (ValueError, (q, k, k[:, :4]), {}),
        (ValueError, (t(2, 4, 3, 64), k, k), {}), (ValueError, (t(2, 4, 4, 96), t(2, 5, 2, 96), t(2, 5, 2, 96)), {}),
        (ValueError, (q, k, k), dict(kv_lens=t(2, dtype=torch.int64))),
        (ValueError, (q, k, k), dict(kv_lens=t(3, dtype=torch.int32))),
        (ValueError, (q, k, k), dict(key_mask=t(2, 5, dtype=torch.uint8))),
        (ValueError, (q, k, k), dict(key_mask=t(2, 4, dtype=torch.bool))),
        (ValueError, (q, k, k), dict(lse=t(2, 4, 4))),
        (ValueError, (q, k, k), dict(out=t(2, 4, 4, 32))),
    ]
    for error, args, kw in bad:
        with pytest.raises(error):
            ops.cross_attention(*args, **kw)
    with pytest.raises(ValueError):
        ops.cross_attention_bwd(q[:, :3], q, k, k, q, t(2, 4, 4, dtype=torch.float32))
    c, table, lens = ops.KV8Cache.empty(4, 2, 64), t(2, 3, dtype=torch.int32), t(2, dtype=torch.int32)
    for error, args in [
        (TypeError, (q.float(), c, table, lens)), (ValueError, (t(2, 4, 3, 64), c, table, lens)),
        (ValueError, (t(2, 4, 4, 128), c, table, lens)), (ValueError, (q, c, table.long(), lens)),
        (ValueError, (q, c, table, lens[:1])), (ValueError, (q, c, t(3, 2, dtype=torch.int32).T, lens)),
        (TypeError, (q, ops.KV8Cache(c.k.float(), c.v, c.k_scale, c.v_scale), table, lens)),
        (ValueError, (q, ops.KV8Cache(c.k, c.v[:2], c.k_scale, c.v_scale), table, lens)),
    ]:
        with pytest.raises(error):
            ops.kv8_attention(*args)
    with pytest.raises(TypeError):
        ops.kv8_append(c, k.float(), k.float(), table, lens)
    with pytest.raises(ValueError):
        ops.kv8_append(c, t(2, 5, 3, 64), t(2, 5, 3, 64), table, lens)
    with pytest.raises(TypeError):
        ops.kv8_read(c, table, lens, 10, dtype=torch.int8)
    with pytest.raises(TypeError):
        ops.KV8Cache.empty(4, 2, 64, dtype=torch.uint8)
    with pytest.raises(ValueError):
        ops.KV8Cache.empty(4, 2, 64, block_tokens=48)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            ops._scale(scale, 64)


def test_custom_operator_shapes():
    with FakeTensorMode():
        def f(*shape, dtype=BF16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        q, k = f(2, 7, 4, 64), f(2, 9, 2, 64)
        o, lse = torch.ops.h3b.cross_attention(q, k, k, None, None, None)
        assert o.shape == q.shape and o.dtype == BF16 and lse.shape == (2, 4, 7) and lse.dtype == torch.float32
        dq, dk, dv = torch.ops.h3b.cross_attention_bwd(o, q, k, k, o, lse, None, None, None)
        assert (dq.shape, dk.shape, dv.shape) == (q.shape, k.shape, k.shape)
        codes, scale = f(8, 2, 64, 64, dtype=torch.int8), f(8, 2, dtype=torch.float32)
        table, lens = f(2, 3, dtype=torch.int32), f(2, dtype=torch.int32)
        assert torch.ops.h3b.kv8_append(k, k, codes, codes.clone(), scale, scale.clone(), table, lens, None) is None
        assert torch.ops.h3b.kv8_attention(q, codes, codes, scale, scale, table, lens, False, None).shape == q.shape
    with pytest.raises(NotImplementedError):
        torch.ops.h3b.cross_attention(t(1, 4, 2, 64), t(1, 5, 2, 64), t(1, 5, 2, 64), None, None, None)


def fma32(a, b, c):
    """The product is exact in 64 bits; the sum rounds twice, which moves no
    code (a second rounding is off by 2^-53 of the value)."""
    return (a.astype(np.float64) * b.astype(np.float64) + c.astype(np.float64)).astype(np.float32)


@pytest.mark.parametrize("top", [127.0, 448.0])
def test_codes_by_corrected_quotient(top):
    """The append kernel's x / s (r = 1 / s; q = x r; q + (x - q s) r) gives
    the codes of a true division over the whole range of scales: s from 1e-12
    / 448 to the largest float / 127, |x| up to s * top, rows of 16-bit types
    and rescaled ones (any 32-bit value), ties included."""
    rng = np.random.default_rng(7)
    n = 1 << 20
    f = np.float32
    e = rng.uniform(-48.9, 120.9, n)
    s = np.exp2(e).astype(f)
    s[:4] = [f(1e-12) / f(448), f(1e-12) / f(127), f(3.4028235e38) / f(127), 1]
    with np.errstate(over="ignore"):  # (products past the largest float are dropped below)
        x = (s * rng.uniform(-top, top, n).astype(f)).astype(f)
    half = rng.integers(0, 2 * int(top), n // 4)   # near and on the borders between codes
    with np.errstate(over="ignore"):
        x[: n // 4] = ((half + 0.5).astype(f) * s[: n // 4]).astype(f)
    tiny = rng.integers(0, 1 << 31, n // 8).astype(np.uint32).view(f)
    small = np.isfinite(tiny) & (np.abs(tiny) < 2.0 ** -80)
    x[-(n // 8):][small] = tiny[small]
    x[::3] = (x[::3].view(np.uint32) & 0xffff0000).view(f)  # bf16 values
    keep = np.isfinite(x) & (np.abs(x) <= s.astype(np.float64) * top)
    x, s = x[keep], s[keep]
    assert x.size > n // 2
    with np.errstate(under="ignore"):
        r = (f(1) / s).astype(f)
        q = (x * r).astype(f)
        got = fma32(fma32(-q, s, x), r, q)
        want = (x / s).astype(f)
    assert r.min() >= np.finfo(f).tiny
    if top == 127.0:
        codes = [np.clip(np.rint(y), -127, 127) for y in (got, want)]
    else:
        codes = [torch.from_numpy(y).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy() & 0x7f
                 for y in (got, want)]
    assert (codes[0] == codes[1]).all()
