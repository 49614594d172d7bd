"""GPU: cross attention where sizes of values, not of tensors, are unusual:
gradients far above and below 1 in f16, weights far apart, NaN in kept places,
tensors that start between 16-byte borders.

Tolerance as in test_gpu_cross_attention (4 u of the 2-norm).  An f16 result
below 2^-14 is rounded to multiples of 2^-24, which adds half of that a value;
``check`` leaves room for it where ``small`` is set."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cross_attention import UNIT, formula, make
from test_gpu_cross_attention import check as check_norm

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def check(got, want, dtype, name="", small=False):
    if not small:
        return check_norm(got, want, dtype, name)
    want = want.to(got.device)
    assert got.dtype == dtype and got.shape == want.shape
    held = want.abs() < 65000  # (f16's largest number is 65504: what lies beyond is an infinity)
    got, want = got[held], want[held]
    assert torch.isfinite(got).all(), name
    err, norm = (got.double() - want).norm().item(), want.norm().item()
    assert err <= 4 * UNIT[dtype] / 2 * norm + 2.0 ** -25 * math.sqrt(want.numel()), (name, err / max(norm, 1e-300))


def gradients(q, k, v, do, **kept):
    from minixmax_h3_b200 import _lib, ops

    lse = torch.empty(q.shape[0], q.shape[2], q.shape[1], device=q.device)
    o = ops.cross_attention(q, k, v, lse=lse, **kept)
    grads = ops.cross_attention_bwd(do, q, k, v, o, lse, **kept)
    assert _lib.device_status() == (0, 0, 0, 0)
    return o, lse, grads


# ----------------------------------------------------------------------------- f16 gradients


def parts(q, k, v, keep, do):
    """fp64 on the CPU: P, dS without the scale, and k and v of each query head."""
    q, k, v, do = (t.double().cpu() for t in (q, k, v, do))
    g = q.shape[2] // k.shape[2]
    kk, vv = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, kk) * q.shape[-1] ** -0.5
    p = torch.softmax(s.masked_fill(~keep.cpu()[:, None, None], -math.inf), -1)
    dp = torch.einsum("bihd,bjhd->bhij", do, vv)
    return p, p * (dp - (p * dp).sum(-1, keepdim=True)), kk, vv


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s_kv,kept", [(1, 1), (2, 2), (77, 1), (77, 3), (300, 2), (300, 3)])
@pytest.mark.parametrize("by_mask", [False, True])
def test_f16_dq_of_large_gradients_beside_left_out_keys(cuda, d, s_kv, kept, by_mask):
    """A few keys with low scores, delta = do . o above f16's largest number:
    the padding of a tile and left-out keys add nothing to dq."""
    g = torch.Generator(device=cuda).manual_seed(s_kv + kept + d)
    q = 0.6 + 0.1 * torch.randn(2, 9, 4, d, generator=g, device=cuda)
    k = -0.6 + 0.1 * torch.randn(2, s_kv, 2, d, generator=g, device=cuda)
    v = 1.0 + torch.randn(2, s_kv, 2, d, generator=g, device=cuda)
    do = 12 * 6000 / d + 100 * torch.randn(2, 9, 4, d, generator=g, device=cuda)
    q, k, v, do = (t.to(F16) for t in (q, k, v, do))
    keep = torch.zeros(2, s_kv, dtype=torch.bool, device=cuda)
    if by_mask:  # across the tiles
        keep[:, torch.linspace(0, s_kv - 1, kept, device=cuda).long()] = True
    else:
        keep[:, :kept] = True
    how = dict(key_mask=keep) if by_mask else dict(kv_lens=torch.full((2,), kept, dtype=torch.int32, device=cuda))
    o, lse, grads = gradients(q, k, v, do, **how)
    want = formula(q, k, v, keep, None, do)
    assert (do.double().cpu() * want[0]).sum(-1).abs().max() > 65504  # (of some rows)
    check(o, want[0], F16, "o")
    # Value by value, since keys with a common part make dq a sum that cancels:
    # dq's own rounding, dS's, and (delta from the rounded o, where the keys
    # take more than a tile) delta's; fp32 and ex2 to 2^-20 of the products.
    p, ds, kk, vv = parts(q, k, v, keep, do)
    u, scale = UNIT[F16], d ** -0.5
    many = s_kv > 128 and by_mask
    size = (do.double().cpu() * want[0]).abs().sum(-1).permute(0, 2, 1) if many else torch.zeros(2, 4, 9)
    most = torch.einsum("bihd,bjhd->bhij", do.double().cpu().abs(), vv.abs()).amax(-1)
    spread = torch.einsum("bhij,bjhd->bihd", ds.abs() + p * size[..., None], kk.abs())
    fine = torch.einsum("bhij,bjhd->bihd", p * most[..., None], kk.abs())
    bound = u * want[2].abs() + scale * (u * spread + 2.0 ** -20 * fine)
    assert torch.isfinite(grads[0]).all()
    assert ((grads[0].double().cpu() - want[2]).abs() <= bound).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e-3, 1e3])
@pytest.mark.parametrize("s_kv", [100, 1024])
def test_f16_dq_of_any_size(cuda, d, size, s_kv):
    """dS = P (dP - delta) enters a product in 16 bits: its error follows the
    gradient's size, not f16's range.  (Large keys keep dq itself in range.)"""
    q, k, v, do = make(cuda, 1, 512, s_kv, 4, 2, d, F16, seed=d + s_kv)
    q, k, do = q / 32, k * 32, (do.float() * size).to(F16)
    do[:, ::3] *= 0.125  # rows of different size
    check(gradients(q, k, v, do)[2][0], formula(q, k, v, None, None, do)[2], F16, "dq", small=True)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e-3, 1e3])
@pytest.mark.parametrize("s_kv", [100, 1024])
def test_f16_dk_and_dv_of_any_size(cuda, d, size, s_kv):
    """The same for dk, with large queries; samples and heads of different
    size do not share what their gradients are scaled by."""
    q, k, v, do = make(cuda, 2, 512, s_kv, 4, 2, d, F16, seed=d + s_kv + 1)
    q, k, do = q * 32, k / 32, (do.float() * size).to(F16)
    do[1] = (do[1].float() * 0.01).to(F16)
    want = formula(q, k, v, None, None, do)
    _, dk, dv = gradients(q, k, v, do)[2]
    for b in range(2):
        check(dk[b], want[3][b], F16, "dk", small=True)
        check(dv[b], want[4][b], F16, "dv", small=True)


@pytest.mark.parametrize("d", [64, 128])
def test_f16_dk_of_large_gradients(cuda, d):
    """Two keys and gradients of several thousands: dS passes f16's largest
    number, dq, dk and dv do not."""
    q, k, v, do = make(cuda, 2, 4, 2, 2, 2, d, F16, seed=d)
    q, k, do = q / 4, k / 4, (do.float() * 8e3 * (128 / d) ** 0.5).to(F16)
    want = formula(q, k, v, None, None, do)
    s = torch.einsum("bihd,bjhd->bhij", do.double().cpu(), v.double().cpu())
    assert d == 64 or (s[..., 0] - s[..., 1]).abs().max() * 0.25 > 65504  # (at 64 the largest dS is just below)
    for got, w, name in zip(gradients(q, k, v, do)[2], want[2:], ("dq", "dk", "dv")):
        check(got, w, F16, name)


def test_f16_gradients_of_nothing(cuda):
    """do of zero, values of zero, rows without a key beside others: zeros,
    not 0 times the largest power of two."""
    q, k, v, do = make(cuda, 2, 70, 60, 4, 2, 64, F16)
    mask = torch.ones(2, 60, dtype=torch.bool, device=cuda)
    mask[1] = False
    want = formula(q, k, v, mask, None, do)
    for got, w in zip(gradients(q, k, v, do, key_mask=mask)[2], want[2:]):
        check(got, w, F16)
        assert (got[1] == 0).all()
    for grad in gradients(q, k, v, torch.zeros_like(do))[2]:
        assert (grad == 0).all()
    dq, dk, _ = gradients(q, k, torch.zeros_like(v), do)[2]
    assert (dq == 0).all() and (dk == 0).all()


# ----------------------------------------------------------------------------- weights far apart


@pytest.mark.parametrize("s_q", [1, 200])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_long_tail_beside_a_dominant_key(cuda, s_q, dtype):
    """One key 17 to 18 nats above many equal ones: each of their weights is
    about 2^-25 of the first, their sum is not.  The dominant value is small
    (absent where the rows' kernel has normal f16 weights), so that the sum
    shows."""
    from minixmax_h3_b200 import ops

    n, h, d = 65536, 4, 64
    gap = torch.tensor([17.0, 17.5, 18.0, 17.25], dtype=torch.float64)
    q = (gap / 8)[None, None, :, None].expand(1, s_q, h, d).to(cuda, dtype).contiguous()  # (exact in 8 bits)
    k, v = torch.zeros(1, n, h, d, dtype=dtype, device=cuda), torch.ones(1, n, h, d, dtype=dtype, device=cuda)
    k[:, 0], v[:, 0] = 1.0, 0.0 if s_q == 1 else 1 / 64
    lse = torch.empty(1, h, s_q, device=cuda)
    o = ops.cross_attention(q, k, v, lse=lse)
    top = torch.exp(gap)
    want = (top * v[0, 0, 0, 0].item() + n - 1) / (top + n - 1)
    check(o, want[None, None, :, None].expand(1, s_q, h, d), dtype)
    assert torch.allclose(lse.double().cpu(), torch.log(top + n - 1)[None, :, None].expand(1, h, s_q), atol=2e-5, rtol=2e-6)


# ----------------------------------------------------------------------------- NaN in kept places


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("s_q,s_kv", [(3, 40), (3, 300), (200, 40), (200, 300)])
def test_nan_is_not_hidden(cuda, dtype, s_q, s_kv):
    """A query row with a NaN gives NaN in o, lse and dq, and changes no other
    row of them; a kept key with one gives NaN everywhere."""
    q, k, v, do = make(cuda, 1, s_q, s_kv, 2, 2, 64, dtype)
    want_o, want_lse, want = gradients(q, k, v, do)
    q[0, 1, 0, 5] = math.nan
    o, lse, grads = gradients(q, k, v, do)
    bad = torch.zeros(1, s_q, 2, dtype=torch.bool, device=cuda)
    bad[0, 1, 0] = True
    for got, clean in ((o, want_o), (lse.transpose(1, 2)[..., None], want_lse.transpose(1, 2)[..., None])):
        assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])
    assert torch.isnan(grads[0][bad]).all()
    assert torch.isfinite(grads[0][~bad]).all()
    assert torch.isnan(grads[1][:, :, 0]).all() and torch.equal(grads[1][:, :, 1], want[1][:, :, 1])
    q[0, 1, 0, 5] = 1.0
    k[0, s_kv - 1, 1, 0] = math.nan
    o, lse, grads = gradients(q, k, v, do)
    assert torch.isnan(o[:, :, 1]).all() and torch.isnan(lse[:, 1]).all() and torch.isnan(grads[0][:, :, 1]).all()
    assert torch.isfinite(o[:, :, 0]).all() and torch.isfinite(lse[:, 0]).all()


# ----------------------------------------------------------------------------- layouts


def shifted(t):
    """A contiguous copy that starts one element behind a 16-byte border."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = buf[1:].view(t.shape)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out


@pytest.mark.parametrize("s_q", [3, 150])
def test_contiguous_tensors_between_16_byte_borders(cuda, s_q):
    """Layouts that cannot be read in place are copied, a contiguous tensor at
    an odd address too."""
    from minixmax_h3_b200 import ops

    q, k, v, do = make(cuda, 2, s_q, 50, 4, 2, 64, BF16)
    o, lse, grads = gradients(q, k.contiguous(), v.contiguous(), do)
    got = torch.empty_like(lse)
    assert torch.equal(ops.cross_attention(shifted(q), shifted(k), shifted(v), lse=got), o) and torch.equal(got, lse)
    assert torch.equal(ops.cross_attention(q, k.contiguous(), shifted(v)), o)
    for odd in ((0,), (1, 2), (3,), (4,), (0, 1, 2, 3, 4)):
        args = [shifted(t) if i in odd else t for i, t in enumerate((do, q, k, v, o))]
        assert all(torch.equal(a, b) for a, b in zip(ops.cross_attention_bwd(*args, lse), grads)), odd
    c = ops.KV8Cache.empty(2, 2, 64, device=cuda)
    c2 = ops.KV8Cache.empty(2, 2, 64, device=cuda)
    table, lens = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([[0], [1]], [0, 0]))
    ops.kv8_append(c, k, v, table, lens)
    ops.kv8_append(c2, shifted(k), shifted(v), table, lens)
    assert torch.equal(c.k, c2.k) and torch.equal(c.v, c2.v) and c.k.any()
    assert torch.equal(ops.kv8_attention(shifted(q), c, table, lens + 50), ops.kv8_attention(q, c, table, lens + 50))
