"""Attention entry points with the reference's signatures.

``h3_attention_bnsd`` (ops/fa_h3.py:224-304) and ``fusion_attention_bnsd``
(ops/attention.py:100-131) take q/k/v as [B=1, H, S, D] and return
[1, H, S_q, D]; both run the tcgen05 flash-attention kernel reading the BNSD
strides in place.  There is one backend and no SDPA fallback: unsupported
inputs raise.  The reference's sequence-parallel entries are here too:
``gather_fa_bnsd`` / ``sp_gather_fa`` (K/V all-gathered, then attention) and
``ring_attention_bnsd`` (the K/V ring with log-sum-exp merges).

``cross_attention`` (no reference counterpart) is the differentiable form of
``ops.cross_attention``: a batch of query tokens against an encoder's states,
and ``rotary`` that of ``ops.rotary``, their positions.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from . import ops


def fusion_attention_bnsd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                          scale: Optional[float] = None) -> torch.Tensor:
    if q.dim() != 4:
        raise ValueError("expected 4D qkv [B, N, S, D]")
    if q.shape[0] != 1:
        raise ValueError("batch must be 1 (the reference's DiT runs B=1, model/dit.py:765-766)")
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    qt = q[0].permute(1, 0, 2)  # [S, H, D] view of BNSD storage
    kt = k[0].permute(1, 0, 2)
    vt = v[0].permute(1, 0, 2)
    if kt.stride() != vt.stride():
        kt, vt = kt.contiguous(), vt.contiguous()
    out = torch.empty((1, q.shape[1], q.shape[2], d), dtype=torch.bfloat16, device=q.device)
    ops.attention(qt, kt, vt, scale=scale, out=out[0].permute(1, 0, 2))
    return out


def h3_attention_bnsd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None,
                      gathered: bool = False) -> torch.Tensor:
    """Entry for the DiT: q/k/v [1, H, S, D]; ``gathered`` (KV already global)
    only matters to the reference's ring backend and is accepted for parity."""
    del gathered
    return fusion_attention_bnsd(q, k, v, scale=scale)


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv_lens, key_mask, scale):
        lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device)
        o = ops.cross_attention(q, k, v, kv_lens=kv_lens, key_mask=key_mask, scale=scale, lse=lse)
        ctx.save_for_backward(q, k, v, o, lse, kv_lens, key_mask)
        ctx.scale = scale
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, kv_lens, key_mask = ctx.saved_tensors
        if torch.is_grad_enabled():  # create_graph
            return (*_CrossAttentionGrad.apply(do, q, k, v, o, lse, kv_lens, key_mask, ctx.scale), None, None, None)
        return (*ops.cross_attention_bwd(do, q, k, v, o, lse, kv_lens=kv_lens, key_mask=key_mask, scale=ctx.scale),
                None, None, None)


class _CrossAttentionGrad(torch.autograd.Function):
    """The gradients as a node of a graph, so that a second derivative raises
    where it reaches them (without a node it would silently lack their part)."""

    @staticmethod
    def forward(ctx, do, q, k, v, o, lse, kv_lens, key_mask, scale):
        return ops.cross_attention_bwd(do, q, k, v, o, lse, kv_lens=kv_lens, key_mask=key_mask, scale=scale)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("cross_attention has no second derivatives")


def refuse_tangents(*ts: Optional[torch.Tensor], name: str = "cross_attention") -> None:
    """Raises if a tensor carries a forward-mode tangent: the kernels' results
    would come back without one.  (Where reverse mode is recorded too, the
    autograd function raises by itself.)"""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError(f"{name} has no forward-mode derivatives")


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """ops.cross_attention (q [B, Sq, H, D], k and v [B, Skv, Hkv, D]; see
    there for kv_lens and key_mask), differentiable by autograd in q, k and v.
    The backward pass is one call of ops.cross_attention_bwd; it keeps q, k,
    v, the result and a log-sum-exp per row, and is bit-reproducible.  There
    are no second derivatives and no forward-mode ones: asking for them raises."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, kv_lens, key_mask, scale)
    refuse_tangents(q, k, v)
    return ops.cross_attention(q, k, v, kv_lens=kv_lens, key_mask=key_mask, scale=scale)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rope, inverse):
        ctx.save_for_backward(positions)
        ctx.rope, ctx.inverse = rope, inverse
        ctx.shapes = q.shape, None if k is None else k.shape
        ctx.set_materialize_grads(False)  # zeros, for a result that nothing used, need not be turned
        return ops.rotary(q, k, positions, rope, inverse=inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        # linear, so its gradient is the other rotation, which has one in turn
        given, wanted = (dq, dk), ctx.needs_input_grad[:2]
        turn = [i for i in (0, 1) if wanted[i] and given[i] is not None]
        if turn:
            turned = rotary(given[turn[0]], given[1] if len(turn) == 2 else None, ctx.saved_tensors[0], ctx.rope,
                            inverse=not ctx.inverse)
        like = dk if dq is None else dq
        grads = [turned[turn.index(i)] if i in turn else like.new_zeros(ctx.shapes[i]) if wanted[i] and like is not None
                 else None for i in (0, 1)]
        return *grads, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: "ops.Rotary", *,
           inverse: bool = False) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """ops.rotary (q [B, S, H, D], k [B, S, Hkv, D] or None; see there for
    positions and rope), differentiable by autograd in q and k, any number of
    times; nothing but the positions is kept for the backward pass.  There are
    no forward-mode derivatives: asking for them raises."""
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, positions, rope, inverse)
    refuse_tangents(q, k, name="rotary")
    return ops.rotary(q, k, positions, rope, inverse=inverse)


def _tokens(t: torch.Tensor) -> torch.Tensor:
    """[1, H, S, D] or [H, S, D] (BNSD) -> a [S, H, D] token-major view."""
    if t.dim() == 4:
        if t.shape[0] != 1:
            raise ValueError("batch must be 1 (the reference's DiT runs B=1, model/dit.py:765-766)")
        t = t[0]
    if t.dim() != 3:
        raise ValueError("expected [1, H, S, D] or [H, S, D]")
    return t.permute(1, 0, 2)


def gather_fa_bnsd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None,
                   gathered: bool = False) -> torch.Tensor:
    """ops/gather_fa.py:130-181: this rank's queries [1, H, Sq, D] attend over
    every rank's keys.  Unless ``gathered``, the local K/V shards ([1, H, Sk, D]
    or [H, Sk, D]) are first all-gathered along the sequence in rank order
    (ulysses.all_gather_kv).  One attention kernel serves every
    ``H3_GATHER_FA_MODE`` of the reference (its tiled and head-chunked modes
    exist to fit NPU memory).  Returns [1, H, Sq, D] bf16."""
    from .dist import is_distributed
    from .ulysses import all_gather_kv

    qt, kt, vt = _tokens(q), _tokens(k), _tokens(v)
    if not gathered and is_distributed():
        kt, vt = all_gather_kv(kt.contiguous(), vt.contiguous())
    elif kt.stride() != vt.stride():
        kt, vt = kt.contiguous(), vt.contiguous()
    s_q, heads, d = qt.shape
    out = torch.empty((1, heads, s_q, d), dtype=torch.bfloat16, device=q.device)
    ops.attention(qt, kt, vt, scale=scale, out=out[0].permute(1, 0, 2))
    return out


def sp_gather_fa(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                 scale: Optional[float] = None) -> torch.Tensor:
    """ops/gather_fa.py:184-192: the DiT's gathered-attention entry on
    [H, S_local, D] q/k/v; returns [H, S_local, D]."""
    return gather_fa_bnsd(q.unsqueeze(0), k, v, scale=scale, gathered=False)[0]


def ring_attention_bnsd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                        scale: Optional[float] = None) -> torch.Tensor:
    """ops/ring_attention.py:67-123: local shards [1, H, S_local, D] in, the
    same shape out.  Under a process group the K/V shards travel around the
    ring and the chunk results merge through their log-sum-exps
    (ulysses.ring_attention); on one process it is plain attention."""
    from .dist import is_distributed
    from .ulysses import ring_attention

    if not is_distributed():
        return fusion_attention_bnsd(q, k, v, scale=scale)
    o = ring_attention(_tokens(q), _tokens(k), _tokens(v), scale=scale)
    return o.permute(1, 0, 2).unsqueeze(0).contiguous()
