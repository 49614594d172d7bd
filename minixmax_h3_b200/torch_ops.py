"""``torch.ops.h3b.*``: the hot path's kernels as torch custom operators.

The reference registers its gathered attention as a custom operator
(``torch.library.custom_op("h3::gather_fa_bnsd", mutates_args=())`` with a
``register_fake``, ops/gather_fa.py:195-206) so that it composes with torch's
tracing.  Importing this module registers the same kind of operator for each
kernel of the path:

    h3b::quant_i8_rows(x, convrot_group) -> (q int8 [m, k], scale fp32 [m])
    h3b::gemm_i8(q, xs, w, ws, bias, epilogue) -> y bf16 [m, n] ([m, n/2] SwiGLU)
    h3b::quant_nvfp4(x, hi_first) -> (codes u8 [m, k/2], blocked scales u8, gs fp32 [1])
    h3b::gelu_amax_scan(y, ymax2) -> None  (updates ymax2[1]; see ops.gelu_amax_scan)
    h3b::quant_nvfp4_gelu(y, ymax2, hi_first) -> (codes, blocked scales, gs) of bf16(gelu(y))
    h3b::gemm_nvfp4(a_codes, a_sf, a_gs, w_codes, w_sf, w_gs, bias, epilogue) -> y bf16
    h3b::attention(q, k, v, scale) -> o bf16 [S, H, 128]          (token-major)
    h3b::attention_bnsd(q, k, v, scale) -> o bf16 [1, H, S, 128]  (h3_attention_bnsd)
    h3b::rmsnorm_modulate(x, weight, shift, scale, eps, row_sel) -> h bf16 [m, hidden]
    h3b::rmsnorm_modulate_quant_i8(x, weight, shift, scale, eps, row_sel, convrot_group)
        -> (q int8 [m, hidden], scale fp32 [m])
    h3b::cross_attention(q, k, v, kv_lens, key_mask, scale)
        -> (o [B, Sq, H, D], lse fp32 [B, H, Sq]); differentiable in q, k, v
           through o (a loss that uses lse raises, and so does forward mode)
    h3b::cross_attention_bwd(dout, q, k, v, out, lse, kv_lens, key_mask, scale) -> (dq, dk, dv)
    h3b::kv8_append(k, v, codes and scales of K and V, block_table, lens, new_lens) -> None  (updates the cache)
    h3b::kv8_attention(q, codes and scales, block_table, lens, causal, scale) -> o [B, Sq, H, D]
    h3b::rotary(x, positions, turns, sections, interleaved, factor, inverse) -> x turned (the fields of
        ops.Rotary); differentiable in x, any number of times
    h3b::layer_norm(x, weight, bias, eps) -> (y, stats fp32 [2, rows]); differentiable in x, weight and
        bias through y
    h3b::layer_norm_bwd(dout, x, stats, weight) -> (dx, dweight, dbias), empty without a weight
    h3b::orthogonalize(x, steps, a, b, c, eps) -> x's shape and type (no gradient)

Each is registered for CUDA tensors only, so tensors on any other device raise
(there is no CPU fallback).  Each forwards to the ``ops`` function of the same
name, where a failing status code becomes a RuntimeError.  Each has a fake
implementation giving the output shapes and dtypes without running anything.
The operators write only fresh outputs (``mutates_args=()``; gelu_amax_scan
declares the one fp32 pair it updates, kv8_append the cache's four tensors), so the epilogue
that updates a residual in place (EPI_GATE_RES) is refused here; the modules
use it through ``ops`` directly.  NVFP4 operands are in the tensor cores'
nibble order (``ops.quant_nvfp4(hi_first=False)``, ``QuantLinear.prepare_cube``).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .attention import h3_attention_bnsd, refuse_tangents

_GEMM_EPILOGUES = (ops.EPI_STORE, ops.EPI_GELU, ops.EPI_SWIGLU)


def _rows_of(x: torch.Tensor) -> int:
    n = 1
    for d in x.shape[:-1]:
        n *= d
    return n


def _gemm_cols(n: int, epilogue: int) -> int:
    if epilogue not in _GEMM_EPILOGUES:
        raise ValueError(f"epilogue {epilogue}: the operator offers EPI_STORE, EPI_GELU and EPI_SWIGLU "
                         "(EPI_GATE_RES updates its residual in place; use ops.gemm_* for it)")
    return n // 2 if epilogue == ops.EPI_SWIGLU else n


# ----------------------------------------------------------------------------- implementations


def _quant_i8_rows(x: torch.Tensor, convrot_group: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.quant_i8_rows(x, convrot_group=convrot_group)


def _gemm_i8(q: torch.Tensor, xs: torch.Tensor, w: torch.Tensor, ws: torch.Tensor,
             bias: Optional[torch.Tensor] = None, epilogue: int = 0) -> torch.Tensor:
    _gemm_cols(w.shape[0], epilogue)
    return ops.gemm_i8(q, xs, w, ws, bias, epilogue=epilogue)


def _quant_nvfp4(x: torch.Tensor, hi_first: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    t = ops.quant_nvfp4(x, hi_first=hi_first)
    return t.codes, t.sf, t.gs


def _gelu_amax_scan(y: torch.Tensor, ymax2: torch.Tensor) -> None:
    ops.gelu_amax_scan(y, ymax2)


def _quant_nvfp4_gelu(y: torch.Tensor, ymax2: torch.Tensor,
                      hi_first: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    t = ops.quant_nvfp4_gelu(y, ymax2, hi_first=hi_first)
    return t.codes, t.sf, t.gs


def _gemm_nvfp4(a_codes: torch.Tensor, a_sf: torch.Tensor, a_gs: torch.Tensor, w_codes: torch.Tensor,
                w_sf: torch.Tensor, w_gs: torch.Tensor, bias: Optional[torch.Tensor] = None,
                epilogue: int = 0) -> torch.Tensor:
    _gemm_cols(w_codes.shape[0], epilogue)
    k = 2 * a_codes.shape[1]
    if w_codes.shape[1] * 2 != k:
        raise ValueError(f"gemm_nvfp4: activation K {k} vs weight K {w_codes.shape[1] * 2}")
    a = ops.NVFP4Tensor(a_codes, a_sf, a_gs, a_codes.shape[0], k, False)
    w = ops.NVFP4Tensor(w_codes, w_sf, w_gs, w_codes.shape[0], k, False)
    return ops.gemm_nvfp4(a, w, bias, epilogue=epilogue)


def _attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    return ops.attention(q, k, v, scale=scale)


def _attention_bnsd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    scale: Optional[float] = None) -> torch.Tensor:
    return h3_attention_bnsd(q, k, v, scale=scale)


def _rmsnorm_modulate(x: torch.Tensor, weight: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float,
                      row_sel: Optional[torch.Tensor] = None) -> torch.Tensor:
    return ops.rmsnorm_modulate(x.contiguous(), weight, shift, scale, eps, row_sel=row_sel)


def _rmsnorm_modulate_quant_i8(x: torch.Tensor, weight: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor,
                               eps: float, row_sel: Optional[torch.Tensor] = None,
                               convrot_group: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.rmsnorm_modulate_quant_i8(x, weight, shift, scale, eps, row_sel=row_sel, convrot_group=convrot_group)


def _cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_lens: Optional[torch.Tensor] = None,
                     key_mask: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> tuple[torch.Tensor, torch.Tensor]:
    refuse_tangents(q, k, v)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device)
    return ops.cross_attention(q, k, v, kv_lens=kv_lens, key_mask=key_mask, scale=scale, lse=lse), lse


def _cross_attention_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                         lse: torch.Tensor, kv_lens: Optional[torch.Tensor] = None,
                         key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None
                         ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return ops.cross_attention_bwd(dout, q, k, v, out, lse, kv_lens=kv_lens, key_mask=key_mask, scale=scale)


def _kv8_append(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                new_lens: Optional[torch.Tensor] = None) -> None:
    ops.kv8_append(ops.KV8Cache(k_codes, v_codes, k_scale, v_scale), k, v, block_table, lens, new_lens=new_lens)


def _kv8_attention(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, causal: bool = False,
                   scale: Optional[float] = None) -> torch.Tensor:
    return ops.kv8_attention(q, ops.KV8Cache(k_codes, v_codes, k_scale, v_scale), block_table, lens, causal=causal,
                             scale=scale)


def _rotary(x: torch.Tensor, positions: torch.Tensor, turns: torch.Tensor, sections: list[int],
            interleaved: bool = False, factor: float = 1.0, inverse: bool = False) -> torch.Tensor:
    refuse_tangents(x, name="rotary")
    return ops.rotary(x, None, positions, ops.Rotary(turns, tuple(sections), interleaved, factor), inverse=inverse)[0]


def _layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    refuse_tangents(x, weight, bias, name="layer_norm")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm: an axis of at least one element is normalised")
    stats = torch.empty((2, x.numel() // x.shape[-1]), dtype=torch.float32, device=x.device)
    return ops.layer_norm(x, weight, bias, eps, stats=stats), stats


def _layer_norm_bwd(dout: torch.Tensor, x: torch.Tensor, stats: torch.Tensor, weight: Optional[torch.Tensor] = None
                    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    dx, dw, db = ops.layer_norm_bwd(dout, x, stats, weight)
    return dx, x.new_empty(0) if dw is None else dw, x.new_empty(0) if db is None else db


def _orthogonalize(x: torch.Tensor, steps: int = 5, a: float = 3.4445, b: float = -4.7750, c: float = 2.0315,
                   eps: float = 1e-7) -> torch.Tensor:
    return ops.orthogonalize(x, steps=steps, coefficients=(a, b, c), eps=eps)


# ----------------------------------------------------------------------------- registration

quant_i8_rows = torch.library.custom_op("h3b::quant_i8_rows", mutates_args=(), device_types="cuda")(_quant_i8_rows)
gemm_i8 = torch.library.custom_op("h3b::gemm_i8", mutates_args=(), device_types="cuda")(_gemm_i8)
quant_nvfp4 = torch.library.custom_op("h3b::quant_nvfp4", mutates_args=(), device_types="cuda")(_quant_nvfp4)
gemm_nvfp4 = torch.library.custom_op("h3b::gemm_nvfp4", mutates_args=(), device_types="cuda")(_gemm_nvfp4)
gelu_amax_scan = torch.library.custom_op("h3b::gelu_amax_scan", mutates_args=("ymax2",),
                                         device_types="cuda")(_gelu_amax_scan)
quant_nvfp4_gelu = torch.library.custom_op("h3b::quant_nvfp4_gelu", mutates_args=(),
                                           device_types="cuda")(_quant_nvfp4_gelu)
attention = torch.library.custom_op("h3b::attention", mutates_args=(), device_types="cuda")(_attention)
attention_bnsd = torch.library.custom_op("h3b::attention_bnsd", mutates_args=(),
                                         device_types="cuda")(_attention_bnsd)
rmsnorm_modulate = torch.library.custom_op("h3b::rmsnorm_modulate", mutates_args=(),
                                           device_types="cuda")(_rmsnorm_modulate)
rmsnorm_modulate_quant_i8 = torch.library.custom_op("h3b::rmsnorm_modulate_quant_i8", mutates_args=(),
                                                    device_types="cuda")(_rmsnorm_modulate_quant_i8)

cross_attention = torch.library.custom_op("h3b::cross_attention", mutates_args=(),
                                          device_types="cuda")(_cross_attention)
cross_attention_bwd = torch.library.custom_op("h3b::cross_attention_bwd", mutates_args=(),
                                              device_types="cuda")(_cross_attention_bwd)
kv8_append = torch.library.custom_op("h3b::kv8_append", mutates_args=("k_codes", "v_codes", "k_scale", "v_scale"),
                                     device_types="cuda")(_kv8_append)
kv8_attention = torch.library.custom_op("h3b::kv8_attention", mutates_args=(), device_types="cuda")(_kv8_attention)
rotary = torch.library.custom_op("h3b::rotary", mutates_args=(), device_types="cuda")(_rotary)
layer_norm = torch.library.custom_op("h3b::layer_norm", mutates_args=(), device_types="cuda")(_layer_norm)
layer_norm_bwd = torch.library.custom_op("h3b::layer_norm_bwd", mutates_args=(), device_types="cuda")(_layer_norm_bwd)
orthogonalize = torch.library.custom_op("h3b::orthogonalize", mutates_args=(), device_types="cuda")(_orthogonalize)


@quant_i8_rows.register_fake
def _(x, convrot_group=0):
    m, k = _rows_of(x), x.shape[-1]
    return x.new_empty((m, k), dtype=torch.int8), x.new_empty((m,), dtype=torch.float32)


@gemm_i8.register_fake
def _(q, xs, w, ws, bias=None, epilogue=0):
    return q.new_empty((q.shape[0], _gemm_cols(w.shape[0], epilogue)), dtype=torch.bfloat16)


@quant_nvfp4.register_fake
def _(x, hi_first=False):
    m, k = _rows_of(x), x.shape[-1]
    sf_bytes = ops.sf_blocked_bytes(m, k) if m else 0
    return (x.new_empty((m, k // 2), dtype=torch.uint8), x.new_empty((sf_bytes,), dtype=torch.uint8),
            x.new_empty((1,), dtype=torch.float32))


@gelu_amax_scan.register_fake
def _(y, ymax2):
    return None


@quant_nvfp4_gelu.register_fake
def _(y, ymax2, hi_first=False):
    m, k = _rows_of(y), y.shape[-1]
    return (y.new_empty((m, k // 2), dtype=torch.uint8), y.new_empty((ops.sf_blocked_bytes(m, k),), dtype=torch.uint8),
            y.new_empty((1,), dtype=torch.float32))


@gemm_nvfp4.register_fake
def _(a_codes, a_sf, a_gs, w_codes, w_sf, w_gs, bias=None, epilogue=0):
    return a_codes.new_empty((a_codes.shape[0], _gemm_cols(w_codes.shape[0], epilogue)), dtype=torch.bfloat16)


@attention.register_fake
def _(q, k, v, scale=None):
    return q.new_empty(tuple(q.shape), dtype=torch.bfloat16)


@attention_bnsd.register_fake
def _(q, k, v, scale=None):
    return q.new_empty(tuple(q.shape), dtype=torch.bfloat16)


@rmsnorm_modulate.register_fake
def _(x, weight, shift, scale, eps, row_sel=None):
    return x.new_empty((_rows_of(x), x.shape[-1]), dtype=torch.bfloat16)


@rmsnorm_modulate_quant_i8.register_fake
def _(x, weight, shift, scale, eps, row_sel=None, convrot_group=0):
    m, hidden = _rows_of(x), x.shape[-1]
    return x.new_empty((m, hidden), dtype=torch.int8), x.new_empty((m,), dtype=torch.float32)


@cross_attention.register_fake
def _(q, k, v, kv_lens=None, key_mask=None, scale=None):
    return q.new_empty(tuple(q.shape)), q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32)


@cross_attention_bwd.register_fake
def _(dout, q, k, v, out, lse, kv_lens=None, key_mask=None, scale=None):
    return q.new_empty(tuple(q.shape)), k.new_empty(tuple(k.shape)), v.new_empty(tuple(v.shape))


def _cross_attention_setup(ctx, inputs, output):
    q, k, v, kv_lens, key_mask, scale = inputs
    ctx.save_for_backward(q, k, v, *output, kv_lens, key_mask)
    ctx.scale = scale
    ctx.set_materialize_grads(False)  # (a gradient of lse is None unless something has used it)


def _cross_attention_grad(ctx, dout, dlse):
    if dlse is not None:
        raise RuntimeError("h3b::cross_attention has no gradient through lse (it is for the backward pass): detach it")
    q, k, v, out, lse, kv_lens, key_mask = ctx.saved_tensors
    grads = torch.ops.h3b.cross_attention_bwd(dout, q, k, v, out, lse, kv_lens, key_mask, ctx.scale)
    return (*grads, None, None, None)


cross_attention.register_autograd(_cross_attention_grad, setup_context=_cross_attention_setup)


@kv8_append.register_fake
def _(k, v, k_codes, v_codes, k_scale, v_scale, block_table, lens, new_lens=None):
    return None


@kv8_attention.register_fake
def _(q, k_codes, v_codes, k_scale, v_scale, block_table, lens, causal=False, scale=None):
    return q.new_empty(tuple(q.shape))


@rotary.register_fake
def _(x, positions, turns, sections, interleaved=False, factor=1.0, inverse=False):
    return x.new_empty(tuple(x.shape))


@layer_norm.register_fake
def _(x, weight=None, bias=None, eps=1e-5):
    return x.new_empty(tuple(x.shape)), x.new_empty((2, _rows_of(x)), dtype=torch.float32)


@layer_norm_bwd.register_fake
def _(dout, x, stats, weight=None):
    if weight is None:
        return x.new_empty(tuple(x.shape)), x.new_empty(0), x.new_empty(0)
    return (x.new_empty(tuple(x.shape)), *(weight.new_empty(tuple(weight.shape)) for _ in range(2)))


@orthogonalize.register_fake
def _(x, steps=5, a=3.4445, b=-4.7750, c=2.0315, eps=1e-7):
    return x.new_empty(tuple(x.shape))


def _rotary_setup(ctx, inputs, output):
    _, positions, turns, *ctx.rest = inputs
    ctx.save_for_backward(positions, turns)


def _rotary_grad(ctx, dout):
    sections, interleaved, factor, inverse = ctx.rest
    dx = torch.ops.h3b.rotary(dout, *ctx.saved_tensors, sections, interleaved, factor, not inverse)
    return dx, None, None, None, None, None, None


rotary.register_autograd(_rotary_grad, setup_context=_rotary_setup)


def _layer_norm_setup(ctx, inputs, output):
    x, weight, bias, _ = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.with_bias = bias is not None
    ctx.set_materialize_grads(False)


def _layer_norm_grad(ctx, dout, dstats):
    if dstats is not None:
        raise RuntimeError("h3b::layer_norm has no gradient through stats (they are for the backward pass): detach them")
    x, weight, stats = ctx.saved_tensors
    dx, dw, db = torch.ops.h3b.layer_norm_bwd(dout, x, stats, weight)
    return dx, None if weight is None else dw, db if ctx.with_bias else None, None


layer_norm.register_autograd(_layer_norm_grad, setup_context=_layer_norm_setup)
