"""Torch-facing wrappers over the C ABI (device memory, streams, shapes).

Each wrapper validates dtypes/devices, allocates its outputs with the caching
allocator, and launches on the current CUDA stream.  There is no CPU path:
non-CUDA tensors raise.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from dataclasses import dataclass, replace
from typing import Optional, Sequence

import torch

from ._lib import call

EPI_STORE, EPI_GELU, EPI_GATE_RES, EPI_SWIGLU, EPI_STORE_POSMAX = 0, 1, 2, 3, 4


def _stream(t: torch.Tensor) -> int:
    # The raw handle of the current stream: 0.15 us against 2.3 us for a
    # torch.cuda.Stream object, on calls of 5 to 10 us.
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _cuda(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("minixmax_h3_b200 ops run on CUDA tensors only (no CPU fallback)")


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """Views x as [m, k] with unit column stride; returns (x2, m, k, ld)."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    ld = x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]
    return x2, x2.shape[0], x2.shape[1], ld


# ----------------------------------------------------------------------------- INT8


def quant_i8_rows(x: torch.Tensor, *, convrot_group: int = 0,
                  x_rot_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-row dynamic INT8 quantisation -> (q int8 [m,k], scale fp32 [m]).

    convrot_group=256 first rotates every 256-column group by the regular
    Hadamard matrix (ConvRot, ops/hadamard.py:35-44); x_rot_out, if given
    (dense [m, k], x's dtype), receives the rotated activation."""
    _cuda(x, x_rot_out)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("quant_i8_rows expects bf16/fp16 input")
    x2, m, k, ld = _rows(x)
    q = torch.empty((m, k), dtype=torch.int8, device=x.device)
    s = torch.empty((m,), dtype=torch.float32, device=x.device)
    if m == 0:  # empty batch (a zero-size tensor may carry a null pointer)
        return q, s
    dt = 0 if x.dtype == torch.bfloat16 else 1
    if convrot_group:
        if x_rot_out is not None and (x_rot_out.shape != (m, k) or x_rot_out.dtype != x.dtype
                                      or not x_rot_out.is_contiguous()):
            raise ValueError("x_rot_out must be a dense [m, k] tensor of x's dtype")
        call("h3b_quant_i8_rows_convrot", x2.data_ptr(), dt, m, k, ld, int(convrot_group), q.data_ptr(),
             s.data_ptr(), x_rot_out.data_ptr() if x_rot_out is not None else None, _stream(x))
    else:
        call("h3b_quant_i8_rows", x2.data_ptr(), dt, m, k, ld, q.data_ptr(), s.data_ptr(), _stream(x))
    return q, s


def gemm_i8(q: torch.Tensor, xs: torch.Tensor, w: torch.Tensor, ws: torch.Tensor,
            bias: Optional[torch.Tensor] = None, *, epilogue: int = EPI_STORE,
            resid: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
            row_sel: Optional[torch.Tensor] = None, amax_out: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = epi(acc * xs[m] * ws[n] + bias) in bf16; w is the [N, K] int8 weight.

    EPI_GATE_RES: y = resid + v * gate[row_sel[m]] with gate a [rows, N] table
    (a strided view is fine) and resid updated in place when out is None.
    EPI_SWIGLU: w rows interleaved by swiglu_interleave_perm; y is [m, N/2].
    """
    _cuda(q, xs, w, ws, bias, resid, gate, row_sel, amax_out, out)
    m, k = q.shape
    n = w.shape[0]
    if out is None:
        out = resid if epilogue == EPI_GATE_RES else torch.empty(
            (m, n // 2 if epilogue == EPI_SWIGLU else n), dtype=torch.bfloat16, device=q.device)
    if m == 0:
        return out
    gate_ld = _gate_ld(gate)
    call("h3b_gemm_i8_bf16", q.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), _ptr(bias), out.data_ptr(),
         out.stride(0), _ptr(resid), _ptr(gate), gate_ld, _ptr(row_sel), _ptr(amax_out), epilogue, m, n, k,
         _stream(q))
    return out


def gemm_i8_seq2head(q: torch.Tensor, xs: torch.Tensor, w: torch.Tensor, ws: torch.Tensor,
                     bias: Optional[torch.Tensor], recv_ptrs: Sequence[int], rank: int, heads: int) -> None:
    """QKV GEMM whose output rows land in every head owner's receive buffer
    [ws*m, 3, heads/ws, 128] (recv_ptrs in rank order): the seq->head
    Ulysses exchange fused into the epilogue."""
    _cuda(q, xs, w, ws, bias)
    m, k = q.shape
    arr = (ctypes.c_void_p * len(recv_ptrs))(*recv_ptrs)
    call("h3b_gemm_i8_seq2head", q.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), _ptr(bias),
         ctypes.cast(arr, ctypes.c_void_p), len(recv_ptrs), rank, heads, m, w.shape[0], k, _stream(q))


def _gate_ld(gate: Optional[torch.Tensor]) -> int:
    if gate is None:
        return 0
    if gate.stride(-1) != 1:
        raise ValueError("gate table needs unit column stride")
    return gate.stride(0) if gate.dim() == 2 else 0


def gemm_i8_acc(q: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Raw int32 accumulators sum_k q[m,k]*w[n,k] from the tensor cores."""
    _cuda(q, w)
    m, k = q.shape
    n = w.shape[0]
    acc = torch.empty((m, n), dtype=torch.int32, device=q.device)
    call("h3b_gemm_i8_acc_i32", q.data_ptr(), w.data_ptr(), acc.data_ptr(), m, n, k, _stream(q))
    return acc


# ----------------------------------------------------------------------------- NVFP4


@dataclass
class NVFP4Tensor:
    """Packed NVFP4 operand: codes [rows, k/2] u8, blocked e4m3 scales, fp32 gs."""

    codes: torch.Tensor
    sf: torch.Tensor
    gs: torch.Tensor
    rows: int
    k: int
    hi_first: bool


def sf_blocked_bytes(rows: int, k: int) -> int:
    return ((rows + 127) // 128 * 128) * ((k // 16 + 3) // 4 * 4)


def amax(x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    _cuda(x)
    if x.dtype != torch.bfloat16 or not x.is_contiguous():
        raise TypeError("amax expects a contiguous bf16 tensor")
    if out is None:
        out = torch.empty((1,), dtype=torch.float32, device=x.device)
    if x.numel() == 0:
        return out.zero_()
    call("h3b_amax_bf16", x.data_ptr(), x.numel(), out.data_ptr(), _stream(x))
    return out


def quant_nvfp4(x: torch.Tensor, *, hi_first: bool = False,
                amax_t: Optional[torch.Tensor] = None) -> NVFP4Tensor:
    """Dynamic NVFP4 quantisation of a bf16 [.., k] tensor (global scale from amax)."""
    _cuda(x)
    if x.dtype != torch.bfloat16:
        raise TypeError("quant_nvfp4 expects bf16 input")
    x2, m, k, ld = _rows(x)
    if m == 0:  # an empty batch: no codes, and the global scale of an all-zero tensor
        return NVFP4Tensor(torch.empty((0, k // 2), dtype=torch.uint8, device=x.device),
                           torch.empty((0,), dtype=torch.uint8, device=x.device),
                           torch.ones((1,), dtype=torch.float32, device=x.device), 0, k, hi_first)
    if amax_t is None:
        amax_t = amax(x2 if x2.is_contiguous() else x2.contiguous())
    codes = torch.empty((m, k // 2), dtype=torch.uint8, device=x.device)
    sf = torch.empty((sf_blocked_bytes(m, k),), dtype=torch.uint8, device=x.device)
    gs = torch.empty((1,), dtype=torch.float32, device=x.device)
    call("h3b_quant_nvfp4", x2.data_ptr(), m, k, ld, amax_t.data_ptr(), codes.data_ptr(), sf.data_ptr(),
         gs.data_ptr(), 1 if hi_first else 0, _stream(x))
    return NVFP4Tensor(codes, sf, gs, m, k, hi_first)


def gelu_amax_scan(y: torch.Tensor, ymax2: torch.Tensor) -> torch.Tensor:
    """ymax2[1] = max |bf16(gelu(y))| over fc1's bf16 output y when the bound
    from ymax2[0] = max(0, max y) does not settle max |u| (h3b_gelu_amax_scan);
    ymax2 is an fp32 [2] device tensor, ymax2[1] zero on entry."""
    _cuda(y, ymax2)
    if y.dtype != torch.bfloat16:
        raise TypeError("gelu_amax_scan expects bf16 input")
    if ymax2.dtype != torch.float32 or ymax2.numel() != 2 or not ymax2.is_contiguous():
        raise ValueError("ymax2 must be a contiguous fp32 tensor of 2 elements")
    y2, m, k, ld = _rows(y)
    call("h3b_gelu_amax_scan", y2.data_ptr(), m, k, ld, ymax2.data_ptr(), _stream(y))
    return ymax2


def quant_nvfp4_gelu(y: torch.Tensor, ymax2: torch.Tensor, *, hi_first: bool = False) -> NVFP4Tensor:
    """NVFP4 quantisation of u = bf16(gelu(y)) computed from fc1's bf16 output
    y on the fly (h3b_quant_nvfp4_gelu): the MLP activation fused with fc2's
    input quantisation.  ymax2: fp32 [2] from the fc1 GEMM's
    EPI_STORE_POSMAX max and gelu_amax_scan, max-reduced across ranks."""
    _cuda(y, ymax2)
    if y.dtype != torch.bfloat16:
        raise TypeError("quant_nvfp4_gelu expects bf16 input")
    if ymax2.dtype != torch.float32 or ymax2.numel() != 2 or not ymax2.is_contiguous():
        raise ValueError("ymax2 must be a contiguous fp32 tensor of 2 elements")
    y2, m, k, ld = _rows(y)
    if m == 0:
        raise ValueError("quant_nvfp4_gelu needs at least one row")
    codes = torch.empty((m, k // 2), dtype=torch.uint8, device=y.device)
    sf = torch.empty((sf_blocked_bytes(m, k),), dtype=torch.uint8, device=y.device)
    gs = torch.empty((1,), dtype=torch.float32, device=y.device)
    call("h3b_quant_nvfp4_gelu", y2.data_ptr(), m, k, ld, ymax2.data_ptr(), codes.data_ptr(), sf.data_ptr(),
         gs.data_ptr(), 1 if hi_first else 0, _stream(y))
    return NVFP4Tensor(codes, sf, gs, m, k, hi_first)


def swap_nibbles(u8: torch.Tensor) -> torch.Tensor:
    _cuda(u8)
    src = u8.contiguous()
    dst = torch.empty_like(src)
    call("h3b_nvfp4_swap_nibbles", src.data_ptr(), dst.data_ptr(), src.numel(), _stream(src))
    return dst


def gemm_nvfp4_seq2head(a: NVFP4Tensor, w: NVFP4Tensor, bias: Optional[torch.Tensor], recv_ptrs: Sequence[int],
                        rank: int, heads: int) -> None:
    """NVFP4 variant of gemm_i8_seq2head (both operands lo-first)."""
    if a.hi_first or w.hi_first:
        raise ValueError("gemm_nvfp4_seq2head needs tensor-core (lo-first) nibble order")
    _cuda(a.codes, w.codes, bias)
    arr = (ctypes.c_void_p * len(recv_ptrs))(*recv_ptrs)
    call("h3b_gemm_nvfp4_seq2head", a.codes.data_ptr(), a.sf.data_ptr(), a.gs.data_ptr(), w.codes.data_ptr(),
         w.sf.data_ptr(), w.gs.data_ptr(), _ptr(bias), ctypes.cast(arr, ctypes.c_void_p), len(recv_ptrs), rank,
         heads, a.rows, w.rows, a.k, _stream(a.codes))


def swiglu_interleave_perm(n: int, device=None) -> torch.Tensor:
    """Row order of an fc1 weight [n = 2*ffn, K] for EPI_SWIGLU: blocks of 32
    gate rows and the matching 32 up rows alternate, so new row 64b + j is
    gate row 32b + j and new row 64b + 32 + j is up row ffn + 32b + j
    (the halves of model/dit.py:120-129 x.chunk(2, dim=-1))."""
    if n % 64:
        raise ValueError("SwiGLU fc1 needs 2*ffn % 64 == 0")
    ffn = n // 2
    b = torch.arange(ffn // 32).repeat_interleave(32)
    j = torch.arange(32).repeat(ffn // 32)
    gate = 32 * b + j
    perm = torch.stack([gate.view(-1, 32), (ffn + gate).view(-1, 32)], dim=1).reshape(-1)
    return perm.to(device)


def _blocked_index(rows: int, ncols: int, device) -> torch.Tensor:
    """Flat offsets of every (row, scale column) of the 128x4 blocked scale
    layout (ops/nvfp4.py from_blocked), rows padded to 128: [rows_pad, ncols]."""
    rows_pad = (rows + 127) // 128 * 128
    r = torch.arange(rows_pad, device=device).view(-1, 1)
    c = torch.arange(ncols, device=device).view(1, -1)
    ncb = ncols // 4
    return ((r // 128) * ncb + c // 4) * 512 + (r % 32) * 16 + ((r % 128) // 32) * 4 + c % 4


def permute_blocked_rows(sf: torch.Tensor, rows: int, k: int, perm: torch.Tensor) -> torch.Tensor:
    """Reorders the rows of NVFP4 block scales kept in the blocked layout
    (row i of the result = row perm[i]); padding rows stay zero."""
    ncols = k // 16
    idx = _blocked_index(rows, ncols, sf.device)
    dense = sf.reshape(-1)[idx]
    full = torch.cat([perm.to(sf.device), torch.arange(rows, idx.shape[0], device=sf.device)])
    out = torch.zeros_like(sf.reshape(-1))
    out[idx.reshape(-1)] = dense[full].reshape(-1)
    return out.view_as(sf)


def gemm_nvfp4(a: NVFP4Tensor, w: NVFP4Tensor, bias: Optional[torch.Tensor] = None, *,
               epilogue: int = EPI_STORE, resid: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, row_sel: Optional[torch.Tensor] = None,
               amax_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = epi(a_gs*w_gs * A @ W^T + bias) in bf16; both operands lo-first."""
    if a.hi_first or w.hi_first:
        raise ValueError("gemm_nvfp4 needs tensor-core (lo-first) nibble order; repack with swap_nibbles")
    _cuda(a.codes, w.codes, bias, resid, gate, row_sel, amax_out, out)
    m, n, k = a.rows, w.rows, a.k
    if out is None:
        out = resid if epilogue == EPI_GATE_RES else torch.empty(
            (m, n // 2 if epilogue == EPI_SWIGLU else n), dtype=torch.bfloat16, device=a.codes.device)
    if m == 0:
        return out
    call("h3b_gemm_nvfp4_bf16", a.codes.data_ptr(), a.sf.data_ptr(), a.gs.data_ptr(), w.codes.data_ptr(),
         w.sf.data_ptr(), w.gs.data_ptr(), _ptr(bias), out.data_ptr(), out.stride(0), _ptr(resid), _ptr(gate),
         _gate_ld(gate), _ptr(row_sel), _ptr(amax_out), epilogue, m, n, k, _stream(a.codes))
    return out


# ----------------------------------------------------------------------------- attention


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
              amax_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Non-causal attention over token-major views q [Sq,H,128], k/v [Skv,H,128].

    Any strides with a unit last dimension are accepted (e.g. slices of a packed
    [S, 3, H, D] QKV buffer).  Returns o [Sq, H, 128] bf16.
    """
    _cuda(q, k, v, out, lse, amax_out)
    for t in (q, k, v):
        if t.dtype != torch.bfloat16 or t.dim() != 3 or t.shape[-1] != 128 or t.stride(-1) != 1:
            raise ValueError("attention expects bf16 [S, H, 128] views with unit last stride")
    if k.stride() != v.stride():
        raise ValueError("k and v must share strides")
    s_q, heads, d = q.shape
    s_kv = k.shape[0]
    if out is None:
        out = torch.empty((s_q, heads, d), dtype=torch.bfloat16, device=q.device)
    if s_q == 0:
        return out
    scale = d ** -0.5 if scale is None else float(scale)
    call("h3b_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), _ptr(amax_out),
         heads, s_q,
         s_kv, q.stride(0), q.stride(1), k.stride(0), k.stride(1), out.stride(0), out.stride(1), scale, _stream(q))
    return out


def attention_merge_lse(acc: torch.Tensor, acc_lse: torch.Tensor, blk: torch.Tensor, blk_lse: torch.Tensor, *,
                        first: bool, out: Optional[torch.Tensor] = None,
                        amax_out: Optional[torch.Tensor] = None) -> None:
    """Fold one key chunk's attention result (blk bf16 [S, H, 128], blk_lse
    [H, S]) into the running fp32 result acc / acc_lse (ops/fa_h3.py:141-156);
    first=True initialises them.  With out (bf16 [S, H, 128]) given, the merged
    rows go there (and max |out| into amax_out) instead of acc."""
    _cuda(acc, acc_lse, blk, blk_lse, out, amax_out)
    s, heads, d = blk.shape
    if d != 128 or acc.shape != blk.shape or acc_lse.shape != (heads, s) or blk_lse.shape != (heads, s):
        raise ValueError("attention_merge_lse: acc/blk [S, H, 128], lse [H, S]")
    if acc.dtype != torch.float32 or blk.dtype != torch.bfloat16 or acc_lse.dtype != torch.float32 \
            or blk_lse.dtype != torch.float32:
        raise ValueError("attention_merge_lse: acc fp32, blk bf16, lse fp32")
    tensors = (acc, acc_lse, blk, blk_lse) + ((out,) if out is not None else ())
    if not all(t.is_contiguous() for t in tensors):
        raise ValueError("attention_merge_lse: contiguous tensors only")
    if out is not None and (out.shape != blk.shape or out.dtype != torch.bfloat16):
        raise ValueError("attention_merge_lse: out bf16 [S, H, 128]")
    call("h3b_attention_merge_lse", acc.data_ptr(), acc_lse.data_ptr(), blk.data_ptr(), blk_lse.data_ptr(), s, heads,
         1 if first else 0, _ptr(out), _ptr(amax_out), _stream(blk))


def attention_head2seq(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o_ptrs: Sequence[int], *,
                       s_local: int, head0: int, total_heads: int, scale: Optional[float] = None,
                       amax_out: Optional[torch.Tensor] = None) -> None:
    """Attention over this rank's heads (q/k/v [S, H_local, 128] views of all
    S tokens) writing query row t into rank t // s_local's out-projection
    input [s_local, total_heads, 128] (o_ptrs[r]: device pointers valid in
    this process, rank order) at head head0 + h — the head->sequence Ulysses
    exchange fused into the epilogue."""
    _cuda(q, k, v, amax_out)
    for t in (q, k, v):
        if t.dtype != torch.bfloat16 or t.dim() != 3 or t.shape[-1] != 128 or t.stride(-1) != 1:
            raise ValueError("attention expects bf16 [S, H, 128] views with unit last stride")
    if k.stride() != v.stride():
        raise ValueError("k and v must share strides")
    s_q, heads, d = q.shape
    scale = d ** -0.5 if scale is None else float(scale)
    arr = (ctypes.c_void_p * len(o_ptrs))(*o_ptrs)
    call("h3b_attention_fwd_head2seq", q.data_ptr(), k.data_ptr(), v.data_ptr(), ctypes.cast(arr, ctypes.c_void_p),
         len(o_ptrs), s_local, head0, total_heads * d, d, _ptr(amax_out), heads, s_q, k.shape[0], q.stride(0),
         q.stride(1), k.stride(0), k.stride(1), scale, _stream(q))


def qk_rmsnorm_rope(q: torch.Tensor, k: Optional[torch.Tensor], q_weight: torch.Tensor,
                    k_weight: Optional[torch.Tensor], eps: float, pos: torch.Tensor, pos_offset: int,
                    inv_freq: torch.Tensor, n_t: int, n_h: int) -> None:
    """In-place RMSNorm + split-half RoPE of q (and k) [S, H, 128] views."""
    _cuda(q, k, q_weight, k_weight, pos, inv_freq)
    if k is not None and k.stride() != q.stride():
        raise ValueError("q and k must share strides")
    s, heads, d = q.shape
    call("h3b_qk_rmsnorm_rope", q.data_ptr(), _ptr(k), s, heads, q.stride(0), q.stride(1), q_weight.data_ptr(),
         _ptr(k_weight), eps, pos.data_ptr(), pos_offset, inv_freq.data_ptr(), n_t, n_h, _stream(q))


# ----------------------------------------------------------------------------- cross attention

_FLOAT16 = {torch.bfloat16: 0, torch.float16: 1}


def _fits(t: torch.Tensor) -> bool:
    """Whether a [B, S, H, D] tensor can be read in place: unit last stride,
    the others positive multiples of 8 elements (any along an axis of extent
    1), 16-byte aligned."""
    st = t.stride()
    if st[3] != 1 or t.data_ptr() & 15:
        return False
    for n, s in zip(t.shape, st[:3]):
        if n > 1 and (s <= 0 or s & 7):
            return False
    return True


def _check_qkv(name: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> tuple[int, int, int, int, int, int]:
    """Checks q [B, Sq, H, D] and k, v [B, Skv, Hkv, D]; returns (B, H, Hkv,
    D, Sq, Skv), the sizes as the C ABI takes them."""
    dtype = q.dtype
    if dtype not in _FLOAT16 or k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"{name} expects q, k and v of one type, bf16 or fp16")
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape or ks[0] != qs[0] or ks[3] != qs[3]:
        raise ValueError(f"{name} expects q [B, Sq, H, D], k and v [B, Skv, Hkv, D]")
    b, s_q, heads, d = qs
    _, s_kv, kv_heads, _ = ks
    if d not in (64, 128):
        raise ValueError(f"{name}: head dim {d}: the kernels are built for 64 and 128")
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{name}: {heads} query heads cannot share {kv_heads} key heads")
    return b, heads, kv_heads, d, s_q, s_kv


def _dense(t: torch.Tensor) -> torch.Tensor:
    """A copy that _fits (contiguous() keeps a contiguous tensor whose first
    element is not 16-byte aligned)."""
    return t.clone(memory_format=torch.contiguous_format)


def _kv_in_place(k: torch.Tensor, v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    if k.stride() != v.stride() or v.data_ptr() & 15 or not _fits(k):
        k, v = _dense(k), _dense(v)
    return k, v


def _kept_keys(name: str, k: torch.Tensor, kv_lens: Optional[torch.Tensor],
               key_mask: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Checks kv_lens / key_mask; returns the mask with unit key stride."""
    if kv_lens is not None and (kv_lens.dtype != torch.int32 or kv_lens.shape != k.shape[:1]
                                or not kv_lens.is_contiguous()):
        raise ValueError(f"{name}: kv_lens is an int32 tensor of one length per sample")
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape != k.shape[:2]:
            raise ValueError(f"{name}: key_mask is a bool [B, Skv] tensor (True: attended)")
        if key_mask.stride(1) != 1 or key_mask.stride(0) < 0:
            key_mask = key_mask.contiguous()
    return key_mask


def _scale(scale: Optional[float], d: int) -> float:
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("the softmax scale must be positive and finite")
    return scale


@functools.lru_cache(maxsize=512)
def _workspace_bytes(fn: str, device: int, *sizes: int) -> int:
    n = ctypes.c_int64(0)
    call(fn, *sizes, ctypes.addressof(n))
    return n.value


def _workspace(fn: str, t: torch.Tensor, *sizes: int) -> Optional[torch.Tensor]:
    n = _workspace_bytes(fn, t.get_device(), *sizes)
    return t.new_empty(n, dtype=torch.uint8) if n else None


def _check_lse(name: str, lse: Optional[torch.Tensor], q: torch.Tensor) -> None:
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (q.shape[0], q.shape[2], q.shape[1])
                            or not lse.is_contiguous()):
        raise ValueError(f"{name}: lse is a contiguous fp32 [B, H, Sq] tensor")


def _check_out(name: str, out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype != q.dtype or not _fits(out):
        raise ValueError(f"{name}: out has q's shape and type, unit last stride, strides of multiples of 8 and "
                         "16-byte alignment")
    return out


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [B, Sq, H, D] to an encoder's k, v [B, Skv, Hkv, D]
    (bf16 or fp16, D 64 or 128, H a multiple of Hkv): o [B, Sq, H, D].

    kv_lens (int32 [B], device) keeps the first keys of each sample, key_mask
    (bool [B, Skv], True: attended) any of them; with both, the keys that both
    keep.  Left-out keys and values are never used, whatever they hold.  A
    row without a kept key gives zeros (lse -inf).  lse, if given (fp32
    [B, H, Sq]), receives the log-sum-exps that cross_attention_bwd needs.
    Strided q, k and v are read in place (unit last stride, the others
    multiples of 8, k and v alike, as the halves of one projection); other
    layouts are copied first.  For gradients by autograd see
    ``attention.cross_attention``."""
    _cuda(q, k, v, kv_lens, key_mask, out, lse)
    sizes = _check_qkv("cross_attention", q, k, v)
    key_mask = _kept_keys("cross_attention", k, kv_lens, key_mask)
    _check_lse("cross_attention", lse, q)
    out = _check_out("cross_attention", out, q)
    if not _fits(q):
        q = _dense(q)
    k, v = _kv_in_place(k, v)
    ws = _workspace("h3b_cross_attention_workspace", q, *sizes)
    call("h3b_cross_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse),
         _FLOAT16[q.dtype], *sizes, *q.stride()[:3], *k.stride()[:3], *out.stride()[:3],
         _ptr(kv_lens), _ptr(key_mask), 0 if key_mask is None else key_mask.stride(0), _scale(scale, sizes[3]),
         _ptr(ws), 0 if ws is None else ws.numel(), _stream(q))
    return out


def cross_attention_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                        lse: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None,
                        key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None
                        ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of cross_attention for the gradient dout of its
    result out; lse and the other arguments as the forward call had them.
    Heads that share a key head add into its dk and dv; left-out keys get
    zeros.  Sums are fp32 in a fixed order (bit-reproducible)."""
    _cuda(dout, q, k, v, out, lse, kv_lens, key_mask)
    sizes = _check_qkv("cross_attention_bwd", q, k, v)
    if out.shape != q.shape or dout.shape != q.shape or out.dtype != q.dtype or dout.dtype != q.dtype:
        raise ValueError("cross_attention_bwd: out and dout have q's shape and type")
    key_mask = _kept_keys("cross_attention_bwd", k, kv_lens, key_mask)
    _check_lse("cross_attention_bwd", lse, q)
    q, out, dout = (t if _fits(t) else _dense(t) for t in (q, out, dout))
    k, v = _kv_in_place(k, v)
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    ws = _workspace("h3b_cross_attention_bwd_workspace", q, *sizes)
    call("h3b_cross_attention_bwd", dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
         lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _FLOAT16[q.dtype], *sizes,
         *dout.stride()[:3], *q.stride()[:3], *k.stride()[:3], *out.stride()[:3], _ptr(kv_lens), _ptr(key_mask),
         0 if key_mask is None else key_mask.stride(0), _scale(scale, sizes[3]), _ptr(ws),
         0 if ws is None else ws.numel(), _stream(q))
    return dq, dk, dv


# ----------------------------------------------------------------------------- 8-bit key/value cache

_KV8_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_KV8_READ = {**_FLOAT16, torch.float32: 2}


@dataclass
class KV8Cache:
    """Keys and values held in 8 bits: codes k, v [num_blocks, Hkv,
    block_tokens, D] (int8 or float8_e4m3fn) and one fp32 scale per block of
    tokens and head, [num_blocks, Hkv]; a value is code * scale.  The blocks
    of a sequence are named by a block table (int32 [B, max_blocks]), which
    the caller keeps beside the sequences' lengths (int32 [B])."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, num_blocks: int, kv_heads: int, head_dim: int, *, block_tokens: int = 64,
              dtype: torch.dtype = torch.int8, device=None) -> "KV8Cache":
        if dtype not in _KV8_CODES:
            raise TypeError("KV8Cache holds int8 or float8_e4m3fn codes")
        if block_tokens not in (32, 64, 128) or head_dim not in (64, 128):
            raise ValueError("KV8Cache: blocks of 32, 64 or 128 tokens, head dim 64 or 128")
        k, v = (torch.zeros((num_blocks, kv_heads, block_tokens, head_dim), dtype=torch.uint8, device=device).view(dtype)
                for _ in range(2))
        ks, vs = (torch.zeros((num_blocks, kv_heads), dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)

    @property
    def block_tokens(self) -> int:
        return self.k.shape[2]


def _check_cache(name: str, c: KV8Cache, table: torch.Tensor, lens: torch.Tensor) -> tuple[int, int, int, int, int, int]:
    """Checks a cache with its block table and lengths; returns (num_blocks,
    Hkv, block_tokens, D, B, max_blocks).  (Shapes are fetched once: building
    one costs a call of 20 us 0.2 us.)"""
    k, v, ks, vs = c.k, c.v, c.k_scale, c.v_scale
    _cuda(k, v, ks, vs, table, lens)
    dtype = k.dtype
    if dtype not in _KV8_CODES or v.dtype != dtype or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError(f"{name}: the cache holds int8 or float8_e4m3fn codes and fp32 scales")
    shape, scales = k.shape, ks.shape
    if len(shape) != 4 or v.shape != shape or vs.shape != scales or scales != shape[:2]:
        raise ValueError(f"{name}: codes [num_blocks, Hkv, block_tokens, D], scales [num_blocks, Hkv]")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{name}: the cache's tensors are contiguous")
    rows = table.shape
    if table.dtype != torch.int32 or len(rows) != 2 or not table.is_contiguous():
        raise ValueError(f"{name}: the block table is a contiguous int32 [B, max_blocks] tensor")
    if lens.dtype != torch.int32 or lens.shape != rows[:1] or not lens.is_contiguous():
        raise ValueError(f"{name}: lengths are an int32 tensor of one per sequence of the table")
    return (*shape, *rows)


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, *,
               new_lens: Optional[torch.Tensor] = None) -> None:
    """Quantises k, v [B, T, Hkv, D] (bf16 or fp16) into the cache behind the
    lens[b] tokens that each sequence holds (int32 [B], device; not updated
    here); rows behind the table's last block are dropped.  new_lens (int32
    [B]) appends the first new_lens[b] rows of a
    ragged batch.  A block that held tokens keeps the larger of its scale and
    the new rows' one, and its codes are rounded again if it grew.  Rows are
    expected finite: a scale ignores NaN, which int8 stores as code -127 (e4m3
    has a NaN), and an infinity makes the block's scale infinite."""
    nb, kv_heads, bt, d, b, max_blocks = _check_cache("kv8_append", cache, block_table, lens)
    _cuda(k, v, new_lens)
    dtype, rows = k.dtype, k.shape
    if dtype not in _FLOAT16 or v.dtype != dtype:
        raise TypeError("kv8_append expects bf16 or fp16 keys and values")
    if len(rows) != 4 or v.shape != rows or rows[0] != b or rows[2] != kv_heads or rows[3] != d:
        raise ValueError("kv8_append: k and v [B, T, Hkv, D] of the cache's heads")
    if new_lens is not None and (new_lens.dtype != torch.int32 or new_lens.shape != lens.shape
                                 or not new_lens.is_contiguous()):
        raise ValueError("kv8_append: new_lens is an int32 [B] tensor")
    k, v = _kv_in_place(k, v)
    call("h3b_kv8_append", k.data_ptr(), v.data_ptr(), _FLOAT16[dtype], b, rows[1], kv_heads, d,
         *k.stride()[:3], cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
         _KV8_CODES[cache.k.dtype], nb, bt, block_table.data_ptr(), max_blocks, lens.data_ptr(),
         _ptr(new_lens), _stream(k))


def kv8_read(cache: KV8Cache, block_table: torch.Tensor, lens: torch.Tensor, max_len: int, *,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The cache's values in the order of the tokens: k, v [B, max_len, Hkv,
    D] in dtype (bf16, fp16 or fp32), zero behind lens[b]."""
    nb, kv_heads, bt, d, b, max_blocks = _check_cache("kv8_read", cache, block_table, lens)
    if dtype not in _KV8_READ:
        raise TypeError("kv8_read writes bf16, fp16 or fp32")
    shape = (b, max_len, kv_heads, d)
    k, v = cache.k_scale.new_empty(shape, dtype=dtype), cache.k_scale.new_empty(shape, dtype=dtype)
    call("h3b_kv8_read", cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
         _KV8_CODES[cache.k.dtype], nb, kv_heads, bt, d, block_table.data_ptr(), max_blocks,
         lens.data_ptr(), b, max_len, k.data_ptr(), v.data_ptr(), _KV8_READ[dtype], _stream(cache.k))
    return k, v


def kv8_attention(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, lens: torch.Tensor, *,
                  causal: bool = False, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [B, Sq, H, D] (bf16 or fp16, H a multiple of the
    cache's heads) over the lens[b] tokens that each sequence's cache holds:
    o [B, Sq, H, D].  causal: the queries are the sequence's last Sq tokens
    (already appended), each sees the tokens up to its own.  Tokens of a block
    that the table does not name (an entry outside the pool) are left out.  A
    row that sees no token gives zeros (lse, fp32 [B, H, Sq] if given: -inf).
    Where a key head serves more than one tile of 256 query rows (of 33 tokens
    or more), the codes are written out as 16-bit numbers first, into a
    workspace of the table's width and twice the codes' bytes, unless that is
    more than 8 GB."""
    nb, kv_heads, bt, d, b, max_blocks = _check_cache("kv8_attention", cache, block_table, lens)
    _cuda(q, out, lse)
    dtype, rows = q.dtype, q.shape
    if dtype not in _FLOAT16:
        raise TypeError("kv8_attention expects bf16 or fp16 queries")
    if len(rows) != 4 or rows[0] != b or rows[3] != d or kv_heads == 0 or rows[2] % kv_heads:
        raise ValueError("kv8_attention expects q [B, Sq, H, D], H a multiple of the cache's heads")
    _, s_q, heads, _ = rows
    _check_lse("kv8_attention", lse, q)
    out = _check_out("kv8_attention", out, q)
    if not _fits(q):
        q = _dense(q)
    ws = _workspace("h3b_kv8_attention_workspace", q, b, heads, kv_heads, d, s_q, bt, max_blocks)
    call("h3b_kv8_attention", q.data_ptr(), out.data_ptr(), _ptr(lse), _FLOAT16[dtype], b, heads, kv_heads, d, s_q,
         *q.stride()[:3], *out.stride()[:3], cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
         cache.v_scale.data_ptr(), _KV8_CODES[cache.k.dtype], nb, bt, block_table.data_ptr(), max_blocks,
         lens.data_ptr(), 1 if causal else 0, _scale(scale, d), _ptr(ws), 0 if ws is None else ws.numel(), _stream(q))
    return out


# ----------------------------------------------------------------------------- rotary positions

_FLOATS = {**_FLOAT16, torch.float32: 2}


def _call_on(t: torch.Tensor, name: str, *args) -> None:
    """call() with t's device current (its streams and kernels belong to it)."""
    if t.get_device() == torch._C._cuda_getDevice():
        call(name, *args)
    else:
        with torch.cuda.device(t.device):
            call(name, *args)


def _workspace_on(fn: str, t: torch.Tensor, *sizes: int) -> torch.Tensor:
    """A workspace on t's device (its size may follow the SM count)."""
    device = t.get_device()
    if device == torch._C._cuda_getDevice():
        return t.new_empty(_workspace_bytes(fn, device, *sizes), dtype=torch.uint8)
    with torch.cuda.device(device):
        return t.new_empty(_workspace_bytes(fn, device, *sizes), dtype=torch.uint8)


def _one_device(name: str, t: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    device = t.get_device()
    for o in others:
        if o is not None and o.get_device() != device:
            _cuda(t, *others)
            raise ValueError(f"{name}: tensors on different devices")
    if device < 0 or not t.is_cuda:
        _cuda(t)


# 2^190 / 2 pi: a frequency's product with it keeps 64 bits of a turn and more
_TURN = 249757942369376157889070878929404173453413734678272424196


def _turns(radians: float) -> int:
    """radians / 2 pi as a multiple of 2^-64, modulo one turn, as an int64."""
    n, d = radians.as_integer_ratio()  # d is a power of two
    shift = 190 - 64 + d.bit_length() - 1
    t = ((n * _TURN + (1 << (shift - 1))) >> shift) & ((1 << 64) - 1)
    return t - (1 << 64) if t >> 63 else t


@dataclass(frozen=True, eq=False)
class Rotary:
    """The rotations of ``rotary``: how far a pair of channels turns at each
    position.  turns [pairs] (int64) holds radians / 2 pi as multiples of
    2^-64 (modulo one turn), so that whole turns of far positions drop out;
    sections are the pairs that each axis of the positions turns, in order;
    factor multiplies the turned channels.  Pairs are channels (i, i + R/2) of
    the first R = 2 * pairs of a head, or (2i, 2i + 1) if interleaved."""

    turns: torch.Tensor
    sections: tuple[int, ...]
    interleaved: bool = False
    factor: float = 1.0

    def __post_init__(self) -> None:
        if self.turns.dtype is not torch.int64 or self.turns.dim() != 1:
            raise TypeError("Rotary: turns is an int64 tensor [pairs]")
        object.__setattr__(self, "sections", tuple(self.sections))
        if not 1 <= len(self.sections) <= 3 or min(self.sections) < 0 or sum(self.sections) != self.turns.shape[0]:
            raise ValueError(f"Rotary: sections {self.sections} of {self.turns.shape[0]} pairs (one to three axes)")

    def to(self, device) -> "Rotary":
        """The same rotations on ``device`` (themselves, if they are there)."""
        turns = self.turns.to(device)
        return self if turns is self.turns else replace(self, turns=turns)

    @classmethod
    def from_frequencies(cls, frequencies: Sequence[float] | torch.Tensor, *, sections: Optional[Sequence[int]] = None,
                         interleaved: bool = False, factor: float = 1.0, device="cuda") -> "Rotary":
        """frequencies: radians a position of each pair (64-bit floats are
        used as they are)."""
        if isinstance(frequencies, torch.Tensor):
            frequencies = frequencies.detach().double().cpu().tolist()
        w = [float(f) for f in frequencies]
        if not all(math.isfinite(f) for f in w) or not math.isfinite(factor):
            raise ValueError("Rotary: frequencies and factor are finite")
        sections = (len(w),) if sections is None else tuple(int(n) for n in sections)
        return cls(torch.tensor([_turns(f) for f in w], dtype=torch.int64, device=device), sections, bool(interleaved),
                   float(factor))

    @classmethod
    def build(cls, dims: int | Sequence[int], *, theta: float = 10000.0, interleaved: bool = False,
              scaling: Optional[str] = None, scale: float = 1.0, trained_len: int = 0, fast: float = 32.0,
              slow: float = 1.0, factor: Optional[float] = None, device="cuda") -> "Rotary":
        """dims: the turned channels of a head (even), or those of each axis
        of the positions (up to three).  Pair i of an axis with d channels
        turns by theta^(-2i/d) radians a position, and for contexts ``scale``
        times longer than trained:

        * "linear": every frequency divided by scale;
        * "base": theta multiplied by scale^(d/(d-2)), which leaves the fastest
          pair as it is and divides the slowest one by scale;
        * "by_parts": pairs that make at least ``fast`` turns over trained_len
          positions stay, those of at most ``slow`` are divided by scale, those
          between by a share linear in the turns (a checkpoint made with a
          share linear in the pair's index takes ``from_frequencies``); the
          turned channels are multiplied by factor, 0.1 ln(scale) + 1 if None.

        Without a factor the others leave the channels' size as it is."""
        dims = (dims,) if isinstance(dims, int) else tuple(dims)
        if any(d < 0 or d & 1 for d in dims) or not dims:
            raise ValueError(f"Rotary: turned channels {dims} are even numbers")
        if scaling not in (None, "linear", "base", "by_parts"):
            raise ValueError(f"Rotary: scaling {scaling!r}")
        if not (theta > 0 and scale > 0 and math.isfinite(theta) and math.isfinite(scale)):
            raise ValueError("Rotary: theta and scale are positive and finite")
        if scaling == "by_parts" and not (trained_len > 0 and fast > slow):
            raise ValueError("Rotary: by_parts needs trained_len and fast > slow")
        if factor is None:
            factor = 0.1 * math.log(scale) + 1 if scaling == "by_parts" and scale > 1 else 1.0
        w = []
        for d in dims:
            base = theta * scale ** (d / (d - 2)) if scaling == "base" and d > 2 else theta
            for i in range(d // 2):
                f = base ** (-2 * i / d)
                if scaling == "linear":
                    f /= scale
                elif scaling == "by_parts":
                    turns = trained_len * f / (2 * math.pi)
                    keep = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
                    f = f / scale * (1 - keep) + f * keep
                w.append(f)
        return cls.from_frequencies(w, sections=[d // 2 for d in dims], interleaved=interleaved, factor=factor,
                                    device=device)


# h3b_rotary_args: one packed argument (35 by themselves took a third of a small call's time)
_ROTARY_ARGS = struct.Struct("@6P6q15q2qd4i")


def _rotary_out(out: Optional[torch.Tensor], x: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    if out.shape != x.shape or out.dtype != x.dtype or (out.shape[3] > 1 and out.stride(3) != 1):
        raise ValueError("rotary: an output has its input's shape and type and unit last stride")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError("rotary: an output has elements of its own")
    return out


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: Rotary, *,
           inverse: bool = False, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [B, S, H, D] and k [B, S, Hkv, D] (bf16, fp16 or fp32; k may be None)
    with the channels that ``rope`` pairs turned by the tokens' positions, the
    others as they are: (q, k), new tensors or q_out / k_out, which may be the
    inputs themselves and else overlap nothing.

    positions: int32 or int64, any value, [S] or [B, S] (any strides), with a
    last axis of one position per section where rope has several.  inverse
    turns the other way: with the same factor this is the transpose, which
    takes the gradients of the results to those of q and k
    (``attention.rotary`` does so under autograd).  Strided inputs are read in
    place (unit last stride; other layouts are copied).  Angles are off by
    |position| 2^-65 turns at most (2^-34 at 2^31, an eighth of a turn at
    2^62: frequencies are multiples of 2^-64), and what is left of them beside
    the nearest quarter turn is rounded to 32 bits (2^-28 of a turn at most);
    results are rounded once."""
    turns, sections, dtype = rope.turns, rope.sections, q.dtype
    _one_device("rotary", q, k, positions, turns, q_out, k_out)
    if dtype not in _FLOATS or (k is not None and k.dtype is not dtype):
        raise TypeError("rotary expects q and k of one type, bf16, fp16 or fp32")
    if q.dim() != 4:
        raise ValueError("rotary expects q [B, S, H, D] and k [B, S, Hkv, D]")
    b, s, heads, d = q.shape
    pairs, axes = turns.shape[0], len(sections)
    if 2 * pairs > d or d & 1:
        raise ValueError(f"rotary: {2 * pairs} turned channels of a head of {d} (an even number)")
    if positions.dtype is not torch.int32 and positions.dtype is not torch.int64:
        raise TypeError("rotary: positions are int32 or int64")
    shape, p = positions.shape, positions.stride()
    if axes == 1:
        p = (*p, 0)
    elif shape[-1:] == (axes,):
        shape = shape[:-1]
    else:
        shape = ()
    if shape == (s,):
        p = (0, *p)
    elif shape != (b, s):
        raise ValueError(f"rotary: positions [S] or [B, S]{f', each with {axes} axes' if axes > 1 else ''}")
    q_out = _rotary_out(q_out, q)
    qs, qos = q.stride(), q_out.stride()
    if qs[3] != 1:
        q = q.contiguous()
        qs = q.stride()
    if k is None:
        kv_heads, ks, kos, k_in, k_to = 0, (0, 0, 0, 1), (0, 0, 0, 1), 0, 0
    else:
        kb, kn, kv_heads, kd = k.shape if k.dim() == 4 else (-1, -1, -1, -1)
        if kb != b or kn != s or kd != d:
            raise ValueError("rotary expects q [B, S, H, D] and k [B, S, Hkv, D]")
        k_out = _rotary_out(k_out, k)
        ks, kos = k.stride(), k_out.stride()
        if ks[3] != 1:
            k = k.contiguous()
            ks = k.stride()
        k_in, k_to = k.data_ptr(), k_out.data_ptr()
    if not turns.is_contiguous():
        turns = turns.contiguous()
    args = _ROTARY_ARGS.pack(
        q.data_ptr(), k_in, q_out.data_ptr(), k_to, positions.data_ptr(), turns.data_ptr(), b, s, heads, kv_heads, d,
        2 * pairs, *qs[:3], *ks[:3], *qos[:3], *kos[:3], *p, sections[0], sections[1] if axes > 1 else 0, rope.factor,
        _FLOATS[dtype], rope.interleaved, positions.dtype is torch.int64, inverse)
    _call_on(q, "h3b_rotary", args, _stream(q))
    return q_out, None if k is None else k_out


# ----------------------------------------------------------------------------- layer norm


def _check_norm(name: str, x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor]) -> int:
    """Checks types and shapes; returns the code of the weights' type."""
    dtype = x.dtype
    if dtype not in _FLOATS:
        raise TypeError(f"{name} expects bf16, fp16 or fp32 input")
    last = x.shape[-1:]
    if not last or last[0] == 0:
        raise ValueError(f"{name}: an axis of at least one element is normalised")
    if weight is None:
        if bias is not None:
            raise ValueError(f"{name}: a bias comes with a weight")
        return _FLOATS[dtype]
    wdtype = weight.dtype
    if weight.shape != last or (wdtype is not dtype and wdtype is not torch.float32):
        raise ValueError(f"{name}: weight and bias are [{last[0]}] tensors of x's type or fp32")
    if bias is not None and (bias.shape != last or bias.dtype is not wdtype):
        raise ValueError(f"{name}: a bias has its weight's shape and type")
    return _FLOATS[wdtype]


def _check_stats(name: str, stats: Optional[torch.Tensor], m: int) -> None:
    if stats is not None and (stats.dtype != torch.float32 or stats.shape != (2, m) or not stats.is_contiguous()):
        raise ValueError(f"{name}: stats is a contiguous fp32 [2, rows] tensor")


# h3b_layer_norm_args, h3b_layer_norm_bwd_args
_NORM_ARGS, _NORM_BWD_ARGS = struct.Struct("@6P4qd2i"), struct.Struct("@9P6q2i")


def _flat_rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """x as rows of its last axis with unit column stride, and their stride."""
    if x.is_contiguous():
        return x, x.shape[-1]
    x2, _, _, ld = _rows(x)
    return x2, ld


def _packed(w: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return w if w is None or w.is_contiguous() else w.contiguous()


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, *, out: Optional[torch.Tensor] = None,
               stats: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x
    (bf16, fp16 or fp32; weight and bias of x's type or fp32): x's shape and
    type, contiguous, or ``out`` (contiguous).  stats, if given (fp32
    [2, rows]), receives each row's mean and 1 / sqrt(var + eps), which
    layer_norm_bwd needs.  out may be x itself and else overlaps nothing.  Rows
    with a unit last stride and one row stride are read in place, other layouts
    copied first.  A row that holds NaN or an infinity gives NaN.  For gradients
    by autograd see ``modules.layer_norm``."""
    _one_device("layer_norm", x, weight, bias, out, stats)
    wdtype = _check_norm("layer_norm", x, weight, bias)
    if not 0.0 <= eps < float("inf"):
        raise ValueError("layer_norm: eps is not negative and finite")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("layer_norm: out is a contiguous tensor of x's shape and type")
    n = x.shape[-1]
    m = x.numel() // n
    _check_stats("layer_norm", stats, m)
    if m == 0:
        return out
    x2, ld = _flat_rows(x)
    weight, bias = _packed(weight), _packed(bias)
    at = 0 if stats is None else stats.data_ptr()
    args = _NORM_ARGS.pack(x2.data_ptr(), 0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
                           out.data_ptr(), at, at and at + 4 * m, m, n, ld, n, eps, _FLOATS[x.dtype], wdtype)
    _call_on(x, "h3b_layer_norm_fwd", args, _stream(x))
    return out


def layer_norm_bwd(dout: torch.Tensor, x: torch.Tensor, stats: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                   weight_grad: bool = True, bias_grad: bool = True
                   ) -> tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients (dx, dweight, dbias) of layer_norm for the gradient dout of
    its result; x, stats and weight as the forward call had them.  dweight and
    dbias have the weight's type, and are None without a weight or where they
    are not asked for.  Sums are fp32 in a fixed order (bit-reproducible)."""
    _one_device("layer_norm_bwd", dout, x, stats, weight)
    wdtype = _check_norm("layer_norm_bwd", x, weight, None)
    if dout.shape != x.shape or dout.dtype != x.dtype:
        raise ValueError("layer_norm_bwd: dout has x's shape and type")
    n = x.shape[-1]
    m = x.numel() // n
    _check_stats("layer_norm_bwd", stats, m)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    weight = _packed(weight)
    new = torch.zeros_like if m == 0 else torch.empty_like
    dw = new(weight) if weight is not None and weight_grad else None
    db = new(weight) if weight is not None and bias_grad else None
    if m == 0:
        return dx, dw, db
    x2, ldx = _flat_rows(x)
    dout2, lddy = _flat_rows(dout)
    ws = None
    if dw is not None or db is not None:
        ws = _workspace_on("h3b_layer_norm_bwd_workspace", x, m, n)
    at = stats.data_ptr()
    args = _NORM_BWD_ARGS.pack(
        dout2.data_ptr(), x2.data_ptr(), 0 if weight is None else weight.data_ptr(), at, at + 4 * m, dx.data_ptr(),
        0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(), 0 if ws is None else ws.data_ptr(), m, n,
        lddy, ldx, n, 0 if ws is None else ws.numel(), _FLOATS[x.dtype], wdtype)
    _call_on(x, "h3b_layer_norm_bwd", args, _stream(x))
    return dx, dw, db


# ----------------------------------------------------------------------------- orthogonalised updates


def orthogonalize(x: torch.Tensor, *, steps: int = 5,
                  coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Newton-Schulz steps toward the orthogonal factor of each matrix of x
    [..., m, n] (bf16, fp16 or fp32): from x / (|x| + eps), Frobenius norm,
    ``steps`` times X <- a X + (b G + c G G) X with G = X X^T (the transposed
    form where m > n, the same values).  With the default coefficients every
    singular value from about 0.002 of the norm up ends between 0.68 and 1.14.
    Returns a contiguous tensor of x's shape and type, or ``out`` (contiguous;
    x itself may be given).

    Products run in pairs of f16 planes (22 bits) with fp32 sums whatever the
    type, and the result is rounded once: it is as near as 32-bit arithmetic
    comes.  Elements of the iterates must stay below 64, which any coefficients
    that converge keep.  A zero matrix gives zeros (eps > 0); NaN or an
    infinity makes its matrix NaN (with no steps an infinity leaves zeros
    beside it).  The result is bit-reproducible.  Matrices with a unit last
    stride are read in place."""
    _one_device("orthogonalize", x, out)
    if x.dtype not in _FLOATS:
        raise TypeError("orthogonalize expects bf16, fp16 or fp32 matrices")
    if x.dim() < 2 or 0 in x.shape[-2:]:
        raise ValueError("orthogonalize expects matrices [..., m, n] of at least one element")
    if not isinstance(steps, int) or not 0 <= steps <= 1000:
        raise ValueError("orthogonalize: steps is an integer from 0 to 1000")
    a, b, c = (float(v) for v in coefficients)
    if not all(math.isfinite(v) for v in (a, b, c)) or not 0.0 <= eps < float("inf"):
        raise ValueError("orthogonalize: coefficients and eps are finite, eps not negative")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("orthogonalize: out is a contiguous tensor of x's shape and type")
    m, n = x.shape[-2:]
    x3 = x.reshape(-1, m, n)
    batch = x3.shape[0]
    if batch == 0:
        return out
    if n > 1 and x3.stride(2) != 1:
        x3 = x3.contiguous()
    ws = _workspace_on("h3b_orthogonalize_workspace", x, batch, m, n)
    _call_on(x, "h3b_orthogonalize", x3.data_ptr(), out.data_ptr(), _FLOATS[x.dtype], batch, m, n, x3.stride(0),
             x3.stride(1), steps, a, b, c, float(eps), ws.data_ptr(), ws.numel(), _stream(x))
    return out


# ----------------------------------------------------------------------------- block elementwise


def rmsnorm_modulate(x: torch.Tensor, weight: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float,
                     row_sel: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     amax_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """h = rmsnorm(x)*w*(1+scale[row_sel]) + shift[row_sel]; shift/scale are
    [rows, hidden] tables (strided views of the adaLN output are fine)."""
    _cuda(x, weight, shift, scale, row_sel, out, amax_out)
    x2, m, hidden, ld = _rows(x)
    if out is None:
        out = torch.empty((m, hidden), dtype=torch.bfloat16, device=x.device)
    if shift.stride() != scale.stride():
        raise ValueError("shift and scale tables must share strides")
    if out.stride(0) != ld:
        raise ValueError("out must share the row stride of x")
    call("h3b_rmsnorm_modulate", x2.data_ptr(), out.data_ptr(), m, hidden, ld, weight.data_ptr(), shift.data_ptr(),
         scale.data_ptr(), _gate_ld(shift), _ptr(row_sel), eps, _ptr(amax_out), _stream(x))
    return out


def rmsnorm_modulate_quant_i8(x: torch.Tensor, weight: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor,
                              eps: float, row_sel: Optional[torch.Tensor] = None, convrot_group: int = 0,
                              q_out: Optional[torch.Tensor] = None, scale_out: Optional[torch.Tensor] = None
                              ) -> tuple[torch.Tensor, torch.Tensor]:
    """rmsnorm_modulate(x, ...) followed by quant_i8_rows(h, convrot_group)
    in one kernel (h is never written): returns (q [m, hidden] int8,
    per-row scale [m] fp32), the same bits as the two calls."""
    _cuda(x, weight, shift, scale, row_sel, q_out, scale_out)
    x2, m, hidden, ld = _rows(x)
    if shift.stride() != scale.stride():
        raise ValueError("shift and scale tables must share strides")
    if convrot_group not in (0, 256):
        raise NotImplementedError(f"ConvRot group size {convrot_group}: this build rotates 256-column groups")
    q = q_out if q_out is not None else torch.empty((m, hidden), dtype=torch.int8, device=x.device)
    xs = scale_out if scale_out is not None else torch.empty(m, dtype=torch.float32, device=x.device)
    if q.shape != (m, hidden) or not q.is_contiguous() or xs.numel() != m:
        raise ValueError("rmsnorm_modulate_quant_i8: q [m, hidden] contiguous, scale [m]")
    call("h3b_rmsnorm_modulate_quant_i8", x2.data_ptr(), m, hidden, ld, weight.data_ptr(), shift.data_ptr(),
         scale.data_ptr(), _gate_ld(shift), _ptr(row_sel), eps, convrot_group, q.data_ptr(), xs.data_ptr(),
         _stream(x))
    return q, xs


def gate_residual(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor,
                  row_sel: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x += y * gate[row_sel] in place (bf16)."""
    _cuda(x, y, gate, row_sel)
    m, hidden = x.shape
    if y.stride() != x.stride():
        raise ValueError("x and y must share strides")
    call("h3b_gate_residual", x.data_ptr(), y.data_ptr(), m, hidden, x.stride(0), gate.data_ptr(), _gate_ld(gate),
         _ptr(row_sel), _stream(x))
    return x


# ----------------------------------------------------------------------------- reference-named entries


def rotate_activation(x: torch.Tensor, group_size: int) -> torch.Tensor:
    """ops/hadamard.py:35-44: x [..., K] times the regular Hadamard matrix in
    every group_size-column group (ConvRot's online rotation).  This build
    rotates 256-column groups, exactly in fp64 and rounded once to x's dtype;
    the reference's value comes from a 16-bit GEMM, which can differ from the
    exact one by a unit in the last place.  Runs the rotating quantiser and
    keeps its rotated rows."""
    if group_size != 256:
        raise NotImplementedError(f"ConvRot group size {group_size}: this build rotates 256-column groups")
    *lead, k = x.shape
    if k % group_size != 0:
        raise ValueError(f"K={k} not divisible by group_size={group_size}")
    x2 = x.reshape(-1, k)
    out = torch.empty(x2.shape, dtype=x.dtype, device=x.device)
    quant_i8_rows(x2, convrot_group=group_size, x_rot_out=out)
    return out.reshape(*lead, k)


def int8_convrot_linear(x: torch.Tensor, weight_i8: torch.Tensor, weight_scale: torch.Tensor,
                        bias: Optional[torch.Tensor] = None, *, convrot: bool = True, group_size: int = 256,
                        out_dtype: torch.dtype = torch.bfloat16, weight_layout: str = "nk") -> torch.Tensor:
    """ops/int8_convrot.py:114-209: y = W8A8(x) with x [..., K] cast to
    out_dtype, optionally ConvRot-rotated, quantised per row and multiplied
    by the [N, K] int8 weight with its per-channel scales (+ bias).

    The ``nk`` layout is the only one: the reference's ``kn`` / ``nz29`` are
    its NPU Cube packings.  The output is bf16 (the GEMM's epilogue rounds
    once to bf16; an fp16 result would round twice), so other out_dtypes are
    refused rather than approximated.  Non-CUDA tensors raise RuntimeError,
    as the reference does for non-NPU ones."""
    if weight_layout != "nk":
        raise ValueError(f"weight_layout {weight_layout!r}: the tcgen05 GEMM reads the [N, K] int8 weight as stored")
    if out_dtype != torch.bfloat16:
        raise NotImplementedError(f"out_dtype {out_dtype}: the INT8 GEMM writes bf16")
    *lead, k = x.shape
    x2 = x.reshape(-1, k).to(out_dtype)
    q, xs = quant_i8_rows(x2, convrot_group=group_size if convrot else 0)
    b = bias.to(device=x.device, dtype=torch.bfloat16) if bias is not None else None
    y = gemm_i8(q, xs, weight_i8, weight_scale.reshape(-1).to(device=x.device, dtype=torch.float32), b)
    return y.reshape(*lead, weight_i8.shape[0])
