"""GPU: calls from a thread that has not touched CUDA yet.  Such a thread (a
server's worker, autograd's) has no current context until its first call of
the CUDA runtime, and an allocation served from the cache is none."""
from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def in_new_thread(fn):
    out = []

    def work():
        try:
            out.append(fn())
        except Exception as e:  # noqa: BLE001 (raised again below)
            out.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    if isinstance(out[0], Exception):
        raise out[0]
    return out[0]


def calls(cuda):
    from minixmax_h3_b200 import ops

    g = torch.Generator(device=cuda).manual_seed(0)
    q, k, v = (torch.randn(1, n, 2, 128, generator=g, device=cuda).to(torch.bfloat16) for n in (200, 300, 300))
    lse = torch.empty(1, 2, 200, device=cuda)
    o = ops.cross_attention(q, k, v, lse=lse)
    cache = ops.KV8Cache.empty(5, 2, 128, device=cuda)
    table, lens = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([[0, 1, 2, 3, 4]], [300]))
    ops.kv8_append(cache, k, v, table, torch.zeros_like(lens))
    return {
        "attention": lambda: ops.attention(q[0], k[0], v[0]),
        "cross_attention, rows": lambda: ops.cross_attention(q[:, :1], k, v),
        "cross_attention, tiles": lambda: ops.cross_attention(q, k, v),
        "cross_attention_bwd": lambda: torch.cat([t.flatten() for t in ops.cross_attention_bwd(o, q, k, v, o, lse)]),
        "kv8_attention, rows": lambda: ops.kv8_attention(q[:, :1], cache, table, lens),
        "kv8_attention, tiles": lambda: ops.kv8_attention(q, cache, table, lens),
    }


@pytest.mark.parametrize("name", ["attention", "cross_attention, rows", "cross_attention, tiles", "cross_attention_bwd",
                                  "kv8_attention, rows", "kv8_attention, tiles"])
def test_first_call_of_a_thread(cuda, name):
    fn = calls(cuda)[name]
    want = fn()
    fn()  # (two results at a time: what the thread allocates is in the cache)
    torch.cuda.synchronize()
    assert torch.equal(in_new_thread(fn), want)


def test_backward_as_the_first_call_of_autograds_thread(cuda):
    """A process of its own: the thread that runs backward passes is new."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from minixmax_h3_b200.attention import cross_attention
q, k, v = (torch.randn(2, n, 2, 64, device="cuda").to(torch.bfloat16).requires_grad_() for n in (80, 60, 60))
do = torch.randn(2, 80, 2, 64, device="cuda").to(torch.bfloat16)
big = torch.empty(1 << 24, device="cuda"); del big
o = cross_attention(q, k, v)
keep = [torch.empty_like(q) for _ in range(8)]; del keep
grads = torch.autograd.grad(o, (q, k, v), do)
torch.cuda.synchronize()
assert all(torch.isfinite(g).all() for g in grads)
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=Path(__file__).resolve().parents[1], timeout=300)
