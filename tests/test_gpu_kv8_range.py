"""GPU: the 8-bit cache where sizes of values are unusual (zero queries, keys
and scales, weights far apart), every row of absent and cut sequences, and the
cache's step in a CUDA graph."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cross_attention import check
from test_gpu_kv8 import CODES, exact, filled, ints

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("qdt", [BF16, F16])
@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("s_q,causal", [(1, False), (1, True), (20, False), (20, True), (70, True), (513, False)])
def test_zero_queries_and_keys(cuda, qdt, dtype, s_q, causal):
    """A padded query over zero keys: every score is 0, so the result is the
    mean of the values that the row sees."""
    from minixmax_h3_b200 import ops

    n, hkv, d = 77, 2, 64
    g = torch.Generator(device=cuda).manual_seed(s_q)
    v = torch.randn(1, n, hkv, d, generator=g, device=cuda).to(qdt)
    c, table = ops.KV8Cache.empty(2, hkv, d, dtype=dtype, device=cuda), ints([[1, 0]], cuda)
    ops.kv8_append(c, torch.zeros_like(v), v, table, ints([0], cuda))
    q, lse = torch.zeros(1, s_q, 4, d, dtype=qdt, device=cuda), torch.empty(1, 4, s_q, device=cuda)
    o = ops.kv8_attention(q, c, table, ints([n], cuda), causal=causal, lse=lse)
    check(o, exact(q, c, table.cpu(), [n], causal, 64), qdt)
    seen = (n - s_q + 1 + torch.arange(s_q)).clamp(min=0) if causal else torch.full((s_q,), n)
    assert torch.allclose(lse.double().cpu(), torch.log(seen.double())[None, None].expand(1, 4, s_q), atol=2e-5, rtol=2e-6)
