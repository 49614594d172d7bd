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


@pytest.mark.parametrize("qdt", [BF16, F16])
@pytest.mark.parametrize("s_q", [1, 20, 100, 513])
def test_blocks_with_scales_of_zero(cuda, qdt, s_q):
    """A block whose scales are 0 (an empty cache's) holds keys and values of
    0: its tokens take their share of the weights like others."""
    from minixmax_h3_b200 import ops

    hkv, d = 2, 128
    g = torch.Generator(device=cuda).manual_seed(s_q)
    c, table = ops.KV8Cache.empty(3, hkv, d, device=cuda), ints([[0, 2, 1], [1, 0, 0]], cuda)
    c.k.copy_(torch.randint(-127, 128, c.k.shape, generator=g, device=cuda))
    c.v.copy_(torch.randint(-127, 128, c.v.shape, generator=g, device=cuda))
    c.k_scale[2], c.v_scale[2] = 0.01, 3.0
    lens = [150, 100]
    q, lse = torch.randn(2, s_q, 4, d, generator=g, device=cuda).to(qdt), torch.empty(2, 4, s_q, device=cuda)
    o = ops.kv8_attention(q, c, table, ints(lens, cuda), lse=lse)
    assert torch.allclose(lse[1], torch.full_like(lse[1], math.log(100)), atol=2e-5, rtol=2e-6)
    assert o[1].float().abs().max() < 1e-25
    check(o[:1], exact(q, c, table.cpu(), lens, False, 64)[:1], qdt)
    k = c.k[2].double() * 0.01
    s = torch.einsum("ihd,hjd->hij", q[0].double(), k.repeat_interleave(2, 0)) * d ** -0.5
    want = torch.logsumexp(torch.cat([s, torch.zeros(4, s_q, 86, dtype=s.dtype, device=cuda)], -1), -1)
    assert torch.allclose(lse[0].double(), want, atol=2e-5, rtol=2e-6)


@pytest.mark.parametrize("qdt", [BF16, F16])
@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("s_q,b,hkv", [(1, 110, 4), (130, 1, 4), (513, 1, 4)])
def test_long_tail_beside_a_dominant_token(cuda, qdt, dtype, s_q, b, hkv):
    """One token 17 to 18 nats above half a million equal ones: each of their
    weights is about 2^-25 of the first, their sum is not.  The dominant value
    is small (0 where a single row is asked for), so that the sum shows.  (The
    tail's blocks are one block, named again and again.)"""
    from minixmax_h3_b200 import ops

    blocks, bt, d = 8192, 64, 64
    n = blocks * bt
    c = ops.KV8Cache.empty(2, hkv, d, block_tokens=bt, dtype=dtype, device=cuda)
    one = torch.ones((), device=cuda)
    c.v.copy_((64 * one).to(dtype).expand(c.v.shape))
    c.k[0, :, 0], c.v[0, :, 0] = one.to(dtype), ((0 if s_q == 1 else 1) * one).to(dtype)
    c.k_scale.fill_(1.0), c.v_scale.fill_(1 / 64)
    table = torch.ones(b, blocks, dtype=torch.int32, device=cuda)
    table[:, 0] = 0
    gap = torch.tensor([17.0, 17.5, 18.0, 17.25], dtype=torch.float64)
    q = (gap / 8)[None, None, :, None].expand(b, s_q, hkv, d).to(cuda, qdt).contiguous()  # (exact in 8 bits)
    lse = torch.empty(b, hkv, s_q, device=cuda)
    o = ops.kv8_attention(q, c, table, ints([n] * b, cuda), lse=lse)
    top = torch.exp(gap)
    want = (top * (0 if s_q == 1 else 1 / 64) + n - 1) / (top + n - 1)
    check(o, want[None, None, :, None].expand(b, s_q, hkv, d), qdt)
    # (a running fp32 sum is off by 2^-24 a step at most: a warp may take every fourth tile of 32 keys)
    want = torch.log(top + n - 1)[None, :, None].expand(b, hkv, s_q)
    assert torch.allclose(lse.double().cpu(), want, atol=2e-5 + n / 128 * 2.0 ** -24, rtol=2e-6)


@pytest.mark.parametrize("qdt", [BF16, F16])
def test_nan_query_is_not_hidden(cuda, qdt):
    from minixmax_h3_b200 import ops

    lens = [90]
    c, table = filled(cuda, lens, 2, 64, 64, torch.int8)
    for s_q in (1, 40, 513):
        q = torch.randn(1, s_q, 4, 64, generator=torch.Generator(device=cuda).manual_seed(0), device=cuda).to(qdt)
        q[0, s_q - 1, 2, 7] = math.nan
        lse = torch.empty(1, 4, s_q, device=cuda)
        o = ops.kv8_attention(q, c, table, ints(lens, cuda), lse=lse)
        bad = torch.zeros(1, s_q, 4, dtype=torch.bool, device=cuda)
        bad[0, s_q - 1, 2] = True
        assert torch.isnan(o[bad]).all() and torch.isfinite(o[~bad]).all()
        assert torch.equal(torch.isnan(lse.transpose(1, 2)), bad)


@pytest.mark.parametrize("s_q", [1, 130, 513])
def test_lengths_beyond_the_table(cuda, s_q):
    """Lengths beyond the table are cut to it: every row is as with the
    table's own length, absent blocks among them."""
    from minixmax_h3_b200 import ops

    lens = [500, 320, 200]
    c, table = filled(cuda, lens, 2, 128, 64, torch.int8, max_blocks=8)
    table[0, 1], table[0, 4] = -1, 10 ** 6
    table[1] = -5
    q = torch.randn(3, s_q, 4, 128, generator=torch.Generator(device=cuda).manual_seed(0), device=cuda).to(BF16)
    o = ops.kv8_attention(q, c, table, ints([10 ** 9, 10 ** 9, 200], cuda))
    check(o, exact(q, c, table.cpu(), [512, 512, 200], False, 64), BF16)
    assert (o[1] == 0).all()
    assert torch.equal(o, ops.kv8_attention(q, c, table, ints([512, 512, 200], cuda)))


@pytest.mark.parametrize("s_q", [1, 300])
def test_step_in_a_cuda_graph(cuda, s_q):
    """Append, attention and read of a step, and a training step, captured
    once and replayed on other inputs: the same bits as the calls."""
    from minixmax_h3_b200 import ops

    hkv, d, lens = 2, 128, ints([100, 40], cuda)
    g = torch.Generator(device=cuda).manual_seed(0)

    def inputs():
        return [torch.randn(2, s_q, n, d, generator=g, device=cuda).to(F16) for n in (4, hkv, hkv, 4)]

    c0, table = filled(cuda, [100 + s_q, 40 + s_q], hkv, d, 64, torch.int8)

    def step(cache, q, k, v, do):
        ops.kv8_append(cache, k, v, table, lens)
        o = ops.kv8_attention(q, cache, table, lens + s_q, causal=True)
        lse = torch.empty(2, 4, s_q, device=cuda)
        p = ops.cross_attention(q, k, v, lse=lse)
        return (o, *ops.kv8_read(cache, table, lens + s_q, 100 + s_q), p, lse,
                *ops.cross_attention_bwd(do, q, k, v, p, lse))

    def fresh():
        return ops.KV8Cache(*(t.clone() for t in (c0.k, c0.v, c0.k_scale, c0.v_scale)))

    held, cache = inputs(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh(), *held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, *held)
    for _ in range(2):
        new = inputs()
        for a, b in zip(held, new):
            a.copy_(b)
        for a, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), (c0.k, c0.v, c0.k_scale, c0.v_scale)):
            a.copy_(b)
        graph.replay()
        for a, b in zip(got, step(fresh(), *new)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("s_q", [1, 300])
def test_other_stream_of_the_cache(cuda, s_q):
    from minixmax_h3_b200 import ops

    lens = ints([100], cuda)
    c, table = filled(cuda, [100 + s_q], 2, 64, 64, torch.float8_e4m3fn)
    g = torch.Generator(device=cuda).manual_seed(0)
    q, k, v = (torch.randn(1, s_q, n, 64, generator=g, device=cuda).to(BF16) for n in (4, 2, 2))

    def step(cache):
        ops.kv8_append(cache, k, v, table, lens)
        return (ops.kv8_attention(q, cache, table, lens + s_q), *ops.kv8_read(cache, table, lens + s_q, 100 + s_q))

    caches = [ops.KV8Cache(*(t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale))) for _ in range(2)]
    want = step(caches[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(caches[1])
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("s_q", [1, 130, 513])
def test_scales_of_left_out_blocks(cuda, dtype, bad, s_q):
    """Scales of blocks that hold no attended token (absent ones, ones behind
    the length) may be anything, like their codes."""
    from minixmax_h3_b200 import ops

    lens, bt = [300, 70], 32
    c, table = filled(cuda, [320, 96], 2, 64, bt, dtype, max_blocks=12)
    table[0, 3], table[1, 5] = -1, 10 ** 6
    used = torch.cat([table[0, :10], table[1, :3]])
    spare = torch.tensor([i for i in range(c.k.shape[0]) if i not in used.tolist()], device=cuda)
    assert len(spare) == 1  # block table[0, 3] was
    table[0, 10:], table[1, 3] = spare[0].int(), spare[0].int()
    pool = ops.KV8Cache(*(torch.cat([t[spare], t]) for t in (c.k, c.v, c.k_scale, c.v_scale)))  # block 0 is spare too
    table = torch.where((table >= 0) & (table < 10 ** 6), table + 1, table)
    for t in (pool.k_scale, pool.v_scale):
        t[0], t[spare + 1] = bad, bad
    q = torch.randn(2, s_q, 4, 64, generator=torch.Generator(device=cuda).manual_seed(0), device=cuda).to(BF16)
    for causal in (False, True):
        o = ops.kv8_attention(q, pool, table, ints(lens, cuda), causal=causal)
        check(o, exact(q, pool, table.cpu(), lens, causal, bt), BF16)
