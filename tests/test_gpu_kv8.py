"""GPU: the 8-bit key/value cache (append, read, attention) against its
definition: append and read exactly, attention against 64 bits with the bound
of test_gpu_cross_attention (the codes and scales are exact there)."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cross_attention import check

pytestmark = pytest.mark.gpu

CODES = [torch.int8, torch.float8_e4m3fn]


def top_of(dtype):
    return 127.0 if dtype == torch.int8 else 448.0


def to_code_values(y, dtype):
    """fp32 quotients -> the code values they are rounded to."""
    if dtype == torch.int8:
        return y.round().clamp(-127, 127)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn).float()


class Model:
    """The cache by its definition, on the CPU: per block and head a scale and
    the code values of its rows."""

    def __init__(self, nb, hkv, bt, d, dtype):
        self.dtype, self.bt = dtype, bt
        self.code = torch.zeros(2, nb, hkv, bt, d)
        self.scale = torch.zeros(2, nb, hkv)

    def append(self, kv, table, lens, counts):
        for which in range(2):
            x = kv[which].float().cpu()
            for b in range(x.shape[0]):
                lo, hi = lens[b], lens[b] + counts[b]
                for j in range(lo // self.bt, (hi + self.bt - 1) // self.bt):
                    if hi <= lo or j >= table.shape[1] or not 0 <= table[b, j] < self.code.shape[1]:
                        continue
                    i, s = int(table[b, j]), j * self.bt
                    first, last = max(lo - s, 0), min(hi - s, self.bt)
                    rows = x[b, s + first - lo:s + last - lo].transpose(0, 1)  # [hkv, n, d]
                    most = rows.abs().amax((1, 2)).clamp(min=1e-12) / torch.tensor(top_of(self.dtype))
                    old = self.scale[which, i].clone()
                    new = torch.maximum(old, most) if first else most
                    held = self.code[which, i, :, :first] * old[:, None, None]
                    self.code[which, i] = 0
                    self.code[which, i, :, :first] = to_code_values(held / new[:, None, None], self.dtype)
                    self.code[which, i, :, first:last] = to_code_values(rows / new[:, None, None], self.dtype)
                    self.scale[which, i] = new

    def read(self, table, lens, max_len):
        b, hkv, d = table.shape[0], self.code.shape[2], self.code.shape[4]
        out = torch.zeros(2, b, max_len, hkv, d)
        for which in range(2):
            for i in range(b):
                for t in range(min(int(lens[i]), max_len, table.shape[1] * self.bt)):
                    j = int(table[i, t // self.bt])
                    if 0 <= j < self.code.shape[1]:
                        out[which, i, t] = self.code[which, j, :, t % self.bt] * self.scale[which, j, :, None]
        return out


def new_cache(cuda, nb, hkv, d, bt, dtype):
    from minixmax_h3_b200 import ops

    c = ops.KV8Cache.empty(nb, hkv, d, block_tokens=bt, dtype=dtype, device=cuda)
    for t in (c.k, c.v):  # a pool is not clean: whatever it holds is not used
        t.view(torch.uint8).fill_(0x7f)
    return c


def ints(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("bt,d,src", [(32, 64, torch.float16), (64, 128, torch.bfloat16), (128, 128, torch.float16)])
def test_append_and_read(cuda, dtype, bt, d, src):
    """Several appends of odd lengths, starting inside and at blocks, growing
    and not growing a block's scale; a ragged batch; an absent block."""
    from minixmax_h3_b200 import ops

    hkv, b = 3, 3
    g = torch.Generator(device=cuda).manual_seed(bt + d)
    table = ints([[4, 0, 7, 5, 9], [2, 11, 3, -1, 1], [6, 8, 10, 99, -7]], cuda)
    c, m = new_cache(cuda, 12, hkv, d, bt, dtype), Model(12, hkv, bt, d, dtype)
    lens = [0, 0, 0]
    for n, counts, size in ((bt + 5, None, 1.0), (1, [1, 0, 1], 3.0), (7, [7, 3, 0], 0.2), (2 * bt, None, 1.5), (1, None, 9.0)):
        kv = [(size * torch.randn(b, n, hkv, d, generator=g, device=cuda)).to(src) for _ in range(2)]
        kv[1][:, 0] = 0
        counts = [n] * b if counts is None else counts
        ops.kv8_append(c, kv[0], kv[1], table, ints(lens, cuda), new_lens=ints(counts, cuda) if n > 1 else None)
        if n == 1:
            counts = [1] * b
        m.append([t.cpu() for t in kv], table.cpu(), lens, counts)
        lens = [x + y for x, y in zip(lens, counts)]
        want = m.read(table.cpu(), lens, 5 * bt)
        got = ops.kv8_read(c, table, ints(lens, cuda), 5 * bt, dtype=torch.float32)
        for which in range(2):
            assert torch.equal(got[which].cpu(), want[which]), (n, which)
    for dt in (torch.bfloat16, torch.float16):
        got = ops.kv8_read(c, table, ints(lens, cuda), 3 * bt + 1, dtype=dt)
        assert all(torch.equal(got[i].cpu(), want[i, :, :3 * bt + 1].to(dt)) for i in range(2))


def filled(cuda, lens, hkv, d, bt, dtype, seed=0, max_blocks=None):
    """A cache whose sequences hold `lens` tokens, blocks in random order;
    blocks of very different magnitude."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    per = [-(-n // bt) for n in lens]
    nb = max(1, sum(per))
    c = new_cache(cuda, nb, hkv, d, bt, dtype)
    codes = torch.randint(-127, 128, (2, nb, hkv, bt, d), generator=g, device=cuda).float()
    if dtype != torch.int8:
        codes = codes * 3.0
    c.k.copy_(codes[0].to(dtype)), c.v.copy_(codes[1].to(dtype))
    size = torch.exp(2 * torch.randn(2, nb, hkv, generator=g, device=cuda)) / top_of(dtype)
    c.k_scale.copy_(size[0].clamp(max=2 / top_of(dtype))), c.v_scale.copy_(size[1])
    ids = torch.randperm(nb, generator=g, device=cuda).to(torch.int32)
    table = torch.full((len(lens), max_blocks or max(1, max(per))), -1, dtype=torch.int32, device=cuda)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = ids[at:at + n]
        at += n
        if n and lens[b] % bt:  # rows behind the last token may hold anything, NaN included
            for t in (c.k, c.v):
                t.view(torch.uint8)[table[b, n - 1].long(), :, lens[b] % bt:] = 0x7f
    return c, table


def exact(q, c, table, lens, causal, bt):
    q = q.double().cpu()
    b, s_q, h, d = q.shape
    hkv = c.k.shape[1]
    out = torch.zeros_like(q)
    for i in range(b):
        ks, vs, at = [], [], []
        for t in range(lens[i]):
            j = int(table[i, t // bt])
            if 0 <= j < c.k.shape[0]:
                ks.append((j, t % bt))
                at.append(t)
        if not ks:
            continue
        jj, tt = (torch.tensor(x) for x in zip(*ks))
        k, v = (x.float().cpu().double()[jj, :, tt] * s.double().cpu()[jj][..., None]
                for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)))  # [n, hkv, d]
        at = torch.tensor(at)
        for head in range(h):
            g = head * hkv // h
            s = q[i, :, head] @ k[:, g].T * d ** -0.5
            if causal:
                s = s.masked_fill(at[None] > lens[i] - s_q + torch.arange(s_q)[:, None], -math.inf)
            none = (s == -math.inf).all(-1, keepdim=True)
            p = torch.softmax(s.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
            out[i, :, head] = p @ v[:, g]
    return out


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("qdt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,d,bt,s_q,causal", [
    (1, 1, 128, 64, 1, False), (4, 4, 64, 32, 1, False), (8, 2, 128, 128, 1, True), (8, 1, 64, 64, 3, True),
    (6, 3, 128, 32, 20, False), (2, 2, 128, 64, 63, True), (2, 1, 64, 64, 64, False), (4, 2, 128, 32, 65, True),
    (2, 2, 128, 128, 130, False), (2, 1, 64, 32, 257, True), (3, 3, 128, 64, 300, True)])
def test_attention(cuda, dtype, qdt, h, hkv, d, bt, s_q, causal):
    from minixmax_h3_b200 import _lib, ops

    lens = [300, 1, bt, 0, 3 * bt + 7, 129]  # shorter than s_q among them: causal rows without a key
    c, table = filled(cuda, lens, hkv, d, bt, dtype, seed=s_q)
    g = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn(len(lens), s_q, h, d, generator=g, device=cuda).to(qdt)
    lse = torch.empty(len(lens), h, s_q, device=cuda)
    o = ops.kv8_attention(q, c, table, ints(lens, cuda), causal=causal, lse=lse)
    want = exact(q, c, table.cpu(), lens, causal, bt)
    check(o, want, qdt)
    empty = (want.abs().sum(-1) == 0).permute(0, 2, 1)
    assert torch.equal((lse == -math.inf).cpu(), empty)
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.parametrize("s_q", [1, 130])
def test_absent_blocks(cuda, s_q):
    """Blocks that the table does not name (evicted ones) are left out, all of
    a sequence's too; lengths beyond the table are cut."""
    from minixmax_h3_b200 import ops

    lens = [500, 320, 200]
    c, table = filled(cuda, lens, 2, 128, 64, torch.int8, max_blocks=8)
    table[0, 1], table[0, 4] = -1, 10 ** 6
    table[1] = -5
    q = torch.randn(3, s_q, 4, 128, generator=torch.Generator(device=cuda).manual_seed(0), device=cuda).to(torch.bfloat16)
    o = ops.kv8_attention(q, c, table, ints([10 ** 9, 320, 200], cuda))
    want = exact(q, c, table.cpu(), [512, 320, 200], False, 64)
    # sequence 0: its last block's rows behind token 500 count now (its table names 8 blocks of 64)
    check(o[1:], want[1:], torch.bfloat16)
    assert (o[1] == 0).all()
    o = ops.kv8_attention(q, c, table, ints(lens, cuda))
    check(o, exact(q, c, table.cpu(), lens, False, 64), torch.bfloat16)


def test_long_and_split(cuda):
    """A context long enough to be split, one and many rows, against the dense
    kernel on the values read back."""
    from minixmax_h3_b200 import ops

    lens = [9001]
    c, table = filled(cuda, lens, 2, 128, 64, torch.float8_e4m3fn)
    c.k_scale.fill_(0.004), c.v_scale.fill_(0.01)
    g = torch.Generator(device=cuda).manual_seed(0)
    for s_q in (1, 100, 513):
        q = torch.randn(1, s_q, 4, 128, generator=g, device=cuda).to(torch.float16)
        o = ops.kv8_attention(q, c, table, ints(lens, cuda))
        k, v = ops.kv8_read(c, table, ints(lens, cuda), lens[0], dtype=torch.float32)
        s = torch.einsum("ihd,jhd->hij", q[0].double(), k[0].double().repeat_interleave(2, 1)) * 128 ** -0.5
        want = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[0].double().repeat_interleave(2, 1))[None]
        check(o, want, torch.float16)


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 bytes a side whose last blocks are used."""
    from minixmax_h3_b200 import ops

    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    hkv, d, bt = 8, 128, 128
    nb = (1 << 32) // (hkv * d * bt) + 40
    k = torch.zeros(nb, hkv, bt, d, dtype=torch.int8, device=cuda)
    c = ops.KV8Cache(k, torch.zeros_like(k), torch.ones(nb, hkv, device=cuda), torch.ones(nb, hkv, device=cuda))
    table = ints([[nb - 1, nb - 3]], cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    x = [torch.randn(1, 200, hkv, d, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2)]
    ops.kv8_append(c, x[0], x[1], table, ints([0], cuda))
    kk, vv = ops.kv8_read(c, table, ints([200], cuda), 200, dtype=torch.float32)
    assert (kk - x[0].float()).abs().max() < 0.03 and (vv - x[1].float()).abs().max() < 0.03  # half a step of ~5/127
    for s_q in (1, 70):
        q = torch.randn(1, s_q, hkv, d, generator=g, device=cuda).to(torch.bfloat16)
        check(ops.kv8_attention(q, c, table, ints([200], cuda)), exact(q, c, table.cpu(), [200], False, bt), torch.bfloat16)


def test_custom_operators(cuda):
    import minixmax_h3_b200.torch_ops  # noqa: F401
    from minixmax_h3_b200 import ops

    c, table = new_cache(cuda, 2, 2, 64, 64, torch.int8), ints([[0], [1]], cuda)
    x = torch.randn(2, 9, 2, 64, device=cuda).to(torch.bfloat16)
    args = (c.k, c.v, c.k_scale, c.v_scale, table)
    torch.ops.h3b.kv8_append(x, x, *args, ints([0, 0], cuda), None)
    q = torch.randn(2, 1, 4, 64, device=cuda).to(torch.bfloat16)
    o = torch.ops.h3b.kv8_attention(q, *args, ints([9, 9], cuda), False, None)
    assert torch.equal(o, ops.kv8_attention(q, c, table, ints([9, 9], cuda)))


@pytest.mark.parametrize("axis", [0, 1, 2])
def test_append_any_stride_along_an_axis_of_one(cuda, axis):
    """The stride of an axis of extent 1 is never used, whatever it is."""
    from minixmax_h3_b200 import ops

    shape = [2, 5, 3, 64]
    shape[axis] = 1
    b, n, hkv, d = shape
    src = torch.randn(2, *shape, device=cuda).to(torch.bfloat16)
    odd = [list(t.stride()) for t in src]
    for st in odd:
        st[axis] = 517
    views = [torch.as_strided(src, shape, st, i * src[0].numel()) for i, st in enumerate(odd)]
    table, lens = ints([[i] for i in range(b)], cuda), ints([0] * b, cuda)
    got = []
    for k, v in ((src[0], src[1]), views):
        c = ops.KV8Cache.empty(2, hkv, d, device=cuda)
        ops.kv8_append(c, k, v, table, lens)
        got.append((c.k, c.v, c.k_scale, c.v_scale))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert got[0][0].any() and got[0][1].any()


def test_nothing_to_do(cuda):
    """Appends of no rows, reads of no tokens and calls of no sequences or
    queries return empty results and leave the cache alone."""
    from minixmax_h3_b200 import ops

    c = ops.KV8Cache.empty(2, 2, 64, device=cuda)
    c.k.fill_(3)
    table, lens = ints([[0, 1]], cuda), ints([7], cuda)
    x = torch.zeros(1, 0, 2, 64, dtype=torch.bfloat16, device=cuda)
    ops.kv8_append(c, x, x, table, lens)
    assert [t.shape for t in ops.kv8_read(c, table, lens, 0)] == [(1, 0, 2, 64)] * 2
    assert ops.kv8_attention(x, c, table, lens).shape == (1, 0, 2, 64)
    x, table, lens = x[:0], table[:0], lens[:0]
    ops.kv8_append(c, x, x, table, lens)
    assert [t.shape for t in ops.kv8_read(c, table, lens, 9)] == [(0, 9, 2, 64)] * 2
    assert ops.kv8_attention(torch.zeros(0, 3, 4, 64, dtype=torch.bfloat16, device=cuda), c, table, lens).shape == (0, 3, 4, 64)
    assert bool((c.k == 3).all())
