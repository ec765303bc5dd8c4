# SPDX-License-Identifier: MIT
"""Attention of new tokens over the paged caches (csrc/chunk_attn_kernels.cu) against 64-bit statements.

Tolerance.  The result is rounded to bf16 once, 2^-8 of it.  Probabilities are rounded to bf16 for the products, 2^-8 of each: 2^-8
sum p |v|.  Scores are sums of at most 128 products in fp32 (the sums here, in absolute values times scale, stay below 64: off by less than
128 * 64 * 2^-24 = 2^-11 at the very most, as is every probability), exponentials and sums add less than 2^-14: 2^-8 |want| + (2^-8 + 2^-10) sum p |v|."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops

pytestmark = pytest.mark.gpu


def _g(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(seed, *shape):
    return torch.randn(*shape, generator=_g(seed), device="cuda")


class Case:
    """Requests of given (new, ctx) lengths on scattered blocks of a cache that is NaN wherever no token stands."""

    def __init__(self, heads, block, lens, q4=False, extra=0, seed=0, grow=0.0, spare=3, width=None):
        self.nq, self.nkv, self.hd = heads
        self.block, self.q4 = block, q4
        nq, nkv, hd = heads
        self.new = [n for n, _ in lens]
        self.ctx = [c for _, c in lens]
        pages = [-(-c // block) for c in self.ctx]
        self.width = max(max(pages), 1) if width is None else width
        self.n_blocks = sum(pages) + spare
        order = torch.randperm(self.n_blocks, generator=_g(seed), device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, p in enumerate(pages):
            k = min(p, self.width)
            self.table[b, :k] = order[at:at + k]
            at += p
        self.cu = torch.tensor([0] + self.new, device="cuda").cumsum(0).to(torch.int32)
        self.lens = torch.tensor(self.ctx, dtype=torch.int32, device="cuda")
        rows = sum(self.new)
        self.qkv = _randn(seed + 1, rows, (nq + 2 * nkv) * hd + extra).bfloat16()
        self.scale = 1.0 / math.sqrt(hd)
        slots = []
        for b, c in enumerate(self.ctx):
            t = torch.arange(min(c, self.width * block), device="cuda")
            slots.append((self.table[b].long()[t // block] * block + t % block) if len(t) else t)
        self.slots = slots
        every = torch.cat(slots)
        k, v = _randn(seed + 2, len(every), nkv, hd) + _randn(seed + 3, nkv, hd), _randn(seed + 4, len(every), nkv, hd)
        if grow:  # later keys score higher, again and again: sums are rescaled
            k = k * (1 + grow * torch.cat([torch.arange(len(s), device="cuda") for s in slots]))[:, None, None]
        k, v = k.bfloat16(), v.bfloat16()
        if q4:
            self.cache = ops.kv4_cache(self.n_blocks, nkv, hd, block).fill_(0xFF)
            ops.rope_kv_write_q4(torch.cat([k, v], 1).flatten(1), torch.zeros(len(every), dtype=torch.int32, device="cuda"), every.to(torch.int32), self.cache, 0,
                                 nkv, hd, block, 1e4)
        else:
            self.k = torch.full((self.n_blocks, nkv, block, hd), math.nan, dtype=torch.bfloat16, device="cuda")
            self.v = self.k.clone()
            self.k[every // block, :, every % block] = k
            self.v[every // block, :, every % block] = v

    def run(self, out=None, qkv=None):
        q = self.qkv if qkv is None else qkv
        tail = (self.table, self.cu, self.lens, self.nq, self.nkv, self.hd, self.scale, out)
        return ops.paged_attn_chunk_q4(q, self.cache, *tail) if self.q4 else ops.paged_attn_chunk(q, self.k, self.v, *tail)

    def read(self, slots):
        if self.q4:
            return ops.kv4_read(self.cache, slots.to(torch.int32), self.hd, self.block)
        return self.k[slots // self.block, :, slots % self.block], self.v[slots // self.block, :, slots % self.block]

    def want(self):
        """(result, sum of p |v|) in 64 bits, row by row of every request."""
        nq, nkv, hd = self.nq, self.nkv, self.hd
        out = torch.zeros(self.qkv.shape[0], nkv, nq // nkv, hd, dtype=torch.float64, device="cuda")
        size = out.clone()
        cu = self.cu.tolist()
        for b, (m, c) in enumerate(zip(self.new, self.lens.tolist())):
            t = torch.arange(min(c, self.width * self.block), device="cuda")
            blk = self.table[b].long()[t // self.block] if len(t) else t
            ok = (blk >= 0) & (blk < self.n_blocks)
            t, slots = t[ok], (blk * self.block + t % self.block)[ok]
            if not m or not len(t):
                continue
            k, v = (x.double().transpose(0, 1) for x in self.read(slots))
            q = self.qkv[cu[b]:cu[b] + m, : nq * hd].double().view(m, nkv, nq // nkv, hd).permute(1, 2, 0, 3)
            x = (q @ k[:, None].transpose(2, 3)) * self.scale
            seen = t <= (c - m + torch.arange(m, device="cuda"))[:, None]
            x = x.masked_fill(~seen, -math.inf)
            p = torch.softmax(x, -1).masked_fill(~seen.any(-1)[:, None], 0.0)
            out[cu[b]:cu[b] + m] = (p @ v[:, None]).permute(2, 0, 1, 3)
            size[cu[b]:cu[b] + m] = (p @ v[:, None].abs()).permute(2, 0, 1, 3)
        return out.flatten(1), size.flatten(1)

    def check(self, got):
        want, size = self.want()
        err = (got.double() - want).abs()
        bad = ~(err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * size)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(err[~torch.isnan(err)].max()))


HEADS = [(28, 4, 128), (8, 2, 64), (7, 1, 128), (4, 4, 128), (40, 8, 128), (12, 1, 64), (3, 1, 64), (128, 1, 128), (50, 1, 64)]
LENS = [
    [(1, 1)], [(1, 17)], [(5, 5)], [(5, 333)], [(64, 64)], [(1, 64), (1, 65), (1, 63)],
    [(0, 5), (3, 70), (0, 0), (1, 1), (19, 19), (0, 64), (2, 2)],          # requests without new tokens, and without any
    [(37, 400), (130, 131), (18, 18), (36, 200), (17, 1000)],               # one tile, just two, more
    [(300, 1500)], [(257, 257), (1, 2000)],
]


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", range(len(LENS)))
def test_lengths(heads, lens, q4):
    for block in (16, 64) if heads == HEADS[0] else (16,):
        c = Case(heads, block, LENS[lens], q4, seed=lens)
        c.check(c.run())


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("block", [16, 32, 48, 64, 80, 128, 192])
def test_blocks(block, q4):
    c = Case((14, 2, 128), block, [(40, 300), (3, 191), (1, 192), (1, 193), (7, 1000)], q4, seed=block)
    c.check(c.run())


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("heads", [(28, 4, 128), (12, 1, 64), (4, 4, 128)])
@pytest.mark.parametrize("new", [1, 3, 25])
def test_many_requests(heads, new, q4):
    """Short chunks: pairs of one tile take the two places in turn; more requests than threads."""
    g = torch.Generator().manual_seed(new)
    lens = [(int(n), int(n + c)) for n, c in zip(torch.randint(0, new + 1, (700,), generator=g), torch.randint(0, 150, (700,), generator=g))]
    c = Case(heads, 16, lens, q4, seed=new)
    c.check(c.run())


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("heads,lens", [((28, 4, 128), [(700, 5000), (1, 9000)]), ((40, 8, 128), [(13, 20000), (2, 3)]), ((7, 1, 128), [(1, 40000)]),
                                        ((1, 1, 64), [(400, 3001)]), ((128, 1, 128), [(50, 1000)])])
def test_long(heads, lens, q4):
    c = Case(heads, 32, lens, q4, seed=7)
    c.check(c.run())


@pytest.mark.parametrize("q4", [False, True])
def test_scores_that_grow(q4):
    c = Case((8, 1, 128), 16, [(130, 1500), (1, 700)], q4, seed=3, grow=0.0005)
    c.check(c.run())


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("block", [16, 64])
def test_blocks_that_are_missing(q4, block):
    c = Case((14, 2, 128), block, [(40, 900), (2, 500), (3, 130), (30, 30)], q4, seed=5)
    c.table[0, 2] = -1
    c.table[0, 900 // block // 2] = c.n_blocks
    c.table[0, 900 // block] = 2 ** 31 - 1   # that of the newest tokens
    c.table[1, ::2] = -2 ** 31
    c.table[2] = -1                           # nothing at all: zeros
    got = c.run()
    c.check(got)
    assert (got[42:45] == 0).all()


@pytest.mark.parametrize("q4", [False, True])
def test_tokens_that_see_nothing(q4):
    """More new tokens than there are in all: the first ones are before the first key."""
    c = Case((14, 2, 128), 16, [(10, 40), (70, 200)], q4, seed=6)
    c.lens = torch.tensor([4, 1], dtype=torch.int32, device="cuda")
    got = c.run()
    c.check(got)
    assert (got[:6] == 0).all() and (got[10:79] == 0).all() and (got[79] != 0).any()
    c.lens = torch.tensor([0, -5], dtype=torch.int32, device="cuda")
    assert (c.run() == 0).all()


@pytest.mark.parametrize("q4", [False, True])
def test_tables_that_end_early(q4):
    c = Case((14, 2, 128), 16, [(10, 300), (3, 20)], q4, seed=6, width=4)
    c.check(c.run())
    c.table = c.table[:, :0].contiguous()
    assert (c.run() == 0).all()


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("heads", [(28, 4, 128), (8, 2, 64)])
def test_rows_of_no_request_stay(heads, q4):
    c = Case(heads, 16, [(5, 100), (40, 90)], q4, seed=8)
    want = c.run()
    pad = torch.cat([c.qkv[:7], c.qkv, c.qkv[:20]])
    c.cu = c.cu + 7
    out = torch.full((pad.shape[0], want.shape[1]), 3.25, dtype=torch.bfloat16, device="cuda")
    got = c.run(out, pad)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(got[7:52], want) and (got[:7] == 3.25).all() and (got[52:] == 3.25).all()


@pytest.mark.parametrize("q4", [False, True])
def test_requests_that_share_blocks(q4):
    """A prefix that several requests have, and a block twice in one table: blocks are read only."""
    c = Case((28, 4, 128), 16, [(5, 300), (40, 300), (1, 300)], q4)
    c.table[1, :12] = c.table[0, :12]
    c.table[2] = c.table[0]
    c.table[0, 3] = c.table[0, 2]
    c.check(c.run())


def test_row_offsets_that_fall():
    """Rows that two requests claim hold one's result or the other's, whichever was there last; all others are right."""
    c = Case((8, 2, 64), 16, [(30, 64), (20, 200), (30, 90)])
    want, size = c.want()
    c.cu[2] = 10  # the second has none, the third 70 rows from 10 on
    got = c.run()
    err, room = (got.double() - want).abs(), 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * size
    assert bool((err <= room)[:10].all()) and bool(got.isfinite().all())


def test_row_offsets_that_leave_the_rows():
    """Offsets outside q and lengths out of any range: nothing outside the tensors is touched."""
    c = Case((14, 2, 128), 16, [(30, 100), (10, 60)], seed=8)
    for cu in ([-5, 30, 400], [50, 20, 40], [0, 2 ** 31 - 1, -1], [-2 ** 31, 10, 40]):
        c.cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        c.run()
    c.lens = torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    c.run()
    torch.cuda.synchronize()


@pytest.mark.parametrize("q4", [False, True])
def test_rows_that_lie_apart(q4):
    c = Case((8, 2, 64), 16, [(5, 100), (40, 90)], q4, extra=24, seed=9)
    want = c.run()
    assert torch.equal(c.run(qkv=c.qkv[:, : 8 * 64].contiguous()), want)
    one = Case((8, 2, 64), 16, [(1, 50)], q4, seed=9)
    assert torch.equal(one.run(qkv=one.qkv[:, : 8 * 64 + 3]), one.run())


@pytest.mark.parametrize("at", [10, 300, 463])
def test_values_that_are_no_numbers(at):
    """An infinite value reaches the tokens that see it, and none of more than 63 tokens before it."""
    c = Case((14, 2, 128), 16, [(400, 464)], seed=4)
    clean = c.run()
    s = c.slots[0][at]
    c.v[s // 16, 1, s % 16, 5] = math.inf
    got = c.run()
    first = at - 64  # the new token that stands where the value does
    for r in range(0, 400):
        if r >= first:
            assert not torch.isfinite(got[r, 7 * 128 + 5])
        elif r < first - 63:
            assert torch.equal(got[r], clean[r])
    assert torch.equal(got[:, : 7 * 128], clean[:, : 7 * 128])  # the other head


def test_offsets_beyond_32_bits():
    block, nkv, hd = 16, 4, 128
    n_blocks = 2 ** 31 // (block * nkv * hd) + 40
    k = torch.empty(n_blocks, nkv, block, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    c = Case((8, nkv, hd), block, [(20, 500), (3, 40)], seed=2)
    move = n_blocks - c.n_blocks
    k[move:], v[move:] = c.k, c.v
    want = c.run()
    c.table = torch.where(c.table >= 0, c.table + move, -1).to(torch.int32)
    assert torch.equal(ops.paged_attn_chunk(c.qkv, k, v, c.table, c.cu, c.lens, 8, nkv, hd, c.scale), want)


@pytest.mark.parametrize("q4", [False, True])
def test_streams_and_graphs(q4):
    cases = [Case((28, 4, 128), 16, [(8, 900 + 50 * i), (1, 300), (60, 400)], q4, seed=i) for i in range(3)]
    want = [c.run() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(c.run())
    torch.cuda.synchronize()
    assert all(torch.equal(r, want[i % 3]) for i, r in enumerate(got))
    graphs, outs = [], []
    for c in cases[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run())
        graphs.append(g)
    for _ in range(2):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
    # other lengths at the replay: as many rows, fewer tokens in all
    cases[0].lens.sub_(5)
    graphs[0].replay()
    torch.cuda.synchronize()
    cases[0].check(outs[0])


def test_agrees_with_the_decode_kernels():
    for q4 in (False, True):
        c = Case((28, 4, 128), 16, [(1, 700), (1, 33), (1, 1)], q4, seed=12)
        args = (c.table, c.lens, c.nq, c.nkv, c.hd, c.scale)
        want = ops.paged_attn_decode_q4(c.qkv, c.cache, *args) if q4 else ops.paged_attn_decode(c.qkv, c.k.nan_to_num(0), c.v.nan_to_num(0), *args)
        _, size = c.want()
        assert ((c.run().double() - want.double()).abs() <= 2.0 ** -6 * size).all()


def test_refusals():
    c = Case((14, 2, 128), 16, [(30, 100), (10, 60)], seed=8)
    q4 = Case((14, 2, 128), 16, [(30, 100), (10, 60)], True, seed=8)

    def call(q=c.qkv, k=c.k, v=c.v, table=c.table, cu=c.cu, lens=c.lens, nq=14, nkv=2, hd=128, scale=0.1, out=None):
        ops.paged_attn_chunk(q, k, v, table, cu, lens, nq, nkv, hd, scale, out)

    call()
    wide = torch.zeros(40, 14 * 128 + 4, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(q=c.qkv.float()), dict(q=c.qkv[:, :100]), dict(q=wide), dict(q=wide[:, 4:]), dict(k=c.k[:, :, :8]), dict(k=c.k[:3]), dict(k=c.k.float()),
                dict(table=c.table.long()), dict(table=c.table[:1]), dict(cu=c.cu[:2]), dict(cu=c.cu.cpu()), dict(lens=c.lens[:1]), dict(nq=13), dict(nkv=0), dict(hd=96),
                dict(scale=0.0), dict(scale=math.nan), dict(scale=-1.0), dict(scale=math.inf), dict(out=c.qkv), dict(k=c.k[:0], v=c.v[:0]),
                dict(k=c.k.transpose(1, 2)), dict(k=q4.cache, v=None), dict(q=c.qkv.expand(40, -1).t())):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call(**bad)
    with pytest.raises((RuntimeError, ValueError)):
        ops.paged_attn_chunk_q4(q4.qkv, q4.cache, q4.table, q4.cu, q4.lens, 14, 2, 64, 0.1)
    with pytest.raises((RuntimeError, ValueError)):
        ops.paged_attn_chunk_q4(q4.qkv, q4.cache.view(torch.int8), q4.table, q4.cu, q4.lens, 14, 2, 128, 0.1)
    none = ops.paged_attn_chunk(c.qkv[:0], c.k, c.v, c.table[:0], c.cu[:1], c.lens[:0], 14, 2, 128, 0.1)
    assert none.shape == (0, 14 * 128)
    call()
