# SPDX-License-Identifier: MIT
"""Values that are no numbers reach the tokens that see them and no others, whatever shares a tile with them (csrc/chunk_attn_kernels.cu).

Numbers of a row that are computed once more have scores, probabilities and sums in fp32: of at most 3000 terms, one after another, each addition 2^-24 of the
sum so far, they are off by less than 3000 * 2^-24 < 2^-12 of sum p |v| beside 2^-11 for the scores, which the tolerance of test_chunk_gpu covers; all
others are bit for bit what they are without such values."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops
from test_chunk_gpu import Case

pytestmark = pytest.mark.gpu


def _spoil(c, b, tokens, head, dim, what, key=False):
    """Token(s) of request b get `what` as their value (key) in a dim -- 4-bit cache: in the 32 dims of its group."""
    for t in tokens:
        s = int(c.slots[b][t])
        blk, at = s // c.block, s % c.block
        if c.q4:
            tile = c.cache[blk, head, at // 16]
            par = tile[(16 if key else 18) * c.hd:][: 2 * c.hd].view(torch.bfloat16).view(16, 2, c.hd // 32)
            par[at % 16, 1, dim // 32] = what
        else:
            (c.k if key else c.v)[blk, head, at, dim] = what


def _sees(c, b, t, head, dim):
    """[rows, heads * dims]: where the value of token t in that dim has a say."""
    G = c.nq // c.nkv
    hit = torch.zeros(c.qkv.shape[0], c.nkv, G, c.hd, dtype=torch.bool, device="cuda")
    first = t - (c.ctx[b] - c.new[b])
    lo = int(c.cu[b])
    dims = slice(dim // 32 * 32, dim // 32 * 32 + 32) if c.q4 else dim
    hit[lo + max(first, 0):lo + c.new[b], head, :, dims] = True
    return hit.flatten(1)


def _check(c, clean, want, size, spoiled, reach=None):
    got = c.run()
    seen = torch.zeros_like(clean, dtype=torch.bool)
    for b, t, head, dim in spoiled:
        seen |= _sees(c, b, t, head, dim)
    assert not got[seen].isfinite().any()
    err = (got.double() - want).abs()
    ok = err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * size
    assert bool((ok | seen).all()), (~(ok | seen)).nonzero()[:4].tolist()
    # dims that no such value stands in stay bit for bit
    dims = seen.view(len(got), c.nkv, -1, c.hd).any(0).any(1)  # [nkv, hd], from the rows that see them
    for b, t, head, dim in spoiled:
        dims[head, slice(dim // 32 * 32, dim // 32 * 32 + 32) if c.q4 else dim] = True
    rest = (~dims)[:, None].expand(c.nkv, c.nq // c.nkv, c.hd).reshape(-1)
    assert torch.equal(got[:, rest], clean[:, rest])
    return got


HEADS = [(4, 4, 128), (4, 2, 64), (6, 2, 128), (8, 2, 64), (14, 2, 128), (28, 4, 128), (12, 1, 64), (128, 1, 128)]


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_near_the_end_of_a_pair(heads, what, q4):
    """At the last, the first and the middle token of pairs, of a long request whose pairs are cut and of short ones, which are not."""
    lens = [(600, 1500), (3, 40), (70, 70), (1, 5), (30, 31), (300, 300)]
    c = Case(heads, 16, lens, q4, seed=3)
    clean = c.run()
    want, size = c.want()
    pair = 2 * (128 // (heads[0] // heads[1]))
    spoiled = []
    for b, (n, ctx) in enumerate(lens):
        for i in {pair - 1, min(2 * pair, n) - 1, n // 2, n - 1}:
            if 0 <= i < n:
                spoiled.append((b, ctx - n + i, (b + i) % heads[1], (37 * b + 11 * i) % heads[2]))
    for b, t, head, dim in spoiled:
        _spoil(c, b, [t], head, dim, what)
    _check(c, clean, want, size, spoiled)


@pytest.mark.parametrize("q4", [False, True])
def test_few_tokens_on_long_contexts(q4):
    for heads, lens in (((28, 4, 128), [(5, 3000), (2, 900)]), ((8, 8, 64), [(13, 2100)]), ((40, 8, 128), [(1, 600), (8, 1100), (2, 130)] * 30)):
        c = Case(heads, 32, lens, q4, seed=5)
        clean = c.run()
        want, size = c.want()
        spoiled = [(b, ctx - 1, b % heads[1], 5) for b, (_, ctx) in enumerate(lens)]
        for b, t, head, dim in spoiled:
            _spoil(c, b, [t], head, dim, math.nan)
        got = _check(c, clean, want, size, spoiled)
        assert torch.equal(c.run().view(torch.int16), got.view(torch.int16))


@pytest.mark.parametrize("q4", [False, True])
def test_keys_that_are_no_numbers(q4):
    """A key that is none takes every number of the rows that see it, and none of the others'."""
    c = Case((4, 4, 128), 16, [(300, 700), (20, 60)], q4, seed=8)
    clean = c.run()
    for what in (math.nan, math.inf):
        _spoil(c, 0, [650], 2, 9, what, key=True)
        got = c.run().view(-1, 4, 128)
        first = 650 - 400
        if what != what:
            assert got[first:300, 2].isnan().all()
        keep = torch.ones(320, 4, dtype=torch.bool, device="cuda")
        keep[first:300, 2] = False
        assert torch.equal(got[keep], clean.view(-1, 4, 128)[keep])


@pytest.mark.parametrize("q4", [False, True])
def test_tokens_that_see_nothing_have_zeros(q4):
    c = Case((14, 2, 128), 16, [(40, 60), (5, 30)], q4, seed=6)
    c.lens = torch.tensor([10, 3], dtype=torch.int32, device="cuda")  # the first thirty, and two, are ahead of the first key
    clean = c.run()
    for d in range(0, 128, 32):
        _spoil(c, 0, range(10), 0, d, math.nan)
        _spoil(c, 1, range(3), 1, d, math.inf)
    got = c.run()
    assert (got[:30] == 0).all() and (got[40:42] == 0).all()
    assert torch.equal(got[:40, 7 * 128:], clean[:40, 7 * 128:]) and torch.equal(got[40:, : 7 * 128], clean[40:, : 7 * 128])
    assert not got[30:40, ::32][:, : 28].isfinite().any()


@pytest.mark.parametrize("q4", [False, True])
def test_blocks_that_are_missing(q4):
    """Among the keys that a row sees, and the one that holds the value itself."""
    c = Case((4, 4, 128), 16, [(400, 900)], q4, seed=9)
    c.table[0, 3], c.table[0, 40], c.table[0, 50] = -1, c.n_blocks, 2 ** 31 - 1
    clean = c.run()
    want, size = c.want()
    _spoil(c, 0, [50 * 16 + 3], 1, 64, math.nan)  # in a block that the table does not name
    assert torch.equal(c.run(), clean)
    _spoil(c, 0, [899, 700], 1, 64, math.inf)
    _check(c, clean, want, size, [(0, 899, 1, 64), (0, 700, 1, 64)])


def test_rows_that_lie_apart_and_rows_of_no_request():
    c = Case((8, 2, 64), 16, [(5, 100), (90, 90)], extra=24, seed=9)
    want, size = c.want()
    clean = c.run()
    pad = torch.cat([c.qkv[:7], c.qkv, c.qkv[:20]])
    c.cu = c.cu + 7
    for b, t in ((0, 99), (1, 63)):
        _spoil(c, b, [t], 1, 33, math.nan)
    out = torch.full((pad.shape[0], 512), math.nan, dtype=torch.bfloat16, device="cuda")
    got = c.run(out, pad)
    assert got[:7].isnan().all() and got[102:].isnan().all()
    seen = torch.zeros(95, 8, 64, dtype=torch.bool, device="cuda")
    seen[4, 4:, 33] = seen[68:, 4:, 33] = True
    got, seen = got[7:102], seen.flatten(1)
    assert got[seen].isnan().all()
    assert bool((((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * size) | seen).all())
    same = torch.ones(8, 64, dtype=torch.bool, device="cuda")
    same[4:, 33] = False
    assert torch.equal(got[:, same.flatten()], clean[:, same.flatten()])


@pytest.mark.parametrize("q4", [False, True])
def test_captured(q4):
    """A graph whose replay meets such a value although its capture did not."""
    c = Case((4, 2, 128), 16, [(200, 500), (9, 40)], q4, seed=4)
    clean = c.run()
    want, size = c.want()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.run()
    g.replay()
    assert torch.equal(out, clean)
    _spoil(c, 0, [499], 1, 100, math.nan)
    _spoil(c, 1, [38], 0, 3, math.inf)
    got = _check(c, clean, want, size, [(0, 499, 1, 100), (1, 38, 0, 3)])
    g.replay()
    assert torch.equal(out.view(torch.int16), got.view(torch.int16))


@pytest.mark.parametrize("q4", [False, True])
def test_all_values_are_none(q4):
    """A cache in ruins: rows see such values themselves, and stay as they are."""
    c = Case((28, 4, 128), 16, [(600, 6000), (1, 2000)], q4, seed=2)
    for h in range(4):
        (c.cache[:, h, :, 18 * 128:].view(torch.bfloat16) if q4 else c.v[:, h]).fill_(math.nan)
    assert c.run().isnan().all()


@pytest.mark.parametrize("q4", [False, True])
def test_out_in_the_place_of_the_queries(q4):
    c = Case((14, 2, 128), 16, [(400, 900), (5, 300), (1, 40)], q4, seed=2)
    q = c.qkv[:, : 14 * 128].contiguous()
    want = c.run(qkv=q)
    _spoil(c, 0, [899], 1, 5, math.nan)  # (what is hidden may show: there is nothing left to compute it from)
    assert torch.equal(c.run(q, q)[:, : 7 * 128], want[:, : 7 * 128])
