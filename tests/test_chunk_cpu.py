# SPDX-License-Identifier: MIT
"""The CPU path of attention of new tokens over the paged caches, and its refusals.  In fp32 throughout: sums of at most 100 terms, whose absolute
values stay below 10, are off by less than 100 * 10 * 2^-24 < 2^-13."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops


def _state(block=16, hd=64, nkv=2):
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(12, nkv, block, hd, generator=g) for _ in range(2))
    table = torch.randperm(12, generator=g)[:8].view(2, 4).to(torch.int32)
    q = torch.randn(9, 6 * hd + 5, generator=g)
    return q, k, v, table, torch.tensor([0, 5, 9], dtype=torch.int32), torch.tensor([60, 4], dtype=torch.int32)


def test_against_one_token_at_a_time():
    """New token i of a chunk has what a decode step has with as many tokens in the cache."""
    q, k, v, table, cu, lens = _state()
    got = ops.paged_attn_chunk(q, k, v, table, cu, lens, 6, 2, 64, 0.125)
    for b in range(2):
        n = int(cu[b + 1] - cu[b])
        for i in range(n):
            ctx = torch.tensor([int(lens[b]) - n + i + 1], dtype=torch.int32)
            r = int(cu[b]) + i
            want = ops.paged_attn_decode(q[r:r + 1], k, v, table[b:b + 1], ctx, 6, 2, 64, 0.125)
            assert (got[r] - want[0]).abs().max() < 2.0 ** -13


def test_blocks_that_are_missing_and_tokens_that_see_nothing():
    q, k, v, table, cu, lens = _state()
    table[0, 1], table[1, 0] = -1, 99
    got = ops.paged_attn_chunk(q, k, v, table, cu, lens, 6, 2, 64, 0.125)
    assert torch.isfinite(got).all() and (got[5:] == 0).all() and (got[:5] != 0).any()
    short = ops.paged_attn_chunk(q, k, v, table, cu, torch.tensor([2, 0], dtype=torch.int32), 6, 2, 64, 0.125)
    assert (short[:3] == 0).all() and (short[3:5] != 0).all(-1).all() and (short[5:] == 0).all()


def test_rows_of_no_request_stay():
    q, k, v, table, cu, lens = _state()
    out = torch.full((9, 6 * 64), 7.0)
    cu = torch.tensor([1, 4, 6], dtype=torch.int32)
    got = ops.paged_attn_chunk(q, k, v, table, cu, lens, 6, 2, 64, 0.125, out)
    assert got is out and (out[0] == 7).all() and (out[6:] == 7).all() and (out[1:6] != 7).all(-1).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_the_4_bit_cache_is_what_kv4_read_gives(hd):
    g = torch.Generator().manual_seed(2)
    nkv, block, rows = 2, 32, 40
    kv = torch.randn(rows, 2 * nkv * hd, generator=g)
    cache = ops.kv4_cache(4, nkv, hd, block, "cpu")
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    t = torch.arange(rows)
    slots = (table[0].long()[t // block] * block + t % block).to(torch.int32)
    ops.rope_kv_write_q4(kv, torch.zeros(rows, dtype=torch.int32), slots, cache, 0, nkv, hd, block, 1e4)
    k = torch.zeros(4, nkv, block, hd)
    v = torch.zeros_like(k)
    rk, rv = ops.kv4_read(cache, slots, hd, block)
    s = slots.long()
    k[s // block, :, s % block], v[s // block, :, s % block] = rk.float(), rv.float()
    q = torch.randn(7, 4 * hd, generator=g)
    cu, lens = torch.tensor([0, 7], dtype=torch.int32), torch.tensor([rows], dtype=torch.int32)
    a = ops.paged_attn_chunk_q4(q, cache, table, cu, lens, 4, nkv, hd, 0.1)
    assert torch.equal(a, ops.paged_attn_chunk(q, k, v, table, cu, lens, 4, nkv, hd, 0.1))


def test_refusals():
    q, k, v, table, cu, lens = _state()
    good = dict(q=q, k_cache=k, v_cache=v, block_tables=table, cu_q=cu, ctx_lens=lens, nq=6, nkv=2, hd=64, scale=0.1)
    ops.paged_attn_chunk(**good)
    for bad in (dict(q=q[:, :100]), dict(q=q[0]), dict(k_cache=k[:, :, :8]), dict(k_cache=k[:3]), dict(block_tables=table.long()), dict(block_tables=table[:1]),
                dict(cu_q=cu[:2]), dict(ctx_lens=lens[:1]), dict(nq=5), dict(nkv=0), dict(hd=96), dict(hd=128), dict(scale=0.0), dict(scale=math.nan), dict(scale=-1.0),
                dict(out=torch.empty(9, 100)), dict(out=torch.empty(9, 384, dtype=torch.bfloat16)), dict(k_cache=k[0])):
        with pytest.raises(ValueError):
            ops.paged_attn_chunk(**{**good, **bad})
    cache = ops.kv4_cache(4, 2, 64, 16, "cpu")
    good = dict(q=q, cache=cache, block_tables=table, cu_q=cu, ctx_lens=lens, nq=6, nkv=2, hd=64, scale=0.1)
    for bad in (dict(hd=128), dict(nkv=1), dict(scale=-1.0), dict(nq=7)):
        with pytest.raises(ValueError):
            ops.paged_attn_chunk_q4(**{**good, **bad})
