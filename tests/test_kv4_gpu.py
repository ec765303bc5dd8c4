# SPDX-License-Identifier: MIT
"""The 4-bit key/value cache on the GPU (csrc/kv4_kernels.cu) against 64-bit statements.

Tolerances.  Rotated rows: one rounding to bf16 (half a step, 2^-8 of the value) of a result whose fp32 products and sum are off by
2^-24 each: 2^-8 |want| + 2^-22 (|x| + |y|).  The cache: codes, step and low are the formula's to the bit, so values are equal.
Attention: the result's rounding, 2^-8 |want|, and the probabilities times step in fp16 (2^-11 of every term, its terms
step * code and low in absolute values at most 3 times |value| + range), scores in fp32 (errors below 2^-13 for the scores here):
2^-8 |want| + 2^-10 sum p (|low| + step * code)."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.ops import reference as ref

pytestmark = pytest.mark.gpu


def _g(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(seed, *shape):
    return torch.randn(*shape, generator=_g(seed), device="cuda")


def _dirty_cache(n_blocks, nkv, hd, bs):
    """A cache whose unwritten parts are NaN."""
    return ops.kv4_cache(n_blocks, nkv, hd, bs).fill_(0xFF)


def _rotated(x, pos, nq, nkv, hd, theta):
    x = x.double().cpu().view(x.shape[0], -1, hd)
    ang = pos.double().cpu()[:, None] * theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    y[:, nq + nkv:] = x[:, nq + nkv:]
    return y, a.abs() + b.abs()


HEADS = [(28, 4, 128), (1, 1, 128), (8, 2, 64), (0, 3, 128), (5, 5, 64), (16, 1, 64)]


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("rows", [1, 3, 64, 129, 300])
@pytest.mark.parametrize("block", [16, 48])
@pytest.mark.parametrize("splits", [0, 1, 5])
def test_write(nq, nkv, hd, rows, block, splits):
    n_blocks = rows // block + 4
    width = (nq + 2 * nkv) * hd
    x = _randn(1, max(splits, 1), rows, width) * (1 + 20 * torch.rand(width, generator=_g(2), device="cuda"))
    bias = _randn(3, width).bfloat16() if splits > 1 else None
    pos = torch.randint(0, 131072, (rows,), generator=_g(4), device="cuda", dtype=torch.int32)
    slots = torch.randperm(n_blocks * block, generator=_g(5), device="cuda")[:rows].to(torch.int32)
    if rows > 3:
        slots[1], slots[2] = -1, n_blocks * block + 7  # not kept
    cache = _dirty_cache(n_blocks, nkv, hd, block)
    before = cache.clone()
    if splits:
        qkv = x
        total = x[0]
        for p in x[1:]:
            total = total + p
        whole = (total + bias.float() if bias is not None else total).bfloat16()
        got = ops.rope_kv_write_q4(qkv, pos, slots, cache, nq, nkv, hd, block, 1e6, bias=bias)
    else:
        whole = x[0].bfloat16()
        buf = whole.clone()
        got = ops.rope_kv_write_q4(buf, pos, slots, cache, nq, nkv, hd, block, 1e6)
        assert got.data_ptr() == buf.data_ptr()
        other = torch.empty_like(whole)  # into another buffer: the same, and the rows stay
        keep = whole.clone()
        c2 = before.clone()
        assert ops.rope_kv_write_q4(whole, pos, slots, c2, nq, nkv, hd, block, 1e6, out=other).data_ptr() == other.data_ptr()
        assert torch.equal(other, got) and torch.equal(whole, keep) and torch.equal(c2, cache)
    want, size = _rotated(whole, pos, nq, nkv, hd, 1e6)
    err = (got.double().cpu().view_as(want) - want).abs()
    slack = 2.0 ** -22 * torch.cat([size, size], -1)
    assert bool((err <= 2.0 ** -8 * want.abs() + slack).all())
    # the cache: what the formula makes of the rotated rows, and nothing else touched
    mine = before.cpu()
    rot = got.cpu().view(rows, -1, hd)
    ref.kv4_write(mine, slots.cpu(), rot[:, nq:nq + nkv], rot[:, nq + nkv:], block)
    assert torch.equal(mine, cache.cpu())
    k, v = ops.kv4_read(cache, slots, hd, block)
    wk, wv = ref.kv4_read(mine, slots.cpu(), hd, block)
    assert torch.equal(k.cpu(), wk) and torch.equal(v.cpu(), wv)


@pytest.mark.parametrize("splits", [0, 2])
def test_write_of_many_rows(splits):
    """Beyond the rows that get blocks of their own; not a multiple of the rows of a block."""
    nq, nkv, hd, rows = 3, 2, 128, 700
    x = _randn(6, max(splits, 1), rows, 7 * hd)
    whole = (x[0] + x[1]).bfloat16() if splits else x[0].bfloat16()
    pos = torch.arange(rows, dtype=torch.int32, device="cuda") * 37
    slots = torch.arange(rows, dtype=torch.int32, device="cuda").flip(0).contiguous()
    cache = _dirty_cache(44, nkv, hd, 16)
    got = ops.rope_kv_write_q4(x if splits else whole.clone(), pos, slots, cache, nq, nkv, hd, 16, 1e6)
    want, size = _rotated(whole, pos, nq, nkv, hd, 1e6)
    assert bool(((got.double().cpu().view_as(want) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * torch.cat([size, size], -1)).all())
    mine = torch.full_like(cache.cpu(), 0xFF)
    rot = got.cpu().view(rows, -1, hd)
    ref.kv4_write(mine, slots.cpu(), rot[:, nq:nq + nkv], rot[:, nq + nkv:], 16)
    assert torch.equal(mine, cache.cpu())


def test_rope_alone_and_no_rows():
    x = _randn(1, 9, 6 * 128).bfloat16()
    pos = torch.arange(9, dtype=torch.int32, device="cuda") * 1000
    a = ops.rope_kv_write_q4(x.clone(), pos, None, None, 4, 1, 128, 16, 1e4)
    want, size = _rotated(x, pos, 4, 1, 128, 1e4)
    assert bool(((a.double().cpu().view_as(want) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * torch.cat([size, size], -1)).all())
    cache = ops.kv4_cache(2, 1, 128)
    e = torch.empty(0, 6 * 128, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert ops.rope_kv_write_q4(e, none, none, cache, 4, 1, 128, 16, 1e4).shape == (0, 768)
    assert ops.kv4_read(cache, none, 128)[0].shape == (0, 1, 128)


def test_groups_of_one_value_and_of_no_finite_range():
    hd, nkv = 128, 1
    x = torch.zeros(6, 2, hd, device="cuda")
    x[0] = 3.5                       # one value: step 0
    x[1, :, 40] = float("inf")       # the group reads as NaN, the others as they are
    x[2, :, 70] = float("nan")
    x[3, :, 3], x[3, :, 9] = 3e38, -3e38   # a range beyond fp32
    x[4, :, 96:] = torch.arange(32, device="cuda") * 1e-40  # below the smallest normal numbers
    x[5, :, :32] = torch.linspace(-1, 1, 32, device="cuda")
    x = x.bfloat16()
    cache = _dirty_cache(1, nkv, hd, 16)
    slots = torch.arange(6, dtype=torch.int32, device="cuda")
    ops.rope_kv_write_q4(x.view(6, -1).contiguous(), torch.zeros_like(slots), slots, cache, 0, nkv, hd, 16, 1e6)
    for key, t in zip((True, False), ops.kv4_read(cache, slots, hd)):
        t = t[:, 0].cpu()
        assert torch.equal(t[0], torch.full((hd,), 3.5, dtype=torch.bfloat16))
        for row, group in ((1, 1), (2, 2), (3, 0)):
            bad = torch.zeros(hd, dtype=torch.bool)
            bad[32 * group:32 * group + 32] = True
            if key and row != 3:  # RoPE of a key at position 0: infinity * sin 0 is NaN in the rotation partner, 64 dims on
                bad[(32 * group + 64) % hd:(32 * group + 64) % hd + 32] = True
            assert bool(t[row][bad].isnan().all()) and not bool(t[row][~bad].any())
        # half a step of bf16(2 / 15), and the roundings to bf16 of what goes in (below 1: 2^-9) and what is read (2^-8 up to 2)
        assert float((t[5, :32].float() - torch.linspace(-1, 1, 32)).abs().max()) <= (1 + 2.0 ** -8) / 15 + 2.0 ** -9 + 2.0 ** -8
    mine = torch.full_like(cache.cpu(), 0xFF)
    ref.kv4_write(mine, slots.cpu(), x.cpu()[:, :1], x.cpu()[:, 1:], 16)
    a, b = ref.kv4_read(mine, slots.cpu(), hd, 16), ops.kv4_read(cache, slots, hd)
    for p, q in zip(a, b):
        assert torch.equal(p.nan_to_num(7), q.cpu().nan_to_num(7))


def _filled(seed, lens, nkv, hd, block, extra=3, holes=(), k_scale=1.0, v_scale=1.0):
    """A cache with the requests' tokens in scattered blocks, its tables, and the values that it holds (fp64: low, step * code)."""
    b = len(lens)
    per = max(1, max(-(-n // block) for n in lens)) + 1
    n_blocks = sum(-(-n // block) for n in lens) + extra
    ids = torch.randperm(n_blocks, generator=_g(seed), device="cuda").to(torch.int32)
    table = torch.full((b, per), -1, dtype=torch.int32, device="cuda")
    cache = _dirty_cache(n_blocks, nkv, hd, block)
    at, slots = 0, []
    for i, n in enumerate(lens):
        nb = -(-n // block)
        table[i, :nb] = ids[at:at + nb]
        t = torch.arange(n, device="cuda")
        slots.append(table[i].long()[t // block] * block + t % block)
        at += nb
    slots = torch.cat(slots).to(torch.int32) if sum(lens) else torch.empty(0, dtype=torch.int32, device="cuda")
    rows = slots.numel()
    kv = _randn(seed + 1, rows, 2 * nkv, hd)
    kv[:, :nkv] = (kv[:, :nkv] + _randn(seed + 2, nkv, hd) * 2) * k_scale
    kv[:, nkv:] *= v_scale
    if rows:
        ops.rope_kv_write_q4(kv.bfloat16().view(rows, -1), torch.zeros_like(slots), slots, cache, 0, nkv, hd, block, 1e6)
    for i, page in holes:
        table[i, page] = -1 if page % 2 else n_blocks + 5
    return cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _attention_64(q, cache, table, lens, nq, nkv, hd, scale):
    """(result, sum p (|low| + step * code)) in 64 bits."""
    cache, table = cache.cpu(), table.cpu()
    bs, G = cache.shape[2] * 16, nq // nkv
    out = torch.zeros(q.shape[0], nq * hd, dtype=torch.float64)
    size = torch.zeros_like(out)
    byte, shift, ps, pl = ref._kv4_maps(hd)["v"]
    for b, n in enumerate(lens.tolist()):
        t = torch.arange(min(n, table.shape[1] * bs))
        blk = table[b].long()[t // bs]
        ok = (blk >= 0) & (blk < cache.shape[0])
        slots = (blk * bs + t % bs)[ok]
        if len(slots) == 0:
            continue
        k, v = (x.double() for x in ref.kv4_values(cache, slots, hd, bs))
        p = torch.softmax(torch.einsum("hgd,thd->hgt", q[b, :nq * hd].double().cpu().view(nkv, G, hd), k) * scale, -1)
        out[b] = torch.einsum("hgt,thd->hgd", p, v).flatten()
        low = v.unflatten(-1, (-1, 32)).amin(-1, keepdim=True).abs()  # (of the values held: the group's low or above)
        wide = (low + (v.unflatten(-1, (-1, 32)) - v.unflatten(-1, (-1, 32)).amin(-1, keepdim=True))).flatten(-2)
        size[b] = torch.einsum("hgt,thd->hgd", p, wide.abs()).flatten()
    return out, size


def _check(got, want, size):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * size).all()), float((err - 2.0 ** -8 * want.abs()).max())


@pytest.mark.parametrize("nq,nkv,hd", [(28, 4, 128), (1, 1, 128), (8, 1, 128), (9, 1, 128), (16, 1, 128), (32, 2, 64), (8, 2, 64),
                                       (12, 1, 64), (3, 3, 64), (40, 8, 128)])
@pytest.mark.parametrize("block", [16, 32, 80])
@pytest.mark.parametrize("lens", [[1], [0, 1, 2], [15, 16, 17, 0, 33], [129, 640, 7, 300, 1, 1000, 31]])
def test_attention(nq, nkv, hd, block, lens):
    cache, table, ctx = _filled(10, lens, nkv, hd, block)
    q = 2 * _randn(20, len(lens), (nq + 2 * nkv) * hd)
    q = q.bfloat16()
    scale = 1 / math.sqrt(hd)
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, nq, nkv, hd, scale)
    want, size = _attention_64(q, cache, table, ctx, nq, nkv, hd, scale)
    _check(got, want, size)
    for i, n in enumerate(lens):
        if n == 0:
            assert not bool(got[i].any())
    # an output of one's own, rows of another pitch
    wide = torch.full((len(lens), q.shape[1] + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 8:8 + q.shape[1]] = q
    out = torch.empty_like(got)
    assert ops.paged_attn_decode_q4(wide[:, 8:8 + q.shape[1]], cache, table, ctx, nq, nkv, hd, scale, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, got)


@pytest.mark.parametrize("nq,nkv,hd,block,lens", [
    (28, 4, 128, 16, [20011]), (8, 2, 64, 32, [9000, 1, 30000]), (16, 2, 128, 64, [5000] * 3 + [1] * 5 + [0] * 4),
    (7, 1, 128, 16, [n * 37 % 1500 for n in range(150)]), (14, 2, 128, 16, [64] * 130)])
def test_attention_long_and_uneven(nq, nkv, hd, block, lens):
    cache, table, ctx = _filled(30, lens, nkv, hd, block)
    q = _randn(40, len(lens), nq * hd).bfloat16()
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, nq, nkv, hd, 0.2)
    _check(got, *_attention_64(q, cache, table, ctx, nq, nkv, hd, 0.2))
    again = ops.paged_attn_decode_q4(q, cache, table, ctx, nq, nkv, hd, 0.2)
    assert torch.equal(got, again)


@pytest.mark.parametrize("repeat", [1, 500, 16384])
@pytest.mark.parametrize("nq,hd", [(7, 128), (12, 64)])
def test_attention_of_very_long_contexts(repeat, nq, hd):
    """The same 1024 tokens over and over (the table names their blocks again): the result does not change, however long the sums.
    Means over many tokens are small beside the values, so sums must not lose their last places: of the result's norm at most the
    rounding to bf16 (2^-8 / sqrt 3 of a binade, 1.3 being the least root mean square in one: 1.74e-3), and p step in fp16 (2^-12 of terms
    of twice a value's deviation, 1024 of them: 6e-4 of results of 0.02)."""
    n = 1024
    kv = _randn(95, n, 2, hd).bfloat16()
    cache = ops.kv4_cache(n // 16, 1, hd)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    ops.rope_kv_write_q4(kv.view(n, -1), torch.zeros_like(slots), slots, cache, 0, 1, hd, 16, 1e6)
    k, v = (t[:, 0].double() for t in ref.kv4_values(cache.cpu(), slots.cpu(), hd, 16))
    q = 0.1 * _randn(96, 1, nq * hd).bfloat16()
    want = torch.softmax(q.double().cpu().view(nq, hd) @ k.T * 0.09, -1) @ v
    table = torch.arange(n // 16, dtype=torch.int32, device="cuda").repeat(repeat)[None].contiguous()
    ctx = torch.tensor([n * repeat], dtype=torch.int32, device="cuda")
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, nq, 1, hd, 0.09).double().cpu().view(nq, hd)
    assert float((got - want).norm() / want.norm()) < math.hypot(1.74e-3, 6e-4) * 1.05


@pytest.mark.parametrize("k_scale,v_scale", [(1.0, 1e-6), (1.0, 3e4), (1e-5, 1.0), (60.0, 1e-20), (1.0, 1e30)])
def test_attention_sizes_of_values(k_scale, v_scale):
    """Steps far from 1: the products are held in types of narrow range inside."""
    lens = [200, 40, 777]
    cache, table, ctx = _filled(50, lens, 2, 128, 16, k_scale=k_scale, v_scale=v_scale)
    q = (_randn(60, 3, 8 * 128) / k_scale).bfloat16()
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, 8, 2, 128, 0.09)
    _check(got, *_attention_64(q, cache, table, ctx, 8, 2, 128, 0.09))


def test_attention_values_that_grow():
    """The largest step arrives last, the largest score too: what was summed before is rescaled."""
    lens = [4000]
    cache, table, ctx = _filled(51, lens, 1, 128, 16)
    n, hd = 4000, 128
    grow = torch.exp(torch.linspace(-12, 12, n, device="cuda"))[:, None, None]
    kv = torch.cat([_randn(52, n, 1, hd) * torch.linspace(0, 3, n, device="cuda")[:, None, None], _randn(53, n, 1, hd) * grow], 1).bfloat16()
    t = torch.arange(n, device="cuda")
    slots = (table[0].long()[t // 16] * 16 + t % 16).to(torch.int32)
    ops.rope_kv_write_q4(kv.view(n, -1), torch.zeros_like(slots), slots, cache, 0, 1, hd, 16, 1e6)
    q = _randn(54, 1, 8 * hd).bfloat16()
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, 8, 1, hd, 0.1)
    _check(got, *_attention_64(q, cache, table, ctx, 8, 1, hd, 0.1))


def test_attention_without_blocks():
    """Table entries that name no block leave their tokens out; requests of which nothing is left get zeros."""
    lens = [100, 70, 16, 333]
    cache, table, ctx = _filled(70, lens, 2, 128, 16, holes=[(0, 0), (0, 3), (1, 4), (2, 0), (3, 7), (3, 8), (3, 20)])
    q = _randn(71, 4, 14 * 128).bfloat16()
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, 14, 2, 128, 0.1)
    _check(got, *_attention_64(q, cache, table, ctx, 14, 2, 128, 0.1))
    assert not bool(got[2].any())
    # lengths beyond the table, and below zero
    ctx2 = torch.tensor([10 ** 9, -5, 16, 333], dtype=torch.int32, device="cuda")
    got = ops.paged_attn_decode_q4(q, cache, table, ctx2, 14, 2, 128, 0.1)
    _check(got[2:], *(t[2:] for t in _attention_64(q, cache, table, ctx2.clamp(0, 400), 14, 2, 128, 0.1)))
    assert not bool(got[1].any())


def test_attention_of_values_that_are_not_finite():
    """A NaN group of a value reaches its own dims only; of a key, its own heads only."""
    lens = [50, 50]
    cache, table, ctx = _filled(80, lens, 2, 128, 16)
    q = _randn(81, 2, 8 * 128).bfloat16()
    clean = ops.paged_attn_decode_q4(q, cache, table, ctx, 8, 2, 128, 0.1)
    row = torch.zeros(1, 4, 128, device="cuda")
    row[0, 3, 33] = float("inf")  # value of head 1, group 1
    slot = (table[0, 2] * 16 + 5).reshape(1)
    ops.rope_kv_write_q4(row.bfloat16().view(1, -1), torch.zeros_like(slot), slot, cache, 0, 2, 128, 16, 1e6)
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, 8, 2, 128, 0.1).view(2, 8, 128)
    bad = torch.zeros(2, 8, 128, dtype=torch.bool, device="cuda")
    bad[0, 4:, 32:64] = True
    assert torch.equal(got.isnan(), bad)
    row[0, 3], row[0, 0, 0] = 0.0, float("nan")  # key of head 0
    ops.rope_kv_write_q4(row.bfloat16().view(1, -1), torch.zeros_like(slot), slot, cache, 0, 2, 128, 16, 1e6)
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, 8, 2, 128, 0.1).view(2, 8, 128)
    bad[:] = False
    bad[0, :4] = True
    assert torch.equal(got.isnan(), bad) and torch.equal(got[1], clean.view(2, 8, 128)[1])


def test_offsets_beyond_32_bits():
    """A cache of more than 4 GB: its last block."""
    nkv, hd, bs = 8, 128, 16
    n_blocks = (1 << 32) // (nkv * 20 * hd) + 40
    cache = torch.empty(n_blocks, nkv, 1, 20 * hd, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[n_blocks - 1, 3, n_blocks - 2]], dtype=torch.int32, device="cuda")
    t = torch.arange(48, device="cuda")
    slots = (table[0].long()[t // bs] * bs + t % bs).to(torch.int32)
    kv = _randn(90, 48, 2 * nkv * hd).bfloat16()
    ops.rope_kv_write_q4(kv, torch.zeros_like(slots), slots, cache, 0, nkv, hd, bs, 1e6)
    small = ops.kv4_cache(3, nkv, hd, bs)
    s2 = torch.arange(48, dtype=torch.int32, device="cuda")
    ops.rope_kv_write_q4(kv, torch.zeros_like(s2), s2, small, 0, nkv, hd, bs, 1e6)
    assert all(torch.equal(a, b) for a, b in zip(ops.kv4_read(cache, slots, hd), ops.kv4_read(small, s2, hd)))
    q = _randn(91, 1, 8 * hd).bfloat16()
    ctx = torch.tensor([48], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.paged_attn_decode_q4(q, cache, table, ctx, 8, nkv, hd, 0.1),
                       ops.paged_attn_decode_q4(q, small, torch.arange(3, dtype=torch.int32, device="cuda")[None], ctx, 8, nkv, hd, 0.1))


def test_streams_and_graphs():
    """Two captured calls replayed on two streams at once, beside an eager one on a third: each has a workspace of its own."""
    sets = []
    for i in range(3):
        cache, table, ctx = _filled(100 + 10 * i, [3000 + 500 * i, 1, 800], 2, 128, 16)
        sets.append((_randn(101 + 10 * i, 3, 14 * 128).bfloat16(), cache, table, ctx))
    want = [ops.paged_attn_decode_q4(*s, 14, 2, 128, 0.1) for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attn_decode_q4(*s, 14, 2, 128, 0.1))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    eager = []
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            eager.append(ops.paged_attn_decode_q4(*sets[2], 14, 2, 128, 0.1))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and all(torch.equal(e, want[2]) for e in eager)


def test_refusals():
    cache = ops.kv4_cache(4, 2, 128)
    q = _randn(1, 2, 8 * 128).bfloat16()
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    ctx = torch.ones(2, dtype=torch.int32, device="cuda")
    ok = dict(q=q, cache=cache, block_tables=table, ctx_lens=ctx, nq=8, nkv=2, hd=128, scale=0.1)
    ops.paged_attn_decode_q4(**ok)
    for bad in (dict(nq=7), dict(nq=34), dict(nkv=1), dict(hd=64), dict(hd=256), dict(q=q.float()), dict(q=q[:, ::2]), dict(q=q[:, :512]),
                dict(q=q[:, 4:]), dict(cache=cache.cpu()), dict(cache=cache.float()), dict(cache=cache[:, :1]), dict(block_tables=table[:1]),
                dict(block_tables=table.long()), dict(ctx_lens=ctx[:1]), dict(ctx_lens=ctx.cpu()), dict(out=q.float())):
        with pytest.raises((RuntimeError, TypeError)):
            ops.paged_attn_decode_q4(**{**ok, **bad})
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            ops.paged_attn_decode_q4(**{**ok, "scale": scale})
    x = _randn(2, 2, 12 * 128).bfloat16()
    w = dict(qkv=x, positions=ctx, slots=ctx, cache=cache, nq=8, nkv=2, hd=128, block_size=16, theta=1e6)
    for bad in (dict(hd=64), dict(nq=7), dict(block_size=32), dict(block_size=8), dict(positions=ctx[:1]), dict(slots=ctx.long()), dict(slots=None),
                dict(qkv=x.half()), dict(qkv=x[:, 2:]), dict(bias=x[0]), dict(theta=0.0), dict(out=x[:1]), dict(cache=cache.cpu())):
        with pytest.raises((RuntimeError, TypeError)):
            ops.rope_kv_write_q4(**{**w, **bad})
    with pytest.raises(RuntimeError):
        ops.kv4_read(cache, ctx, 64)
    with pytest.raises(RuntimeError):
        ops.kv4_read(cache, ctx.long(), 128)
    with pytest.raises(ValueError):
        ops.kv4_cache(4, 2, 96)
    with pytest.raises(ValueError):
        ops.kv4_cache(2 ** 28, 1, 64)
