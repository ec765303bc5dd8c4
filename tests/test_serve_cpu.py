# SPDX-License-Identifier: MIT
"""The CPU path of the 4-bit cache, request layouts and rules on logits: against statements of their own, written with loops."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.ops import reference as ref


def _g(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("hd", [64, 128])
def test_tile_layout_is_a_partition(hd):
    """Every nibble of a tile belongs to one code or one parameter, and every byte to one token."""
    nibbles, owner = [], {}
    for name in "kv":
        byte, shift, ps, pl = ref._kv4_maps(hd)[name]
        for r in range(16):
            for d in range(hd):
                nibbles.append(2 * int(byte[r, d]) + int(shift[r, d]) // 4)
                assert owner.setdefault(int(byte[r, d]), r) == r
            for a in range(hd // 32):
                for at in (ps, pl):
                    nibbles += [2 * int(at[r, a]) + j for j in range(4)]
    assert sorted(nibbles) == list(range(40 * hd))


@pytest.mark.parametrize("hd,block", [(64, 16), (128, 48)])
def test_cache_holds_the_formula(hd, block):
    """Within half a step of every element: step = bf16((max - min) / 15), so half of it and the part of its rounding that 15 steps add up
    to, 15 * 2^-9 / 15 of the range."""
    nkv, rows = 3, 40
    cache = ops.kv4_cache(3 if block == 16 else 1, nkv, hd, block, "cpu")
    kv = (torch.randn(rows, 2 * nkv, hd, generator=_g(1)) * 3 + torch.randn(hd, generator=_g(2))).bfloat16()
    slots = torch.randperm(48, generator=_g(3))[:rows].to(torch.int32)
    slots[7] = -1
    ops.rope_kv_write_q4(kv.view(rows, -1).clone(), torch.zeros(rows, dtype=torch.int32), slots, cache, 0, nkv, hd, block, 1e6)
    k, v = ref.kv4_values(cache, slots.clamp(min=0), hd, block)
    for got, x in ((k, kv[:, :nkv]), (v, kv[:, nkv:])):
        x = x.double().unflatten(-1, (-1, 32))
        span = x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)
        err = (got.double().unflatten(-1, (-1, 32)) - x).abs()
        keep = torch.arange(rows) != 7
        assert bool((err <= span * (0.5 / 15 * (1 + 2 ** -8) + 2 ** -8))[keep].all())
    assert not bool(ops.kv4_read(cache, slots, hd, block)[0][7].any())


def test_rope_matches_the_bf16_path():
    x = torch.randn(5, 4 * 64, generator=_g(4))
    pos = torch.tensor([0, 3, 100, 7, 50], dtype=torch.int32)
    a = ops.rope_kv_write_q4(x.clone(), pos, None, None, 2, 1, 64, 16, 1e4)
    b = ops.rope_kv_write(x.clone(), pos, None, None, None, 2, 1, 64, 16, 1e4)
    assert float((a - b).abs().max()) < 1e-4  # (fp32 angles there: 100 rad * 2^-23, twice)


def test_attention_over_the_cache():
    nq, nkv, hd, bs = 4, 2, 64, 16
    cache = ops.kv4_cache(6, nkv, hd, bs, "cpu")
    kv = torch.randn(40, 2 * nkv, hd, generator=_g(5)).bfloat16()
    table = torch.tensor([[4, 1, 2], [5, -1, 9]], dtype=torch.int32)
    t = torch.arange(40)
    slots = (table[0].long()[t // 16] * 16 + t % 16).to(torch.int32)
    zero = torch.zeros(40, dtype=torch.int32)
    ops.rope_kv_write_q4(kv.view(40, -1).clone(), zero, slots, cache, 0, nkv, hd, bs, 1e6)
    ops.rope_kv_write_q4(kv[:16].view(16, -1).clone(), zero[:16], (80 + t[:16]).to(torch.int32), cache, 0, nkv, hd, bs, 1e6)
    q = torch.randn(2, nq * hd, generator=_g(6))
    got = ops.paged_attn_decode_q4(q, cache, table, torch.tensor([40, 40], dtype=torch.int32), nq, nkv, hd, 0.125)
    k, v = (x.double() for x in ref.kv4_values(cache, slots, hd, bs))
    for b, n in ((0, 40), (1, 16)):
        for h in range(nq):
            s = k[:n, h // 2] @ q[b].double().view(nq, hd)[h] * 0.125
            want = torch.softmax(s, 0) @ v[:n, h // 2]
            assert float((got[b].view(nq, hd)[h] - want).abs().max()) < 1e-5
    assert not bool(ops.paged_attn_decode_q4(q, cache, table, torch.tensor([0, 0], dtype=torch.int32), nq, nkv, hd, 0.125).any())


def test_layout_by_hand():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    table, ring = i32(3, -1, -1, 7, 5, -1, 2, -1, -1).view(3, 3), i32(6, -1, -1, -1, 1, 0, 4, 8)
    r = ops.paged_layout(i32(20, -1, 1), i32(10, 20, 16), table, ring, i32(4, 5, 0), 23, 16)
    assert r.cu.tolist() == [0, 20, 20, 21] and r.ctx_lens.tolist() == [30, 0, 17]
    assert r.positions.tolist() == list(range(10, 30)) + [16, 0, 0]
    assert r.slots.tolist() == list(range(58, 64)) + list(range(16, 30)) + [0, -1, -1]
    assert table.tolist() == [[3, 1, -1], [7, 5, -1], [2, 0, -1]]
    assert r.free_range.tolist() == [6, 5, 0] and ring.tolist() == [6, 7, 5, -1, 1, 0, 4, 8]
    short = ops.paged_layout(i32(100), i32(0), torch.full((1, 7), -1, dtype=torch.int32), i32(4, 9), i32(0, 1, 0), 100, 16)
    assert short.free_range.tolist() == [1, 0, 6] and (short.slots >= 0).sum() == 16 and short.slots[0] == 64


def test_rules_by_hand():
    r = ops.LogitRules.empty(2, 40, "cpu", bias_entries=3, masked=True)
    ops.count_tokens(r, torch.tensor([5, 5, 39, 7, 5, 99, -1], dtype=torch.int32), torch.tensor([0, 3, 7], dtype=torch.int32),
                     torch.tensor([1, 3], dtype=torch.int32))
    assert r.counts[0, 5] == 1 and r.counts[0, 39] == 1 and int(r.counts.sum()) == 2
    assert [int(w) & 0xffffffff for w in r.seen.flatten()] == [32, 1 << 7, 32 | 128, 0]
    r.penalties[:] = torch.tensor([2.0, 0.25, 0.5])
    r.bias_ids[0], r.bias[0] = torch.tensor([3, -1, 3]), torch.tensor([1.5, 100.0, 2.0])
    r.mask[1, 0], r.mask[1, 1] = 1 << 5 | 1 << 9, 0
    x = torch.ones(2, 40)
    x[:, 7] = -1.0
    y = ops.logits_process(x, r)
    assert y[0, 5] == 0.5 - 0.5 - 0.25 and y[0, 39] == -0.25 and y[0, 3] == 4.5 and y[0, 7] == -1 and y[0, 0] == 1
    assert y[1, 5] == 0.5 and y[1, 9] == 1 and int((y[1] == -math.inf).sum()) == 38
    assert ops.logits_argmax(x, r)[0].tolist() == [3, 9]
    r.mask[1] = 0
    assert ops.logits_argmax(x, r)[0].tolist() == [3, -1]


def test_refusals():
    with pytest.raises(ValueError):
        ops.kv4_cache(2, 1, 80, 16, "cpu")
    with pytest.raises(ValueError):
        ops.kv4_cache(2, 1, 64, 24, "cpu")
    cache = ops.kv4_cache(2, 1, 64, 16, "cpu")
    x, i = torch.zeros(2, 3 * 64), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(hd=32), dict(nq=2), dict(slots=None), dict(cache=cache.float()), dict(block_size=32), dict(positions=i[:1])):
        with pytest.raises(ValueError):
            ops.rope_kv_write_q4(**{**dict(qkv=x, positions=i, slots=i, cache=cache, nq=1, nkv=1, hd=64, block_size=16, theta=1e4), **bad})
    with pytest.raises(ValueError):
        ops.count_tokens(ops.LogitRules.empty(2, 10, "cpu"), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.LogitRules(bias_ids=i)
