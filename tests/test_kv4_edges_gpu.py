# SPDX-License-Identifier: MIT
"""The 4-bit key/value cache on the GPU where its numbers leave the ordinary: values without steps, queries that are no numbers, waits that run out.
Tolerances and 64-bit statements are those of test_kv4_gpu.py."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine, Qwen2Config, Qwen2Model
from barlink_sm86_b200.parallel import TPComm
from test_kv4_gpu import _attention_64, _check, _filled, _randn

pytestmark = pytest.mark.gpu


def _rewrite(cache, table, request, kv, block=16, first=0):
    """Keys and values kv [tokens, 2 nkv, hd] in place of a request's tokens from `first` on."""
    n, heads, hd = kv.shape
    t = torch.arange(first, first + n, device="cuda")
    slots = (table[request].long()[t // block] * block + t % block).to(torch.int32)
    ops.rope_kv_write_q4(kv.bfloat16().reshape(n, -1), torch.zeros_like(slots), slots, cache, 0, heads // 2, hd, block, 1e6)


@pytest.mark.parametrize("level", [1e-25, 1.0, -1e10, 1e12, 1e30, -3e38])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (12, 1, 64)])
def test_values_without_steps(level, nq, nkv, hd):
    """Groups of one value each (step 0), whatever its size: the mean over tokens is one of numbers that fp32 holds."""
    lens = [1, 40, 700]
    cache, table, ctx = _filled(200, lens, nkv, hd, 16)
    for i, n in enumerate(lens):
        kv = _randn(201 + i, n, 2 * nkv, hd)
        kv[:, nkv:] = level * (0.25 + 0.75 * torch.rand(n, nkv, 1, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda"))
        _rewrite(cache, table, i, kv)
    q = _randn(210, 3, nq * hd).bfloat16()
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, nq, nkv, hd, 0.1)
    _check(got, *_attention_64(q, cache, table, ctx, nq, nkv, hd, 0.1))


def _again(table, n, repeat, block=16):
    """A table that names a request's n tokens (whole blocks) over and over, so that a warp's run holds many of them; the softmax's mean
    does not change.  With its length."""
    return table[:, :n // block].repeat(1, repeat).contiguous(), torch.tensor([n * repeat], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("repeat", [1, 512])
@pytest.mark.parametrize("grows", [False, True])
def test_values_without_steps_behind_zeros(grows, repeat):
    """Zeros, then constants, then ordinary values, one group of them constant: the sums are in scale for each of them.  grows: the
    scores rise along the way."""
    n, nkv, hd, nq = 1600, 1, 128, 8
    cache, table, ctx = _filled(220, [n], nkv, hd, 16)
    kv = _randn(221, n, 2, hd)
    if grows:
        kv[:, 0] = torch.linspace(0, 1, n, device="cuda")[:, None]
    kv[:400, 1] = 0
    kv[400:800, 1] = 1e12
    kv[800:1200, 1] *= 1e-12
    kv[1200:, 1, 32:64] = -1e25
    _rewrite(cache, table, 0, kv)
    q = torch.full((1, nq * hd), 1.0, device="cuda").bfloat16() if grows else _randn(222, 1, nq * hd).bfloat16()
    for m in (n, 800, 1200, 400):
        t, c = _again(table, m, repeat)
        ctx.fill_(m)
        got = ops.paged_attn_decode_q4(q, cache, t, c, nq, nkv, hd, 0.1)
        _check(got, *_attention_64(q, cache, table, ctx, nq, nkv, hd, 0.1))


@pytest.mark.parametrize("repeat", [1, 512])
def test_a_group_at_the_end_of_the_range(repeat):
    """3e38 beside ordinary values, and behind them: its own dims."""
    n, hd, nq = 912, 128, 4
    cache, table, ctx = _filled(230, [n], 1, hd, 16)
    kv = _randn(231, n, 2, hd)
    kv[500:, 1, 64:96] = 3e38
    _rewrite(cache, table, 0, kv)
    q = _randn(232, 1, nq * hd).bfloat16()
    t, c = _again(table, n, repeat)
    got = ops.paged_attn_decode_q4(q, cache, t, c, nq, 1, hd, 0.1)
    want, size = _attention_64(q, cache, table, ctx, nq, 1, hd, 0.1)
    own = (torch.arange(nq * hd) % hd // 32 == 2)[None]
    _check(got[:, own[0].cuda()], want[own][None], size[own][None])
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("repeat", [1, 512])
@pytest.mark.parametrize("nq,hd", [(8, 128), (16, 128), (3, 64), (12, 64)])
def test_a_query_that_is_no_number_spoils_its_own_head(nq, hd, repeat):
    """Head 0 is NaN; head 1's scores rise by 46 in log2 late in the context, where nothing else moves."""
    n = 1024
    cache, table, ctx = _filled(240, [n], 1, hd, 16)
    kv = _randn(241, n, 2, hd)
    kv[:, 0] *= 0.01
    kv[993:, 0, :32] = 10.0
    _rewrite(cache, table, 0, kv)
    t, c = _again(table, n, repeat)
    q = torch.zeros(1, nq, hd, device="cuda")
    q[0, 1, :32] = 1.0
    want, size = _attention_64(q.view(1, -1).bfloat16(), cache, table, ctx, nq, 1, hd, 0.1)
    q[0, 0, 5] = math.nan
    got = ops.paged_attn_decode_q4(q.view(1, -1).bfloat16(), cache, t, c, nq, 1, hd, 0.1)
    assert bool(got[0, :hd].isnan().all())
    _check(got[:, hd:], want[:, hd:], size[:, hd:])


@pytest.fixture
def polls(ext):
    """Sets how often a wait looks; back to what it was afterwards, and the error word to 0."""
    before = ext.kv4_wait_polls(0)
    yield ext.kv4_wait_polls
    ext.kv4_wait_polls(before)
    torch.cuda.synchronize()
    ext.kv4_error_clear(0)


@pytest.mark.parametrize("nq,nkv,hd,lens", [(14, 2, 128, [3000, 0, 1, 800]), (16, 1, 128, [90000]), (8, 8, 64, [700] * 300), (12, 1, 64, [40] * 9)])
def test_a_wait_that_runs_out(ext, polls, nq, nkv, hd, lens):
    """A run that gives up says so and leaves NaN, not what the workspace held; requests without tokens and later calls are as ever."""
    polls(1 << 24)
    cache, table, ctx = _filled(250, lens, nkv, hd, 16)
    q = _randn(251, len(lens), nq * hd).bfloat16()
    want = ops.paged_attn_decode_q4(q, cache, table, ctx, nq, nkv, hd, 0.1)
    torch.cuda.synchronize()
    assert ext.kv4_error_flag(0) == 0
    polls(0)
    got = ops.paged_attn_decode_q4(q, cache, table, ctx, nq, nkv, hd, 0.1)
    assert ext.kv4_error_flag(0) == 1
    for i, n in enumerate(lens):
        assert bool(got[i].isnan().all()) if n else not bool(got[i].any())
    ext.kv4_error_clear(0)
    # some look once or twice, and may be in time: a head is right or NaN, and NaN only where the word says so
    for n in (1, 2):
        polls(n)
        got = ops.paged_attn_decode_q4(q, cache, table, ctx, nq, nkv, hd, 0.1)
        bad = got.view(-1, hd).isnan()
        assert torch.equal(bad.all(1), bad.any(1)) and bool(bad.any()) == bool(ext.kv4_error_flag(0))
        assert torch.equal(torch.where(bad, 0, got.view(-1, hd)), torch.where(bad, 0, want.view(-1, hd)))
        ext.kv4_error_clear(0)
    polls(1 << 24)
    assert torch.equal(ops.paged_attn_decode_q4(q, cache, table, ctx, nq, nkv, hd, 0.1), want)
    assert ext.kv4_error_flag(0) == 0


def test_the_engine_reports_a_wait_that_ran_out(ext, polls):
    polls(1 << 24)
    cfg = Qwen2Config(hidden=512, layers=2, n_heads=4, n_kv_heads=2, head_dim=128, intermediate=1024, vocab=1000, name="test")
    model = Qwen2Model(cfg, TPComm.single(), "cuda:0", torch.bfloat16, seed=3)
    eng = DecodeEngine(model, 2, 200, use_graph=False, kv_bits=4)
    prompt = torch.arange(60, dtype=torch.int32, device="cuda")
    first = eng.start(prompt, [40, 20]).cpu().pin_memory()
    want = eng.step_host(first).clone()
    eng.finish([0, 1])
    eng.start(prompt, [40, 20])
    polls(0)
    with pytest.raises(RuntimeError, match="gave up"):
        eng.step_host(first)
    polls(1 << 24)
    eng.check()  # (reported once)
    eng.finish([0, 1])
    eng.start(prompt, [40, 20])
    assert torch.equal(eng.step_host(first), want)


def test_a_cache_without_blocks():
    """Nothing is there: zeros."""
    cache = ops.kv4_cache(0, 2, 128)
    slots = torch.tensor([0, -1, 5], dtype=torch.int32, device="cuda")
    assert not any(bool(t.any()) for t in ops.kv4_read(cache, slots, 128))
    q = _randn(260, 3, 4 * 128).bfloat16()
    assert not bool(ops.paged_attn_decode_q4(q, cache, slots[:, None].contiguous(), slots.abs(), 4, 2, 128, 0.1).any())


@pytest.mark.parametrize("nq,nkv,hd", [(3, 2, 128), (5, 1, 64)])
@pytest.mark.parametrize("more", [0, 1, 2, 7])
def test_write_on_both_sides_of_the_line(nq, nkv, hd, more):
    """As many rows as get blocks of their own, and more: the same rows and bytes as in parts."""
    rows = (22 if hd == 128 else 7) * torch.cuda.get_device_properties(0).multi_processor_count + more
    x = _randn(270, rows, (nq + 2 * nkv) * hd).bfloat16()
    pos = torch.arange(rows, dtype=torch.int32, device="cuda") * 11
    slots = torch.arange(rows, dtype=torch.int32, device="cuda").flip(0).contiguous()
    caches = [ops.kv4_cache(rows // 16 + 1, nkv, hd).fill_(0xFF) for _ in range(2)]
    whole = ops.rope_kv_write_q4(x.clone(), pos, slots, caches[0], nq, nkv, hd, 16, 1e6)
    parts = [ops.rope_kv_write_q4(x[i:i + 500].clone(), pos[i:i + 500], slots[i:i + 500], caches[1], nq, nkv, hd, 16, 1e6) for i in range(0, rows, 500)]
    assert torch.equal(whole, torch.cat(parts)) and torch.equal(*caches)
