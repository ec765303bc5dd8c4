# SPDX-License-Identifier: MIT
"""Log probabilities, entropy and most likely tokens (csrc/score_kernels.cu) against 64-bit statements.

Tolerances.  A term e^t has the error of its argument (two roundings of at most |t| 2^-24 each; weighed by e^t, |t| e^t < 0.37) and of the
exponential (2^-22): below 2^-21.  A thread adds up at most 80 terms a lap and up to 13 sums are joined, each addition 2^-24: S is
off by less than 2^-21 + 100 * 2^-24 < 2^-17 of itself and log S by as much; x - m and the subtraction are rounded: 2^-23 of their values.
T's terms have the error of t too, and a joined distance once more: T / S is off by less than 2^-16 (1 + |T / S|)."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops

pytestmark = pytest.mark.gpu


def _g(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(seed, rows, n, dtype, spread=4.0):
    return (torch.randn(rows, n, generator=_g(seed), device="cuda") * spread).to(dtype)


def _check(x, ids, got, top, offset=0, vocab=None):
    """x: the logits that the call was given."""
    rows = x.shape[0]
    n = x.shape[1] if vocab is None else max(0, min(x.shape[1], vocab - offset))
    x = x[:, :n].double()
    logp = x - x.amax(-1, keepdim=True)  # (first: next to 10^38 a logarithm is lost in 64 bits too)
    logp = logp - torch.log(torch.exp(logp).sum(-1, keepdim=True))
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    at = ids.long().view(rows, -1) - offset
    ok = (ids.view(rows, -1) >= 0) & (at >= 0) & (at < n)
    want = torch.where(ok, logp.gather(1, torch.where(ok, at, 0)), -math.inf).view(ids.shape)

    def near(a, b, tol):
        a = a.double()
        fine = torch.isfinite(b)
        assert torch.equal(fine, torch.isfinite(a)) and torch.equal(a[~fine], b[~fine])
        assert ((a - b).abs()[fine] <= tol[fine]).all()

    near(got.logprobs, want, 2.0 ** -17 + 2.0 ** -22 * want.abs())
    near(got.entropy, entropy, 2.0 ** -15 * (1 + entropy.abs()))
    if top:
        order = torch.sort(x, dim=-1, descending=True, stable=True)
        k = min(top, n)
        there = order.values[:, :k] > -math.inf
        assert torch.equal(got.top_ids[:, :k], torch.where(there, order.indices[:, :k] + offset, -1).to(torch.int32))
        assert (got.top_ids[:, k:] == -1).all() and (got.top_logprobs[:, k:] == -math.inf).all()
        best = logp.gather(1, order.indices[:, :k])
        near(got.top_logprobs[:, :k], torch.where(there, best, -math.inf), 2.0 ** -17 + 2.0 ** -22 * best.abs())
    assert got.top_ids.shape == got.top_logprobs.shape == (rows, top) and got.top_ids.dtype == torch.int32


# one element, less than a vector, tile edges, a lap of one block and of eight, more than a lap, a head's width
@pytest.mark.parametrize("n", [1, 7, 8, 2051, 20480, 20481, 32003, 152064, 200001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_sizes(n, dtype, top):
    for rows in (1, 3, 33):
        x = _logits(n + top, rows, n, dtype)
        ids = torch.randint(0, n, (rows,), generator=_g(1), device="cuda", dtype=torch.int32)
        _check(x, ids, ops.token_logprobs(x, ids, top), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("start", [1, 3, 5])
@pytest.mark.parametrize("n", [2, 6, 1001, 50021])
def test_rows_off_their_vectors(dtype, start, n):
    wide = _logits(7, 5, n + 13, dtype)
    x = wide[:, start:start + n]
    ids = torch.randint(0, n, (5, 3), generator=_g(2), device="cuda", dtype=torch.int32)
    got = ops.token_logprobs(x, ids, 9)
    _check(x, ids, got, 9)
    whole = ops.token_logprobs(x.contiguous(), ids, 9)
    assert torch.equal(got.top_ids, whole.top_ids)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [40, 5000, 152064, 170000])
def test_ties_go_to_the_lowest_index(dtype, n):
    same = torch.full((2, n), -3.0, dtype=dtype, device="cuda")
    zeros = torch.zeros(2, n, dtype=dtype, device="cuda")
    zeros[:, ::2] = -0.0
    few = torch.randint(0, 3, (2, n), generator=_g(3), device="cuda").to(dtype)
    late = same.clone()
    late[:, -40:] = 1.0
    ids = torch.tensor([0, n - 1], dtype=torch.int32, device="cuda")
    for x in (same, zeros, few, late):
        _check(x, ids, ops.token_logprobs(x, ids, 32), 32)


@pytest.mark.parametrize("top", [2, 20, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [20480, 81920, 190000])
def test_great_logits_of_few_threads(top, dtype, n):
    """More logits above the border than the list holds: those of a few neighbouring threads are the greatest of the row."""
    per = 16 // dtype.itemsize
    vec = torch.arange(n, device="cuda") // per
    x = _logits(11, 3, n, dtype, 1.0)
    great = (vec % 256) // 4 < top - 1
    x = torch.where(great, x + 40, x)
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    _check(x, ids, ops.token_logprobs(x, ids, top), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [300, 152064])
def test_masked(dtype, n):
    x = _logits(5, 7, n, dtype)
    low = torch.finfo(dtype).min
    x[0] = -math.inf               # nothing is left
    x[1, :] = -math.inf
    x[1, n // 2] = 2.0             # one token
    x[2] = torch.where(torch.rand(n, generator=_g(6), device="cuda") < 0.9, -math.inf, x[2].float()).to(dtype)
    x[3] = low                     # all of the lowest value: as likely as one another
    x[4] = torch.where(torch.rand(n, generator=_g(8), device="cuda") < 0.9, low, x[4].float()).to(dtype)
    x[5, ::3] = -math.inf
    x[5, 1] = torch.finfo(dtype).max
    ids = torch.tensor([0, n // 2, 5, 7, 9, 1, n - 1], dtype=torch.int32, device="cuda")
    for top in (0, 4):
        got = ops.token_logprobs(x, ids, top)
        assert got.logprobs[0] == -math.inf and got.entropy[0] == 0 and (got.top_ids[0] == -1).all() and (got.top_logprobs[0] == -math.inf).all()
        _check(x[1:], ids[1:], ops.TokenLogprobs(*(t[1:] for t in got)), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [9, 152064])
@pytest.mark.parametrize("at", [0, 8])
def test_rows_that_are_no_numbers(dtype, n, at):
    x = _logits(9, 5, n, dtype)
    keep = x.clone()
    x[1, at] = math.nan
    x[2, at] = math.inf
    x[3] = -math.inf
    x[3, at] = math.nan
    ids = torch.full((5,), 3, dtype=torch.int32, device="cuda")
    got = ops.token_logprobs(x, ids, 4)
    for r in (1, 2, 3):
        assert torch.isnan(got.logprobs[r]) and torch.isnan(got.entropy[r]) and torch.isnan(got.top_logprobs[r]).all()
    for r in (0, 4):  # the others are as they were
        _check(keep[r:r + 1], ids[r:r + 1], ops.TokenLogprobs(*(t[r:r + 1] for t in got)), 4)


@pytest.mark.parametrize("offset,vocab", [(0, 900), (1000, 1900), (1000, 1000), (500, 100), (0, 0), (2000, None)])
def test_shards_and_padding(offset, vocab):
    x = _logits(4, 6, 1000, torch.bfloat16)
    if vocab is not None:
        x[:, max(0, vocab - offset):] = math.nan  # what stands behind the vocabulary is of no account
    ids = torch.tensor([[offset, offset + 3, -1, 0], [offset + 999, offset + 1000, 2 ** 31 - 1, -2 ** 31]] * 3, dtype=torch.int32, device="cuda")
    got = ops.token_logprobs(x, ids, 5, offset, vocab)
    if vocab is not None and vocab <= offset:
        assert (got.logprobs == -math.inf).all() and (got.entropy == 0).all() and (got.top_ids == -1).all()
        return
    _check(x, ids, got, 5, offset, vocab)


@pytest.mark.parametrize("world", [2, 8])
@pytest.mark.parametrize("top", [0, 7])
def test_joined_shards(world, top):
    vocab, rows = 32003, 5
    per = -(-vocab // world)
    x = torch.nn.functional.pad(_logits(4, rows, vocab, torch.bfloat16), (0, per * world - vocab), value=math.nan)
    x[1, : per + 3] = -math.inf  # a whole shard masked
    ids = torch.randint(0, vocab, (rows, 2), generator=_g(2), device="cuda", dtype=torch.int32)
    shards = [ops.token_logprob_parts(x[:, r * per:(r + 1) * per], ids, top, r * per, vocab) for r in range(world)]
    got = ops.TokenLogprobs(*ops.ref.token_logprobs_of(*ops.ref.join_token_logprobs(shards)))
    _check(x, ids, got, top, 0, vocab)


def test_many_tokens_of_a_row():
    x = _logits(4, 3, 70000, torch.bfloat16)
    ids = torch.randint(-5, 70005, (3, 700), generator=_g(2), device="cuda", dtype=torch.int32)
    _check(x, ids, ops.token_logprobs(x, ids), 0)
    none = ops.token_logprobs(x, ids[:, :0], 2)
    assert none.logprobs.shape == (3, 0)
    _check(x, ids[:, :0], none, 2)
    empty = ops.token_logprobs(x[:0], ids[:0], 2)
    assert empty.logprobs.shape == (0, 700) and empty.top_ids.shape == (0, 2)


def test_rows_beyond_32_bits():
    """Offsets of rows that 32 bits do not hold."""
    wide = torch.empty(3, 1500000000, dtype=torch.bfloat16, device="cuda")
    x = wide[:, :5000]
    x.copy_(_logits(4, 3, 5000, torch.bfloat16))
    ids = torch.tensor([4, 5, 6], dtype=torch.int32, device="cuda")
    _check(x, ids, ops.token_logprobs(x, ids, 3), 3)


def test_streams_and_graphs():
    xs = [_logits(20 + i, 9, 152064, torch.bfloat16) for i in range(3)]
    ids = torch.arange(9, dtype=torch.int32, device="cuda")
    want = [ops.token_logprobs(x, ids, 6) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(10):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(ops.token_logprobs(x, ids, 6))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i % 3]))
    # two graphs over the same input buffer, replayed in turn
    buf = xs[0].clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.token_logprobs(buf, ids, 6))
        graphs.append(g)
    for i in (1, 2, 0):
        buf.copy_(xs[i])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want[i]))


def test_refusals():
    x = _logits(4, 3, 100, torch.bfloat16)
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.token_logprobs(x, ids, 33), lambda: ops.token_logprobs(x, ids, -1), lambda: ops.token_logprobs(x, ids.long()),
                lambda: ops.token_logprobs(x, ids[:2]), lambda: ops.token_logprobs(x, ids.cpu()), lambda: ops.token_logprobs(x.half(), ids),
                lambda: ops.token_logprobs(x[0], ids), lambda: ops.token_logprobs(x, ids, 1, -1), lambda: ops.token_logprobs(x, ids, 1, 2 ** 31 - 50),
                lambda: ops.token_logprobs(x.t(), ids), lambda: ops.token_logprobs(x, ids, 1, 0, -4),
                lambda: ops.token_logprobs(x[:1].expand(3, -1), ids)):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
