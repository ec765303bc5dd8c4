# SPDX-License-Identifier: MIT
"""Request layouts, token counts and rules on logits (csrc/serve_kernels.cu) against their statements: whole numbers are equal, and so
are logits, whose operations are rounded one by one in the same order on both sides."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.ops import reference as ref

pytestmark = pytest.mark.gpu


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _ints(seed, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=_g(seed), dtype=torch.int32)


def _layout_case(seed, batch, new, past, bs, spare, ended=0.1):
    new_lens, past_lens = _ints(seed, 0, new, batch), _ints(seed + 1, 0, past, batch)
    width = max(1, -(-(past + new) // bs))
    new_lens[torch.rand(batch, generator=_g(seed + 2)) < ended] = -1
    n = batch * width + 2
    ids = torch.randperm(n, generator=_g(seed + 3)).to(torch.int32)
    table = ids[:batch * width].view(batch, width).clone()
    held = torch.arange(width)[None] < ((past_lens + bs - 1) // bs)[:, None]
    free = torch.cat([table[~held], ids[batch * width:]])
    head = n * 2 // 3
    ring = torch.full((n,), -9, dtype=torch.int32)
    ring[(head + torch.arange(free.numel())) % n] = free
    table = torch.where(held, table, -1).contiguous()
    left = max(0, free.numel() - spare) if spare is not None else free.numel()
    return new_lens, past_lens, table, ring, torch.tensor([head, left, 0], dtype=torch.int32)


def _layout_both(args, tokens, bs):
    cpu = [t.clone() for t in args]
    gpu = [t.cuda() for t in args]
    want = ops.paged_layout(*cpu, tokens, bs)
    got = ops.paged_layout(*gpu, tokens, bs)
    for name, a, b in zip(want._fields, want, got):
        assert torch.equal(a, b.cpu()), name
    assert torch.equal(cpu[2], gpu[2].cpu()) and torch.equal(cpu[3], gpu[3].cpu())
    return got


@pytest.mark.parametrize("batch,new,past,bs", [(1, 1, 0, 16), (1, 5000, 0, 16), (3, 40, 100, 32), (64, 1, 4000, 16), (33, 300, 77, 5),
                                               (1024, 3, 40, 16), (1025, 17, 200, 64), (5000, 2, 31, 16), (8192, 1, 15, 16)])
@pytest.mark.parametrize("spare", [None, 0, 10 ** 9])
def test_layout(batch, new, past, bs, spare):
    if spare == 0 and batch > 2000:
        spare = 500
    args = _layout_case(batch + new, batch, new, past, bs, spare)
    total = int(args[0].clamp(min=0).sum())
    for tokens in {total, total + 37, max(0, total - 3)}:
        _layout_both(args, tokens, bs)


@pytest.mark.parametrize("batch,per,tokens", [(1, 1, 1), (5, 1, 5), (64, 1, 64), (7, 4, 28), (7, 4, 25), (3, 2, 9), (700, 5, 3500), (2000, 3, 6000)])
def test_layout_with_equal_rows(batch, per, tokens):
    """Requests that rest or have ended keep their rows, empty; more tokens than rows: the first ones."""
    args = _layout_case(batch + per, batch, per + 1, 60, 16, None, ended=0.2)
    cpu, gpu = [t.clone() for t in args], [t.cuda() for t in args]
    want = ops.paged_layout(*cpu, tokens, 16, rows_per_request=per)
    got = ops.paged_layout(*gpu, tokens, 16, rows_per_request=per)
    for name, a, b in zip(want._fields, want, got):
        assert torch.equal(a, b.cpu()), name
    for b in range(min(batch, tokens // per)):
        n = max(int(args[0][b]), 0)
        assert got.positions[b * per:(b + 1) * per].tolist() == [int(args[1][b]) + i if i < n else 0 for i in range(per)]


def test_layout_edges():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    # nothing new at all; all requests ended; a table too narrow; entries of a shortage before are not given back
    _layout_both((i32(0, 0), i32(0, 5), i32(-1, -1, 3, -1).view(2, 2), i32(0, 1, 2), i32(0, 3, 0)), 4, 16)
    _layout_both((i32(-1, -1), i32(40, 16), i32(0, -1, 2, 5, 9, 9).view(2, 3), i32(1, 3, 4, -9, -9, -9), i32(0, 3, 0)), 0, 16)
    _layout_both((i32(50, 3), i32(20, 0), i32(7, 6, -1, -1).view(2, 2), i32(1, 2, 3), i32(2, 3, 0)), 60, 16)
    # a free list that is full already: nothing is written over
    _layout_both((i32(-1), i32(32), i32(4, 5).view(1, 2), i32(0, 1, 2), i32(1, 3, 0)), 1, 16)
    # lengths below zero and ranges out of order are bounded
    _layout_both((i32(2, 2), i32(-7, 3), i32(-1, 5).view(2, 1), i32(0, 1, 2), i32(1, 3, 0)), 4, 16)


@pytest.mark.parametrize("head", [-1, -2 ** 31, 5, 2 ** 31 - 1])
def test_layout_of_a_head_outside_the_ring(head):
    """A head that names no entry is taken modulo the ring's length."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    _layout_both((i32(20, -1), i32(0, 16), i32(-1, -1, 3, -1).view(2, 2), i32(0, 1, 2), i32(head, 2, 0)), 20, 16)


def test_layout_of_a_run_in_place():
    """Prompts, then steps captured in a graph, in place, while one request ends: no block has two holders, positions count on."""
    bs, batch, width, n = 16, 5, 8, 24
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    ring = torch.arange(n, dtype=torch.int32, device="cuda")
    rng = torch.tensor([0, n, 0], dtype=torch.int32, device="cuda")
    prompt = torch.tensor([30, 1, 16, 0, 47], dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(prompt)
    first = ops.paged_layout(prompt, zero, table, ring, rng, 94, bs)
    ctx, free = first.ctx_lens.clone(), first.free_range.clone()
    new = torch.ones(batch, dtype=torch.int32, device="cuda")
    step = ops.PagedLayout(*(torch.empty(s, dtype=torch.int32, device="cuda") for s in (batch + 1, batch, batch)), ctx, free)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.paged_layout(new, ctx, table, ring, free, batch, bs, into=step)
    lens = prompt.clone()
    for i in range(20):
        if i == 9:
            ended = new.clone()
            ended[0] = -1
            new.copy_(ended)
        g.replay()
        lens = torch.where(new < 0, 0, lens + new)
        assert torch.equal(ctx, lens) and int(free[2]) == 0
        if i == 9:
            new[0] = 0
        rows = [b for b in range(batch) if int(new[b]) == 1]
        for j, b in enumerate(rows):
            p = int(lens[b]) - 1
            assert int(step.positions[j]) == p and int(step.slots[j]) == int(table[b, p // bs]) * bs + p % bs
        held = [x for b in range(batch) for x in table[b, : -(-int(lens[b]) // bs)].tolist()]
        left = [int(ring[(int(free[0]) + k) % n]) for k in range(int(free[1]))]
        assert sorted(held + left) == list(range(n))


@pytest.mark.parametrize("rows,vocab,hist", [(1, 50, 3), (1, 152064, 5000), (7, 32003, 700), (64, 1000, 2500), (130, 33, 9)])
@pytest.mark.parametrize("prompts", [False, True])
def test_count_tokens(rows, vocab, hist, prompts):
    lens = _ints(1, 0, hist, rows)
    cu = torch.zeros(rows + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(lens, 0)
    ids = (torch.rand(int(cu[-1]) + 5, generator=_g(2)) ** 3 * (vocab + 3)).to(torch.int32) - 1  # some out of the vocabulary
    prompt = _ints(3, 0, hist, rows) if prompts else None
    cpu, gpu = ops.LogitRules.empty(rows, vocab, "cpu"), ops.LogitRules.empty(rows, vocab)
    gpu.counts.fill_(3)
    gpu.seen.fill_(5)
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    ops.count_tokens(cpu, ids, cu, prompt, reset=True)
    ops.count_tokens(gpu, c(ids), c(cu), c(prompt), reset=True)
    assert torch.equal(cpu.counts, gpu.counts.cpu()) and torch.equal(cpu.seen, gpu.seen.cpu())
    one = _ints(4, -1, vocab, rows)  # a step's tokens on top
    ops.count_tokens(cpu, one)
    ops.count_tokens(gpu, c(one))
    assert torch.equal(cpu.counts, gpu.counts.cpu()) and torch.equal(cpu.seen, gpu.seen.cpu())


def _rules(seed, rows, vocab, bias, mask, pen=True, hist=200):
    r = ops.LogitRules.empty(rows, vocab, "cpu", bias_entries=bias, masked=mask)
    r.penalties.copy_(torch.rand(rows, 3, generator=_g(seed)) + torch.tensor([0.6, 0.0, -0.2]))
    cu = torch.arange(rows + 1, dtype=torch.int32) * hist
    ids = (torch.rand(rows * hist, generator=_g(seed + 1)) ** 3 * vocab).to(torch.int32)
    ops.count_tokens(r, ids, cu, _ints(seed + 2, 0, hist, rows), reset=True)
    if bias:
        r.bias_ids.copy_(_ints(seed + 3, -1, vocab - 1, rows, bias))
        r.bias_ids[:, -1] = r.bias_ids[:, 0]  # the same token twice
        r.bias.copy_(4 * torch.randn(rows, bias, generator=_g(seed + 4)))
    if mask:
        r.mask.copy_(_ints(seed + 5, -2 ** 31, 2 ** 31 - 1, *r.mask.shape))
        if rows > 1:
            r.mask[1] = 0  # nothing is allowed
    if not pen:
        r.penalties = None
    return r


def _to_gpu(r):
    return ops.LogitRules(*(None if t is None else t.cuda() for t in r._args()), vocab=r.vocab)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 7), (2, 33), (5, 1000), (3, 32003), (1, 152064), (70, 4096)])
@pytest.mark.parametrize("bias,mask,pen", [(0, False, True), (1, True, False), (0, True, True), (17, False, False), (9, True, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rules(rows, vocab, bias, mask, pen, dtype):
    r = _rules(rows + vocab, rows, vocab, bias, mask, pen)
    x = (3 * torch.randn(rows, vocab, generator=_g(9))).to(dtype)
    if vocab > 30:
        x[0, 3], x[0, 20], x[rows - 1, 11] = float("nan"), -math.inf, -0.0
    g, xg = _to_gpu(r), x.cuda()
    want, got = ops.logits_process(x, r), ops.logits_process(xg, g)
    assert torch.equal(want.nan_to_num(123.0), got.cpu().nan_to_num(123.0)) and torch.equal(x.nan_to_num(123.0), xg.cpu().nan_to_num(123.0))
    for a, b in zip(ops.logits_argmax(x, r), ops.logits_argmax(xg, g)):
        assert torch.equal(a, b.cpu())
    # rows of another pitch and alignment, in place
    wide = torch.zeros(rows, vocab + 11, dtype=dtype, device="cuda")
    for at in (0, 3, 8):
        view = wide[:, at:at + vocab]
        view.copy_(xg)
        for a, b in zip(ops.logits_argmax(view, g), ops.logits_argmax(x, r)):
            assert torch.equal(a.cpu(), b)
        assert ops.logits_process(view, g, out=view).data_ptr() == view.data_ptr()
        assert torch.equal(view.cpu().nan_to_num(123.0), want.nan_to_num(123.0))
        wide.zero_()


@pytest.mark.parametrize("offset,n", [(0, 700), (8, 640), (13, 500), (96, 904), (990, 40), (1000, 16)])
def test_rules_on_a_shard(offset, n):
    """Columns that are a slice of the vocabulary, some of them beyond it."""
    rows, vocab = 4, 1000
    r = _rules(3, rows, vocab, 5, True)
    x = torch.randn(rows, n, generator=_g(4)).bfloat16()
    g, xg = _to_gpu(r), x.cuda()
    assert torch.equal(ops.logits_process(x, r, offset), ops.logits_process(xg, g, offset).cpu())
    for a, b in zip(ops.logits_argmax(x, r, offset), ops.logits_argmax(xg, g, offset)):
        assert torch.equal(a, b.cpu())
    r.mask = g.mask = None
    assert torch.equal(ops.logits_process(x, r, offset), ops.logits_process(xg, g, offset).cpu())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rules_where_all_is_seen(dtype):
    """More seen tokens than a block puts off."""
    rows, vocab = 300, 9001
    r = _rules(40, rows, vocab, 2, True, hist=20)
    r.seen.fill_(-1)
    r.counts[:, ::3] = 2
    x = (3 * torch.randn(rows, vocab, generator=_g(41))).to(dtype)
    g, xg = _to_gpu(r), x.cuda()
    want = ops.logits_process(x, r)
    for a, b in zip(ops.logits_argmax(x, r), ops.logits_argmax(xg, g)):
        assert torch.equal(a, b.cpu())
    assert torch.equal(want, ops.logits_process(xg, g).cpu())
    assert torch.equal(want, ops.logits_process(xg, g, out=xg).cpu())


def test_ties_and_empty_rows():
    x = torch.zeros(3, 5000, dtype=torch.bfloat16, device="cuda")
    x[1, 4321] = x[1, 17] = 2.0
    x[2] = -math.inf
    x[0, 5] = -0.0
    idx, val = ops.logits_argmax(x, ops.LogitRules())
    assert idx.tolist() == [0, 17, -1] and val.tolist() == [0.0, 2.0, -math.inf]
    x[2, 4999] = math.inf
    assert ops.logits_argmax(x, ops.LogitRules())[0].tolist() == [0, 17, 4999]
    # -0 and 0 are equal, wherever they stand
    y = torch.full((1, 152064), -1.0, device="cuda")
    y[0, 100], y[0, 90000] = -0.0, 0.0
    assert ops.logits_argmax(y, ops.LogitRules())[0].tolist() == [100]
    # one mask for all rows
    mask = torch.zeros(1, 157, dtype=torch.int32, device="cuda")
    mask[0, 135] = 1 << 1 | 1 << 2
    idx, _ = ops.logits_argmax(x, ops.LogitRules(mask=mask.expand(3, -1), vocab=5000))
    assert idx.tolist() == [4321, 4321, -1]


def test_rules_in_a_graph():
    """A captured step reads tables that change between replays."""
    r = _to_gpu(_rules(5, 3, 2000, 4, True))
    x = torch.randn(3, 2000, device="cuda").bfloat16()
    g = torch.cuda.CUDAGraph()
    ops.logits_argmax(x, r)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        idx, val = ops.logits_argmax(x, r)
        ops.count_tokens(r, idx)
    c = ops.LogitRules(*(t.cpu() for t in r._args()), vocab=2000)
    for _ in range(6):
        g.replay()
        a, b = ops.logits_argmax(x.cpu(), c)
        ops.count_tokens(c, a)
        assert torch.equal(a, idx.cpu()) and torch.equal(b, val.cpu()) and torch.equal(c.counts, r.counts.cpu())


def test_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    ok = dict(new_lens=i(2), past_lens=i(2), block_tables=i(2, 3), free_list=i(4), free_range=i(3), tokens=2, block_size=16)
    ops.paged_layout(**ok)
    for bad in (dict(new_lens=i(2).long()), dict(past_lens=i(3)), dict(block_tables=i(3, 3)), dict(block_tables=i(2, 0)), dict(free_list=i(0)),
                dict(free_range=i(2)), dict(tokens=-1), dict(rows_per_request=-1), dict(block_size=0), dict(block_size=2 ** 30), dict(free_list=i(4).cpu()),
                dict(new_lens=i(0), past_lens=i(0), block_tables=i(0, 3)), dict(new_lens=i(8193), past_lens=i(8193), block_tables=i(8193, 1)),
                dict(into=ops.PagedLayout(i(2), i(2), i(2), i(2), i(3)))):
        with pytest.raises((RuntimeError, TypeError)):
            ops.paged_layout(**{**ok, **bad})
    r = ops.LogitRules.empty(2, 100)
    x = torch.zeros(2, 100, device="cuda")
    for bad in (x.half(), x[0], x.t(), x[:1], x.cpu().cuda().int()):
        with pytest.raises(RuntimeError):
            ops.logits_argmax(bad, r)
    for f in (dict(penalties=i(2, 3)), dict(counts=i(2, 99)), dict(seen=i(2, 3)), dict(mask=i(2, 3)), dict(mask=i(3, 4)),
              dict(bias_ids=i(1, 1), bias=torch.zeros(1, 1, device="cuda")), dict(bias_ids=i(2, 1), bias=torch.zeros(2, 2, device="cuda"))):
        bad = ops.LogitRules(**{**dict(penalties=r.penalties, counts=r.counts, seen=r.seen), **f}, vocab=100)
        with pytest.raises(RuntimeError):
            ops.logits_process(x, bad)
    with pytest.raises(RuntimeError):
        ops.logits_process(x, r, out=x.bfloat16())
    with pytest.raises(RuntimeError):
        ops.logits_process(x, r, offset=-1)
    with pytest.raises(RuntimeError):
        ops.count_tokens(r, i(3))
    with pytest.raises(RuntimeError):
        ops.count_tokens(r, i(5), i(2))
    with pytest.raises(ValueError):
        ops.count_tokens(ops.LogitRules(), i(2))
    with pytest.raises(ValueError):
        ops.LogitRules(penalties=r.penalties)
