# SPDX-License-Identifier: MIT
"""Whose wait ran out: a call, an engine, and nobody else."""
import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine
from test_chunk_gpu import Case
from test_extend_gpu import _ids, _word, model, polls  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def _run(c, error=None):
    tail = (c.table, c.cu, c.lens, c.nq, c.nkv, c.hd, c.scale)
    return ops.paged_attn_chunk_q4(c.qkv, c.cache, *tail, error=error) if c.q4 else ops.paged_attn_chunk(c.qkv, c.k, c.v, *tail, error=error)


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_an_engine_does_not_report_what_others_met(ext, model, polls, kv_bits):  # noqa: F811
    eng = DecodeEngine(model, 2, 128, kv_bits=kv_bits)
    polls(0)
    assert bool(_run(Case((14, 2, 128), 16, [(30, 100)])).isnan().all())
    polls(1 << 24)
    eng.extend(_ids(1, 40), [30, 10])
    assert _word(ext) == 1  # (still to be read by whoever made that call)
    if kv_bits == 4:
        assert eng.running == [True, True]


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_another_engine_does_not_take_the_report(ext, model, polls, kv_bits):  # noqa: F811
    a, b = DecodeEngine(model, 2, 128, kv_bits=kv_bits), DecodeEngine(model, 2, 128, kv_bits=kv_bits)
    polls(1 << 24)
    check, taken = a._check_chunk, []

    def meanwhile():
        """Another engine's whole call between a's passes and a's look."""
        polls(1 << 24)
        try:
            b.extend(_ids(3, 20), [10, 10])
        except RuntimeError:
            taken.append(b)
        check()

    a._check_chunk = meanwhile
    polls(0)
    with pytest.raises(RuntimeError, match="gave up"):
        a.extend(_ids(1, 40), [30, 10])
    assert not taken
    a._check_chunk = check
    a.extend(_ids(1, 40), [30, 10])  # (once reported)
    assert _word(ext) == 0


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_a_call_that_fails_otherwise_leaves_no_report(ext, model, polls, kv_bits):  # noqa: F811
    eng = DecodeEngine(model, 2, 128, kv_bits=kv_bits)
    next_tokens = model.next_tokens

    def fail(*a, **k):
        raise MemoryError("no room")

    try:
        model.next_tokens = fail
        polls(0)
        with pytest.raises(MemoryError):
            eng.extend(_ids(1, 40), [30, 10])
    finally:
        del model.next_tokens
    assert model.next_tokens == next_tokens
    polls(1 << 24)
    eng.extend(_ids(1, 40), [30, 10])


@pytest.mark.parametrize("q4", [False, True])
def test_a_word_of_the_call(ext, polls, q4):  # noqa: F811
    c = Case((14, 2, 128), 16, [(30, 100), (3, 2000)], q4)
    polls(1 << 24)
    mine, other = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    want = _run(c, mine)
    assert int(mine) == 0
    polls(0)
    assert bool(_run(c, mine).isnan().all())
    polls(1 << 24)
    assert torch.equal(_run(c, other), want)
    assert int(mine) == 1 and int(other) == 0 and _word(ext) == 0
    assert torch.equal(_run(c, mine), want) and int(mine) == 1  # (not set back)
    # in a graph: the word is the one that was captured
    mine.zero_()
    g = torch.cuda.CUDAGraph()
    polls(0)
    with torch.cuda.graph(g):
        out = _run(c, mine)
    polls(1 << 24)
    g.replay()
    torch.cuda.synchronize()
    assert bool(out.isnan().all()) and int(mine) == 1 and _word(ext) == 0


def test_refusals(ext):
    c = Case((14, 2, 128), 16, [(3, 10)])
    for bad in (torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises((RuntimeError, ValueError)):
            _run(c, bad)
