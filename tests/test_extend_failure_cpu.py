# SPDX-License-Identifier: MIT
"""An `extend` or `score` that raises, wherever it does, leaves the rules' tables as they were (CPU path)."""
import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine
from test_extend_cpu import _model, _text


def _fail(*a, **k):
    raise MemoryError("no room")


def _second(run):
    """A model's passes, of which the second fails."""
    passes = []

    def wrapped(*a, **k):
        passes.append(0)
        return _fail() if len(passes) == 2 else run(*a, **k)

    return wrapped


# what raises, and how it is reached
PLACES = {
    "first pass": lambda m, eng: (m, "extend_packed", _fail),
    "second pass": lambda m, eng: (m, "extend_packed", _second(m.extend_packed)),
    "choice": lambda m, eng: (m, "next_tokens", _fail),
    "scores": lambda m, eng: (m, "token_logprobs", _fail),
    "attention that gave up": lambda m, eng: (eng, "_check_chunk", _fail),
}


def _engine(m, kv_bits):
    r = ops.LogitRules.empty(3, 500, "cpu")
    r.penalties.copy_(torch.tensor([1.5, 0.5, 0.25]).expand(3, 3))
    eng = DecodeEngine(m, 3, 96, kv_bits=kv_bits, rules=r)
    # (on the 4-bit cache the third request rests, with what an earlier one left in its row)
    lens = [9, 14, 5]
    eng.ids.copy_(eng.extend(torch.cat([_text(i, n) for i, n in enumerate(lens)]), lens))
    if kv_bits == 4:
        eng.finish([2])
    return eng


@pytest.mark.parametrize("kv_bits", [16, 4])
@pytest.mark.parametrize("place", PLACES)
def test_tables_are_as_before(monkeypatch, place, kv_bits):
    m = _model()
    eng = _engine(m, kv_bits)
    before = [t.clone() for t in (eng.rules.counts, eng.rules.seen)]
    with monkeypatch.context() as mp:
        mp.setattr(*PLACES[place](m, eng))
        for _ in range(2):
            with pytest.raises(MemoryError):
                eng.score(_text(7, 26), [0, 6, 20], 2, max_tokens=8)
            if kv_bits == 4 or place == "second pass":
                break
    for t, was in zip((eng.rules.counts, eng.rules.seen), before):
        assert torch.equal(t, was)
    if kv_bits == 4:
        assert eng.running == [True, False, False]


@pytest.mark.parametrize("place", PLACES)
def test_later_steps_are_those_of_an_engine_without_the_failure(monkeypatch, place):
    m = _model()
    a, b = _engine(m, 16), _engine(m, 16)
    with monkeypatch.context() as mp:
        mp.setattr(*PLACES[place](m, a))
        with pytest.raises(MemoryError):
            a.score(_text(7, 26), [0, 6, 20], 2, max_tokens=8)
    for eng in (a, b):
        eng.ids.copy_(eng.extend(_text(8, 7), [4, 3, 0]))
    for _ in range(8):
        assert torch.equal(a.step(), b.step())
    assert torch.equal(a.rules.counts, b.rules.counts) and torch.equal(a.rules.seen, b.rules.seen)
