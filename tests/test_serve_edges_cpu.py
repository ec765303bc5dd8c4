# SPDX-License-Identifier: MIT
"""Serving on the 4-bit cache where a run leaves the ordinary, on the CPU path: blocks run out, requests outgrow their tables."""
import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine, Qwen2Config, Qwen2Model


def _model():
    cfg = Qwen2Config(hidden=128, layers=1, n_heads=4, n_kv_heads=2, head_dim=64, intermediate=256, vocab=500, name="test")
    return Qwen2Model(cfg, seed=5)


def _ids(n):
    return torch.arange(n, dtype=torch.int32)


def test_tokens_without_a_block_stay_counted():
    """The page that got no block is missed once, its tokens with every step; steps, starts and ends behind it forget nothing."""
    eng = DecodeEngine(_model(), 2, 64, kv_bits=4, n_blocks=3)
    eng.start(_ids(50), [30, 20])
    assert eng.blocks_missing() == 1 and eng.tokens_lost() == 4   # tokens 16 .. 19 of request 1
    for i in range(2):
        eng.step()                                                # request 0 fills its second page
        assert eng.tokens_lost() == 5 + i
    eng.finish([0])
    assert eng.blocks_missing() == 0 and eng.tokens_lost() == 6
    for i in range(10):
        eng.step()
        assert eng.blocks_missing() == 0 and eng.tokens_lost() == 7 + i
    eng.step()                                                    # a page of its own: there is a block now
    assert eng.ctx_lens.tolist() == [0, 33] and eng.tokens_lost() == 16 and int(eng.slots[1]) >= 0


def test_tokens_beyond_the_table_are_counted():
    eng = DecodeEngine(_model(), 1, 32, kv_bits=4)
    eng.start(_ids(31), [31])
    eng.step()
    assert eng.tokens_lost() == 0
    for i in range(3):
        eng.step()
        assert eng.tokens_lost() == i + 1 and eng.blocks_missing() == 0


def test_lost_refusals():
    i = torch.zeros(2, dtype=torch.int32)
    call = dict(new_lens=i, past_lens=i, block_tables=i.view(2, 1), free_list=i, free_range=torch.zeros(3, dtype=torch.int32), tokens=2)
    for bad in (i, i[:1].long()):
        with pytest.raises(ValueError):
            ops.paged_layout(**call, lost=bad)


@pytest.mark.parametrize("kv_bits", [4, 16])
@pytest.mark.parametrize("table", ["counts", "seen"])
def test_rules_with_one_of_the_two_tables(kv_bits, table):
    """Without penalties nothing reads them: a run does without either."""
    rules = ops.LogitRules(**{table: torch.zeros(2, 500 if table == "counts" else 16, dtype=torch.int32)}, vocab=500)
    eng = DecodeEngine(_model(), 2, 64, kv_bits=kv_bits, rules=rules)
    eng.ids.copy_(eng.prefill(_ids(20).view(2, 10)))
    assert eng.step().shape == (2,)


def test_a_context_longer_than_the_table():
    eng = DecodeEngine(_model(), 2, 64, kv_bits=4)
    eng.set_context(64)
    assert eng.ctx_lens.tolist() == [64, 64]
    for length in (65, -1):
        with pytest.raises(ValueError):
            eng.set_context(length)
    assert eng.ctx_lens.tolist() == [64, 64]
