# SPDX-License-Identifier: MIT
"""Serving on the 4-bit cache where a run leaves the ordinary, on the CPU path: blocks run out, requests outgrow their tables."""
import ctypes

import pytest
import torch

import barlink_sm86_b200 as bl
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


def test_plain_c_entries_refuse_what_they_cannot_read():
    """No pointer, or one that a 16-byte access would not take, gets as far as a launch; sizes that no workspace has are 0 bytes."""
    p, i, f, d, s, e = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_double, ctypes.c_size_t, ctypes.create_string_buffer(512)
    lib = ctypes.CDLL(bl.load_extension().__file__)

    def refused(name, types, *args):
        fn = getattr(lib, name)
        fn.argtypes = [*types, p, ctypes.c_char_p, s]
        e.value = b""
        return fn(*args, None, e, 512) == -1 and e.value.startswith(b"barlink: ")

    read = ("bl_kv4_read", [p] * 4 + [i] * 5)
    for ptrs in ((None, 16, 16, 16), (16, None, 16, 16), (16, 16, None, 16), (16, 16, 16, None), (24, 16, 16, 16), (16, 16, 8, 16), (16, 16, 16, 4)):
        assert refused(*read, *ptrs, 1, 1, 128, 16, 1)
    lib.bl_paged_attn_decode_q4_ws.restype = s
    for sizes in ((1, 4, 0, 128), (1, 0, 1, 128), (0, 4, 1, 128), (-1, 4, 1, 128)):
        assert lib.bl_paged_attn_decode_q4_ws(*sizes) == 0
    attn = ("bl_paged_attn_decode_q4", [p, i] + [p] * 4 + [i] * 7 + [f, p, s])
    sizes = (1, 4, 1, 128, 16, 1, 1)
    for q, *ptrs in ((None, 16, 16, 16, 16), (16, None, 16, 16, 16), (16, 16, None, 16, 16), (16, 16, 16, None, 16), (16, 16, 16, 16, None)):
        assert refused(*attn, q, 512, *ptrs, *sizes, 0.1, 16, 1 << 30)
    assert refused(*attn, 16, 512, 16, 16, 16, 16, -1, *sizes[1:], 0.1, 16, 1 << 30)
    layout = ("bl_paged_layout", [p] * 10 + [i] * 6)
    for k in range(10):
        assert refused(*layout, *(None if j == k else 16 for j in range(10)), 1, 1, 1, 1, 16, 0)
    count = ("bl_count_tokens", [p] * 5 + [i] * 4)
    for ptrs in ((None, 16, None, 16, 16), (16, 16, None, None, 16), (16, 16, None, 16, None)):
        assert refused(*count, *ptrs, 1, 1, 10, 1)
    assert refused(*count, 16, 16, None, 16, 16, 1, -1, 10, 0) and refused(*count, 16, None, None, 16, 16, 2, 1, 10, 0)
    write = ("bl_rope_kv_write_q4", [p, p, i, s] + [p] * 5 + [i] * 6 + [d])
    for ptrs in ((None, 16, 16, 16, 16), (16, None, 16, 16, 16), (16, 16, None, 16, 16), (16, 16, 16, 16, None), (8, 16, 16, 16, 16), (16, 16, 16, 16, 8)):
        qkv, out, pos, slots, cache = ptrs
        assert refused(*write, qkv, None, 0, 0, None, out, pos, slots, cache, 1, 1, 1, 128, 16, 1, 1e4)


def test_a_start_that_fails_leaves_the_engine_as_it_was(monkeypatch):
    """An error of the model in the middle of the passes: no request holds blocks, and the same call can be made again."""
    m = _model()
    want = DecodeEngine(m, 3, 64, kv_bits=4)
    want.ids.copy_(want.start(_ids(50), [30, 0, 20]))
    eng = DecodeEngine(m, 3, 64, kv_bits=4)
    run, calls = m.prefill_packed, []

    def fails(*a):
        calls.append(a)
        if len(calls) == 2:
            raise MemoryError("no memory")
        return run(*a)

    monkeypatch.setattr(m, "prefill_packed", fails)
    eng.ids.copy_(eng.start(_ids(9), [0, 9, 0]))
    eng.step()
    with pytest.raises(MemoryError):
        eng.start(_ids(50), [30, 0, 20], max_tokens=30)
    assert eng.ctx_lens.tolist() == [0, 10, 0] and eng.running == [False, True, False] and eng.new_lens.tolist() == [0, 1, 0]
    assert int(eng.cache.free_range[1]) == 11
    out = eng.start(_ids(50), [30, 0, 20], max_tokens=30)
    assert out.tolist()[::2] == want.ids.tolist()[::2]
    eng.ids.copy_(out)
    assert eng.step().tolist()[::2] == want.step().tolist()[::2]
