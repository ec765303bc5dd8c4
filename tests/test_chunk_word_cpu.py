# SPDX-License-Identifier: MIT
"""The error word of attention of new tokens: what is refused on the host, and that the CPU path, which waits for nothing, leaves it alone."""
import ctypes

import pytest
import torch

from barlink_sm86_b200 import ops
from test_chunk_cpu import _state
from test_chunk_entries_cpu import PTR, _entry


def _say(**change):
    call = dict(q=PTR, q_stride=4608, k=PTR, v=PTR, cache4=None, tables=PTR, cu=PTR, lens=PTR, out=PTR, tokens=8, batch=2, nq=28, nkv=4, hd=128, block=16,
                blocks=10, width=5, scale=0.1, ws=PTR, bytes=0, error=None, stream=None)
    call.update(change)
    fn, err = _entry("bl_paged_attn_chunk_say"), ctypes.create_string_buffer(512)
    p, i = ctypes.c_void_p, ctypes.c_int
    fn.argtypes = [p, i, p, p, p, p, p, p, p] + [i] * 8 + [ctypes.c_float, p, ctypes.c_size_t, p, p, ctypes.c_char_p, ctypes.c_size_t]
    return fn(*call.values(), err, 512), err.value.decode()


@pytest.mark.parametrize("change,why", [(dict(error=PTR + 2), "error word"), (dict(error=PTR + 1), "error word"), (dict(error=PTR), "workspace"),
                                        (dict(), "workspace"), (dict(hd=96, error=PTR), "head_dim"), (dict(q=None), "needs queries")])
def test_plain_c_entry(change, why):
    rc, err = _say(**change)
    assert rc == -1 and why in err, err


def test_nothing_to_do():
    assert _say(tokens=0, q=None, ws=None, error=PTR)[0] == 0


def test_cpu_path():
    q, k, v, table, cu, lens = _state()
    word = torch.tensor([7], dtype=torch.int32)
    want = ops.paged_attn_chunk(q, k, v, table, cu, lens, 6, 2, 64, 0.125)
    assert torch.equal(ops.paged_attn_chunk(q, k, v, table, cu, lens, 6, 2, 64, 0.125, error=word), want) and int(word) == 7
    for bad in (word.float(), word.long(), word.repeat(2), word[:0]):
        with pytest.raises(ValueError):
            ops.paged_attn_chunk(q, k, v, table, cu, lens, 6, 2, 64, 0.125, error=bad)
