# SPDX-License-Identifier: MIT
"""The plain-C entries of attention of new tokens and of log probabilities: what they refuse, they refuse on the host."""
import ctypes

import pytest

import barlink_sm86_b200 as bl

PTR = 4096  # (aligned, and never looked at)


def _entry(name):
    return getattr(ctypes.CDLL(bl.load_extension().__file__), name)


def _chunk(**change):
    call = dict(q=PTR, q_stride=4608, k=PTR, v=PTR, cache4=None, tables=PTR, cu=PTR, lens=PTR, out=PTR, tokens=8, batch=2, nq=28, nkv=4, hd=128, block=16,
                blocks=10, width=5, scale=0.1, ws=PTR, bytes=0, stream=None)
    call.update(change)
    fn, err = _entry("bl_paged_attn_chunk"), ctypes.create_string_buffer(512)
    p, i = ctypes.c_void_p, ctypes.c_int
    fn.argtypes = [p, i, p, p, p, p, p, p, p] + [i] * 8 + [ctypes.c_float, p, ctypes.c_size_t, p, ctypes.c_char_p, ctypes.c_size_t]
    return fn(*call.values(), err, 512), err.value.decode()


@pytest.mark.parametrize("change,why", [
    (dict(hd=96), "head_dim"), (dict(hd=0), "head_dim"), (dict(nq=27), "nq % nkv"), (dict(nkv=0), "nq % nkv"), (dict(nq=-28, nkv=-4), "nq % nkv"),
    (dict(nq=516), "128 query heads"), (dict(block=8), "multiple of 16"), (dict(block=24), "multiple of 16"), (dict(block=0), "multiple of 16"),
    (dict(block=-16), "multiple of 16"), (dict(tokens=-1), "below 0"), (dict(batch=-1), "below 0"), (dict(width=-1), "below 0"), (dict(blocks=0), "a block"),
    (dict(blocks=2 ** 27), "32 bits"), (dict(width=2 ** 27), "2^30"), (dict(tokens=2 ** 30, width=2 ** 20), "31 bits"), (dict(q_stride=4604), "16-byte"),
    (dict(q_stride=3576), "16-byte"), (dict(q_stride=-8), "16-byte"), (dict(q=None), "needs queries"), (dict(v=None), "one kind of cache"),
    (dict(cache4=PTR), "one kind of cache"), (dict(k=None, v=None), "one kind of cache"), (dict(tables=None), "block tables"), (dict(cu=None), "row offsets"),
    (dict(lens=None), "context lengths"), (dict(out=None), "an output"), (dict(q=PTR + 8), "16-byte"), (dict(k=PTR + 2), "16-byte"), (dict(out=PTR + 4), "16-byte"),
    (dict(ws=PTR + 4), "16-byte"), (dict(k=None, v=None, cache4=PTR + 1), "16-byte"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(ws=None), "workspace")])
def test_attention_of_new_tokens(change, why):
    rc, err = _chunk(**change)
    assert rc == -1 and why in err, err


@pytest.mark.parametrize("change", [dict(tokens=0), dict(batch=0)])
def test_nothing_to_do(change):
    assert _chunk(q=None, k=None, v=None, out=None, ws=None, **change)[0] == 0


def test_workspace_of_what_is_refused():
    fn = _entry("bl_paged_attn_chunk_ws")
    fn.restype = ctypes.c_size_t
    for call in [(0, 28, 4, 128), (5, 28, 0, 128), (5, 2, 4, 128), (5, 28, 4, 96), (5, 129, 1, 64)]:
        assert fn(*call) == 0


class Score(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("ld", ctypes.c_size_t), ("rows", ctypes.c_int), ("n", ctypes.c_int), ("fp32", ctypes.c_int), ("vocab", ctypes.c_int),
                ("offset", ctypes.c_int), ("ids", ctypes.c_void_p), ("n_ids", ctypes.c_int), ("top", ctypes.c_int), ("raw", ctypes.c_int), ("given", ctypes.c_void_p),
                ("entropy", ctypes.c_void_p), ("top_ids", ctypes.c_void_p), ("top_val", ctypes.c_void_p), ("parts", ctypes.c_void_p)]


def _score(**change):
    call = dict(logits=PTR, ld=100, rows=3, n=100, fp32=1, vocab=100, offset=0, ids=PTR, n_ids=1, top=2, raw=0, given=PTR, entropy=PTR, top_ids=PTR, top_val=PTR)
    call.update(change)
    fn, err = _entry("bl_token_logprobs"), ctypes.create_string_buffer(512)
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t]
    return fn(ctypes.byref(Score(**call)), None, err, 512), err.value.decode()


@pytest.mark.parametrize("change,why", [
    (dict(rows=-1), "32 bits"), (dict(n=-1), "32 bits"), (dict(vocab=-1), "32 bits"), (dict(offset=-1), "32 bits"), (dict(offset=2 ** 31 - 50), "32 bits"),
    (dict(n=2 ** 31 - 1), "32 bits"), (dict(top=33), "32 alternatives"), (dict(top=-1), "32 alternatives"), (dict(n_ids=-1), "too many rows"),
    (dict(rows=2 ** 29), "too many rows"), (dict(logits=None), "needs logits"), (dict(ids=None), "needs logits"), (dict(given=None), "needs logits"),
    (dict(entropy=None), "needs logits"), (dict(top_ids=None), "needs logits"), (dict(top_val=None), "needs logits"), (dict(raw=1), "needs logits"),
    (dict(logits=PTR + 2), "boundaries"), (dict(logits=PTR + 1, fp32=0), "boundaries")])
def test_log_probabilities(change, why):
    rc, err = _score(**change)
    assert rc == -1 and why in err, err
    assert _score(rows=0, logits=None)[0] == 0
