# SPDX-License-Identifier: MIT
"""Further tokens on top of the cache, and the log probabilities of a text, on the CPU path and over two gloo ranks."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine, Qwen2Config, Qwen2Model
from barlink_sm86_b200.parallel import TPComm

# Both sides of a comparison are sums in fp32 in different orders: a layer's longest is of 256 terms, and values grow by no more than
# their own size a layer.  2 layers x 3 sums x 256 x 2^-24 is 1e-4 of logits that stay below 4.
TOL = 4e-4


def _model(comm=None, vocab=500):
    cfg = Qwen2Config(hidden=128, layers=2, n_heads=4, n_kv_heads=2, head_dim=64, intermediate=256, vocab=vocab, name="test")
    return Qwen2Model(cfg, comm, seed=5)


def _text(seed, n, vocab=500):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def _whole(m, text):
    """Log probabilities [n, vocab] behind every token of a text, in 64 bits from one dense pass."""
    h = m.prefill(text[None])
    return torch.log_softmax(m.logits_local(h).double()[:, :m.cfg.vocab], -1)


@pytest.mark.parametrize("kv_bits", [16, 4])
@pytest.mark.parametrize("max_tokens", [1, 7, 8192])
def test_pieces_of_a_text(kv_bits, max_tokens):
    m = _model()
    lens = [19, 0, 33, 1]
    texts = [_text(i, n) for i, n in enumerate(lens)]
    eng = DecodeEngine(m, 4, 64, kv_bits=kv_bits)
    eng.ids.fill_(9)
    nxt, lp = eng.score(torch.cat(texts), lens, 3, max_tokens)
    assert nxt[1] == 9 and lp.logprobs.shape == (53,) and lp.top_ids.shape == (53, 3)
    at = 0
    for b, t in enumerate(texts):
        if not len(t):
            continue
        want = _whole(m, t)
        rows = slice(at, at + len(t))
        at += len(t)
        follows = torch.cat([t[1:], nxt[b:b + 1]]).long()
        got = lp.logprobs[rows].double()
        if kv_bits == 16:
            assert int(nxt[b]) == int(want[-1].argmax())
            assert (got - want.gather(1, follows[:, None])[:, 0]).abs().max() < TOL
            assert (lp.top_logprobs[rows].double() - want.topk(3).values).abs().max() < TOL
            assert (lp.entropy[rows].double() + (want.exp() * want).sum(1)).abs().max() < TOL * 8
        else:
            # held to within half of a 4-bit step, 0.08 of the values' deviation: log probabilities stay near
            assert (got - want.gather(1, follows[:, None])[:, 0]).abs().mean() < 0.1
    assert torch.equal(lp.top_ids[:, 0][[18, 51, 52]], nxt[[0, 2, 3]])
    assert (eng.ctx_lens if kv_bits == 4 else eng.positions).tolist() == lens


def test_turns_of_a_conversation_equal_the_whole_text():
    """Prompt, tokens of the model's own, a further turn, tokens again: with the last token chosen at the head of a turn, the text is one."""
    m = _model()
    eng = DecodeEngine(m, 2, 96, logprobs=2)
    out = eng.prefill(torch.stack([_text(1, 12), _text(2, 12)]))
    text = [[_text(1, 12)], [_text(2, 12)]]
    said, chose = [], []
    for turn in range(3):
        eng.ids.copy_(out)
        for b in range(2):
            text[b].append(out[b:b + 1].clone())
        for _ in range(4):
            at = sum(len(t) for t in text[0])
            out = eng.step().clone()
            said.append(eng.logprobs)
            chose.append((at, out))
            for b in range(2):
                text[b].append(out[b:b + 1].clone())
        # request 0 alone gets a turn of 5, request 1 of 9; both begin with the token that no step has consumed
        more = [_text(10 + turn, 5), _text(20 + turn, 9)]
        new = [torch.cat([out[b:b + 1], more[b]]) for b in range(2)]
        for b in range(2):
            text[b].append(more[b])
        out = eng.extend(torch.cat(new), [6, 10], max_tokens=7)
        text = [[torch.cat(t)] for t in text]
        for b in range(2):
            assert int(out[b]) == int(_whole(m, text[b][0])[-1].argmax())
    want = _whole(m, text[0][0])
    for (at, ids), lp in zip(chose, said):
        assert abs(float(lp.logprobs[0]) - float(want[at - 1, int(ids[0])])) < TOL
        assert torch.equal(lp.top_ids[:, 0], ids) and torch.equal(lp.top_logprobs[:, 0], lp.logprobs)


def test_blocks_of_the_4_bit_cache():
    m = _model()
    eng = DecodeEngine(m, 3, 64, kv_bits=4, n_blocks=7)
    eng.ids.copy_(eng.start(torch.cat([_text(1, 17), _text(2, 5)]), [17, 5, 0]))
    eng.step()
    # request 2 rests and starts with its turn; request 0 crosses into a third block
    out = eng.extend(torch.cat([_text(3, 20), _text(4, 3)]), [20, 0, 3])
    assert eng.ctx_lens.tolist() == [38, 6, 3] and eng.running == [True] * 3 and out[1] == eng.ids[1]
    assert eng.blocks_missing() == 0 and eng.tokens_lost() == 0
    held = [int(x) for b, n in enumerate([3, 1, 1]) for x in eng.cache.block_tables[b, :n]]
    head, free = int(eng.cache.free_range[0]), int(eng.cache.free_range[1])
    assert sorted(held + [int(eng.cache.free_list[(head + i) % 7]) for i in range(free)]) == list(range(7))
    eng.ids.copy_(out)
    eng.step()
    assert eng.ctx_lens.tolist() == [39, 7, 4]
    # where blocks run out, the tokens count as lost and the others go on
    eng.extend(_text(5, 50), [0, 50, 0])
    assert eng.blocks_missing() == 1 and eng.tokens_lost() == 57 - 48
    eng.finish([0, 1, 2])
    assert int(eng.cache.free_range[1]) == 7


def test_a_failing_pass_gives_its_blocks_back(monkeypatch):
    m = _model()
    eng = DecodeEngine(m, 2, 64, kv_bits=4)
    eng.start(_text(1, 20), [20, 0])

    def fail(*a, **k):
        raise MemoryError("no room")

    monkeypatch.setattr(m, "extend_packed", fail)
    with pytest.raises(MemoryError):
        eng.extend(_text(2, 9), [0, 9])
    assert eng.ctx_lens.tolist() == [20, 0] and eng.running == [True, False] and int(eng.cache.free_range[1]) == 6


def test_rules_count_the_tokens_given():
    m = _model()

    def engine(kv_bits):
        r = ops.LogitRules.empty(2, 500, "cpu")
        r.penalties.copy_(torch.tensor([1.5, 0.5, 0.25]).expand(2, 3))
        return DecodeEngine(m, 2, 64, kv_bits=kv_bits, rules=r)

    a, b = engine(4), engine(4)
    prompts = torch.cat([_text(1, 9), _text(2, 14)])
    a.start(prompts, [9, 14])
    b.extend(prompts, [9, 14])
    assert torch.equal(a.rules.seen, b.rules.seen) and int(b.rules.counts.sum()) == 2
    b.extend(_text(3, 6), [6, 0])
    assert int(b.rules.counts.sum()) == 3
    for t in _text(3, 6).tolist():
        assert int(b.rules.seen[0, t // 32]) >> (t % 32) & 1
    # a request that rested starts with empty tables
    b.finish([0])
    b.extend(_text(4, 2), [2, 0])
    assert int(b.rules.counts[0].sum()) == 1
    assert sum(bin(int(w) & 0xffffffff).count("1") for w in b.rules.seen[0]) <= 3
    c = engine(16)
    c.extend(prompts, [9, 14])
    assert int(c.rules.counts.sum()) == 2


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_refusals(kv_bits):
    m = _model()
    eng = DecodeEngine(m, 2, 32, kv_bits=kv_bits)
    with pytest.raises(ValueError):
        eng.extend(_text(1, 5), [5])
    with pytest.raises(ValueError):
        eng.extend(_text(1, 5), [5, 1])
    with pytest.raises(ValueError):
        eng.extend(_text(1, 5), [6, -1])
    with pytest.raises(ValueError):
        eng.extend(_text(1, 5), [5, 0], max_tokens=0)
    with pytest.raises(ValueError):
        eng.score(_text(1, 5), [5, 0], top=33)
    with pytest.raises(ValueError):
        DecodeEngine(m, 2, 32, kv_bits=kv_bits, logprobs=33)
    most = 32 if kv_bits == 4 else 31
    eng.extend(_text(1, most - 4), [most - 4, 0])
    before = eng.ctx_lens.clone()
    with pytest.raises(ValueError):
        eng.extend(_text(1, 5), [5, 0])
    assert torch.equal(eng.ctx_lens, before)
    eng.extend(_text(1, 4), [4, 0])
    # a full request is in no one's way
    eng.extend(_text(1, 2), [0, 2])
    nxt, lp = eng.score(_text(1, 0), [0, 0], 2)
    assert torch.equal(nxt, eng.ids) and lp.logprobs.shape == (0,) and lp.top_ids.shape == (0, 2)


def test_ids_of_any_shape():
    m = _model()
    a, b = DecodeEngine(m, 2, 32), DecodeEngine(m, 2, 32)
    ids = torch.stack([_text(1, 9), _text(2, 9)])
    out = a.extend(ids.long(), [9, 9], max_tokens=5)
    assert torch.equal(out, b.extend(ids.reshape(-1), [9, 9], max_tokens=5)) and torch.equal(out, DecodeEngine(m, 2, 32).prefill(ids))


def _run(comm):
    # (an odd vocabulary: the second rank's slice ends in padding)
    m = _model(comm, 501)
    eng = DecodeEngine(m, 3, 64, logprobs=4)
    nxt, lp = eng.score(_text(1, 30, 501), [20, 0, 10], 5, max_tokens=13)
    eng.ids.copy_(nxt)
    out = eng.step().clone()
    return nxt, out, tuple(lp), tuple(eng.logprobs)


def _rank(rank, path):
    dist.init_process_group("gloo", init_method="file://" + os.path.join(path, "meet"), rank=rank, world_size=2)
    torch.save(_run(TPComm(dist.group.WORLD)), os.path.join(path, "out%d.pt" % rank))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_score_as_one(tmp_path):
    nxt, out, *lps = _run(TPComm.single())
    mp.spawn(_rank, args=(str(tmp_path),), nprocs=2)
    for rank in range(2):
        n, o, *got = torch.load(tmp_path / ("out%d.pt" % rank))
        assert torch.equal(n, nxt) and torch.equal(o, out)
        for a, b in zip(got, lps):
            for x, y in zip(a, b):
                assert x.shape == y.shape and (x.double() - y.double()).abs().max() < TOL * 8
