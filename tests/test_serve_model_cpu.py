# SPDX-License-Identifier: MIT
"""The decode engine on a 4-bit cache and under rules, on the CPU path: requests of different lengths that come and go."""
import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine, Qwen2Config, Qwen2Model


def _model():
    cfg = Qwen2Config(hidden=128, layers=2, n_heads=4, n_kv_heads=2, head_dim=64, intermediate=256, vocab=500, name="test")
    return Qwen2Model(cfg, seed=5)


def _prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 500, (n,), generator=g, dtype=torch.int32) for n in lens]


def _alone(m, prompt, steps, rules=None):
    eng = DecodeEngine(m, 1, 100, kv_bits=4, rules=rules)
    toks = [eng.start(prompt, [len(prompt)])]
    eng.ids.copy_(toks[0])
    for _ in range(steps):
        toks.append(eng.step().clone())
    return torch.cat(toks).tolist()


def test_requests_do_not_know_of_each_other():
    m = _model()
    p = _prompts([5, 17, 33, 16])
    want = [_alone(m, q, 12) for q in p]
    eng = DecodeEngine(m, 4, 100, kv_bits=4, n_blocks=20)
    got = [[] for _ in p]
    # requests 0 and 2 begin, 1 and 3 join later, 0 ends and its place is taken by request 1's prompt again
    out = eng.start(torch.cat([p[0], p[2]]), [5, 0, 33, 0])
    got[0].append(int(out[0]))
    got[2].append(int(out[2]))
    eng.ids.copy_(out)
    for i in range(4):
        out = eng.step()
        for b in (0, 2):
            got[b].append(int(out[b]))
    out = eng.start(torch.cat([p[1], p[3]]), [0, 17, 0, 16], max_tokens=20)
    got[1].append(int(out[1]))
    got[3].append(int(out[3]))
    assert int(out[0]) == got[0][-1] and int(out[2]) == got[2][-1]
    eng.ids.copy_(out)
    for i in range(8):
        out = eng.step()
        for b in range(4):
            got[b].append(int(out[b]))
    assert got[0] == want[0] and got[2] == want[2] and got[1] == want[1][:9] and got[3] == want[3][:9]
    eng.finish([0])
    assert eng.ctx_lens.tolist() == [0, 25, 45, 24] and eng.blocks_missing() == 0
    out = eng.start(p[1], [17, 0, 0, 0])
    again = [int(out[0])]
    eng.ids.copy_(out)
    for i in range(5):
        out = eng.step()
        again.append(int(out[0]))
        got[1].append(int(out[1]))
    assert again == want[1][:6] and got[1] == want[1][:13] + got[1][13:]
    # every block has one holder
    c = eng.cache
    held = [x for b in range(4) for x in c.block_tables[b, : -(-int(eng.ctx_lens[b]) // 16)].tolist()]
    head, free = int(c.free_range[0]), int(c.free_range[1])
    assert sorted(held + [int(c.free_list[(head + i) % 20]) for i in range(free)]) == list(range(20))


def test_cache_in_four_bits_stays_near_the_whole_one():
    """A value is held to within half a step, its deviation 0.08 of the values' own; means over tokens are nearer."""
    m = _model()
    ids = torch.stack(_prompts([40, 40, 40], seed=3))
    a, b = DecodeEngine(m, 3, 60), DecodeEngine(m, 3, 60, kv_bits=4)
    assert torch.equal(a.prefill(ids), b.prefill(ids))
    tok = ids[:, 7].contiguous()
    ha = m.decode_hidden(tok, a.positions, a.slots, a.ctx_lens, a.cache)
    c = b.cache
    ops.paged_layout(b.new_lens, b.ctx_lens, c.block_tables, c.free_list, c.free_range, 3, 16, b.layout, rows_per_request=1)
    assert torch.equal(a.positions, b.positions) and torch.equal(a.ctx_lens, b.ctx_lens)
    hb = m.decode_hidden(tok, b.positions, b.slots, b.ctx_lens, c)
    assert float((ha - hb).norm() / ha.norm()) < 0.08
    assert c.nbytes() * 4 < sum(t.numel() * 4 for t in a.cache.k + a.cache.v)


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_rules_in_a_run(kv_bits):
    """No token twice under an unbounded presence penalty; only allowed ones under a mask; a bias wins."""
    m = _model()
    p = torch.stack(_prompts([9, 9], seed=6))
    rules = ops.LogitRules.empty(2, 500, "cpu", bias_entries=2, masked=True)
    rules.penalties[0] = torch.tensor([1.0, 1e6, 0.0])
    rules.mask[1] = 0
    rules.mask[1, 3] = 1 << 4 | 1 << 9
    rules.bias_ids[1, 0], rules.bias[1, 0] = 3 * 32 + 9, 1e4
    eng = DecodeEngine(m, 2, 60, kv_bits=kv_bits, rules=rules)
    toks = [eng.prefill(p)]
    eng.ids.copy_(toks[0])
    for _ in range(20):
        toks.append(eng.step().clone())
    toks = torch.stack(toks, 1)
    assert len(set(toks[0].tolist())) == 21 and toks[1].tolist() == [3 * 32 + 9] * 21
    assert int(rules.counts[0].sum()) == 21 and int(rules.counts[1, 3 * 32 + 9]) == 21
    seen = [t for t in range(500) if int(rules.seen[0, t // 32]) >> (t % 32) & 1]
    assert set(seen) == set(toks[0].tolist()) | set(p[0].tolist())
    # a new run empties the tables
    eng.prefill(p)
    assert int(rules.counts.sum()) == 2


def test_rules_without_counts():
    m = _model()
    mask = torch.zeros(2, 16, dtype=torch.int32)
    mask[:, 2] = 1 << 7
    for kv_bits in (16, 4):
        eng = DecodeEngine(m, 2, 60, kv_bits=kv_bits, rules=ops.LogitRules(mask=mask, vocab=500))
        eng.ids.copy_(eng.prefill(torch.stack(_prompts([9, 9]))))
        assert eng.step().tolist() == [71, 71]
    # nothing allowed: no token, and the run goes on
    eng = DecodeEngine(m, 2, 60, kv_bits=4, rules=ops.LogitRules(mask=torch.zeros_like(mask), vocab=500))
    out = eng.prefill(torch.stack(_prompts([9, 9])))
    assert out.tolist() == [-1, -1]
    eng.ids.copy_(out)
    assert eng.step().tolist() == [-1, -1]


def test_blocks_run_out():
    m = _model()
    eng = DecodeEngine(m, 2, 64, kv_bits=4, n_blocks=3)
    p = _prompts([30, 20])
    eng.start(torch.cat(p), [30, 20])
    assert eng.blocks_missing() == 1 and eng.cache.free_range.tolist()[1] == 0
    eng.step()  # (goes on without the tokens that have no block)
    eng.finish([1])
    assert int(eng.cache.free_range[1]) == 1


def test_refusals():
    m = _model()
    with pytest.raises(ValueError):
        DecodeEngine(m, 1, 32, kv_bits=8)
    with pytest.raises(ValueError):
        DecodeEngine(m, 1, 32, n_blocks=3)
    with pytest.raises(ValueError):
        DecodeEngine(m, 2, 32, rules=ops.LogitRules.empty(3, 500, "cpu"))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_layout(i, i[:1], i.view(2, 1), i, torch.zeros(3, dtype=torch.int32), 2)
    e16, e4 = DecodeEngine(m, 2, 32), DecodeEngine(m, 2, 32, kv_bits=4)
    p = _prompts([4])[0]
    for call in (lambda: e16.start(p, [4, 0]), lambda: e16.finish([0]), lambda: e4.finish([2]), lambda: e4.start(p, [4]),
                 lambda: e4.start(p, [3, 0]), lambda: e4.start(p, [-1, 5]), lambda: e4.start(torch.zeros(33, dtype=torch.int32), [33, 0])):
        with pytest.raises(ValueError):
            call()
    e4.start(p, [4, 0])
    with pytest.raises(ValueError):
        e4.start(p, [4, 0])
    assert torch.equal(e4.start(p[:0], [0, 0]), e4.ids)
