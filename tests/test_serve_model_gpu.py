# SPDX-License-Identifier: MIT
"""The decode engine on a 4-bit cache and under rules, on the GPU: the captured step against the eager one while requests come
and go, and against the bf16 cache."""
import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine, Qwen2Config, Qwen2Model
from barlink_sm86_b200.parallel import TPComm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    cfg = Qwen2Config(hidden=1024, layers=3, n_heads=8, n_kv_heads=2, head_dim=128, intermediate=2816, vocab=4096, name="test")
    return Qwen2Model(cfg, TPComm.single(), "cuda:0", torch.bfloat16, seed=3)


def _ids(seed, n):
    return torch.randint(0, 4096, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()


def _rules(batch):
    r = ops.LogitRules.empty(batch, 4096, bias_entries=1, masked=True)
    r.penalties.copy_(torch.tensor([1.3, 0.4, 0.2]).cuda().expand(batch, 3))
    r.mask[0, ::2] = 0
    r.bias_ids[1, 0], r.bias[1, 0] = 77, 0.5
    return r


def _run(model, graph, ruled, block):
    eng = DecodeEngine(model, 5, 400, use_graph=graph, kv_bits=4, rules=_rules(5) if ruled else None, block_size=block, n_blocks=3200 // block)
    toks = []
    out = eng.start(torch.cat([_ids(1, 130), _ids(2, 7), _ids(3, 33)]), [130, 7, 0, 33, 0])
    eng.ids.copy_(out)
    if graph:
        eng.capture()
        assert torch.equal(eng.ids, out) and eng.ctx_lens.tolist() == [130, 7, 0, 33, 0]
    for i in range(40):
        if i == 9:
            out = eng.start(_ids(4, 61), [0, 0, 61, 0, 0])
            eng.ids.copy_(out)
        if i == 20:
            eng.finish([0, 3])
            out = eng.start(_ids(5, 200), [200, 0, 0, 0, 0])
            eng.ids.copy_(out)
        toks.append(torch.where(eng.new_lens > 0, eng.step(), -1).clone())
    assert eng.ctx_lens.tolist() == [220, 47, 92, 0, 0] and eng.blocks_missing() == 0
    return torch.stack(toks), eng


@pytest.mark.parametrize("ruled", [False, True])
@pytest.mark.parametrize("block", [16, 32])
def test_captured_step_equals_the_eager_one(ext, model, ruled, block):
    a, ea = _run(model, False, ruled, block)
    b, eb = _run(model, True, ruled, block)
    assert torch.equal(a, b)
    if ruled:
        assert torch.equal(ea.rules.counts, eb.rules.counts) and torch.equal(ea.rules.seen, eb.rules.seen)
        assert bool((b[:, 0][b[:, 0] >= 0] // 32 % 2 == 1).all())  # the mask of request 0
    assert ext.gemm_error_flag(0) == 0 and ext.attn_error_flag(0) == 0 and ext.kv4_error_flag(0) == 0


def test_step_stays_near_the_bf16_cache(model):
    """As on the CPU path: a value's deviation of 0.08 of the values' own, means over tokens are nearer; bf16 noise of 0.02 beside it."""
    lens = [300, 17, 64]
    ids = torch.cat([_ids(10 + i, n) for i, n in enumerate(lens)])
    e4 = DecodeEngine(model, 3, 400, use_graph=False, kv_bits=4)
    first = e4.start(ids, lens)
    for b, n in enumerate(lens):
        e16 = DecodeEngine(model, 1, 400, use_graph=False)
        at = sum(lens[:b])
        e16.prefill(ids[at:at + n][None])
        h16 = model.decode_hidden(first[b:b + 1].contiguous(), e16.positions, e16.slots, e16.ctx_lens, e16.cache)
        if b == 0:
            c = e4.cache
            ops.paged_layout(e4.new_lens, e4.ctx_lens, c.block_tables, c.free_list, c.free_range, 3, 16, e4.layout, rows_per_request=1)
            h4 = model.decode_hidden(first, e4.positions, e4.slots, e4.ctx_lens, c)
        assert float((h4[b].float() - h16[0].float()).norm() / h16[0].float().norm()) < 0.1


def test_rules_on_the_bf16_cache(model):
    """The engine's other cache, captured: no token twice under an unbounded presence penalty."""
    r = ops.LogitRules.empty(2, 4096)
    r.penalties[:, 1] = 1e6
    eng = DecodeEngine(model, 2, 120, rules=r)
    out = eng.prefill(torch.stack([_ids(20, 50), _ids(21, 50)]))
    eng.ids.copy_(out)
    eng.capture()
    toks = [out] + [eng.step().clone() for _ in range(60)]
    for t in torch.stack(toks, 1).tolist():
        assert len(set(t)) == 61
    assert r.counts.sum(1).tolist() == [61, 61]
