# SPDX-License-Identifier: MIT
"""Further tokens on top of the cache, log probabilities beside the steps, and waits that run out, on the GPU."""
import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine, Qwen2Config, Qwen2Model
from barlink_sm86_b200.parallel import TPComm
from test_chunk_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    cfg = Qwen2Config(hidden=1024, layers=3, n_heads=8, n_kv_heads=2, head_dim=128, intermediate=2816, vocab=4096, name="test")
    return Qwen2Model(cfg, TPComm.single(), "cuda:0", torch.bfloat16, seed=3)


def _ids(seed, n):
    return torch.randint(0, 4096, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()


@pytest.mark.parametrize("max_tokens", [50, 8192])
def test_pieces_equal_the_dense_pass(ext, model, max_tokens):
    """Two sums of the same terms.  A layer rounds some eight times to bf16, each by 2^-8 / sqrt 3 at most in the mean; where the two differ, so do the
    roundings behind: over three layers and both sides sqrt(2 * 24) * 2^-8 / sqrt 3 = 2^-6 of the final values, in the mean.  Twice that is allowed."""
    lens = [61, 0, 200, 1, 33]
    eng = DecodeEngine(model, 5, 256)
    got = []
    run = model.extend_packed
    try:
        model.extend_packed = lambda *a: got.append(run(*a)) or got[-1]
        ids = _ids(1, sum(lens))
        nxt, lp = eng.score(ids, lens, 5, max_tokens)
    finally:
        del model.extend_packed
    got = torch.cat(got)
    at = 0
    for b, n in enumerate(lens):
        if n:
            want = model.prefill(ids[None, at:at + n]).double()
            diff = (got[at:at + n].double() - want)
            assert float(diff.pow(2).mean().sqrt()) < 2 ** -5 * float(want.pow(2).mean().sqrt())
            at += n
    # the log probabilities are those of the pass's own logits: sums of 4096 terms in fp32, logits below 16
    p = torch.log_softmax(model.logits_local(got).double(), -1)
    follows = torch.cat([ids[1:], ids[:1]])
    ends = torch.tensor([60, 260, 261, 294], device="cuda")
    follows[ends] = nxt[[0, 2, 3, 4]]
    assert (lp.logprobs.double() - p.gather(1, follows.long()[:, None])[:, 0]).abs().max() < 1e-4
    assert (lp.top_logprobs.double() - p.topk(5).values).abs().max() < 1e-4
    assert (lp.entropy.double() + (p.exp() * p).sum(1)).abs().max() < 1e-3
    assert torch.equal(lp.top_ids[ends, 0], nxt[[0, 2, 3, 4]]) and nxt[1] == eng.ids[1]


def _talk(model, graph, kv_bits):
    """A conversation of three requests: prompts, steps, turns of other lengths, steps, and the whole scored."""
    eng = DecodeEngine(model, 3, 512, use_graph=graph, kv_bits=kv_bits, logprobs=4)
    if kv_bits == 4:
        out = eng.start(torch.cat([_ids(1, 130), _ids(2, 7)]), [130, 7, 0])
    else:
        out = eng.prefill(torch.stack([_ids(i, 40) for i in range(3)]))
    eng.ids.copy_(out)
    if graph:
        eng.capture()
    toks, scores = [], []
    for turn in range(3):
        for _ in range(5):
            toks.append(eng.step().clone())
            scores.append(tuple(t.clone() for t in eng.logprobs))
        new = [torch.cat([eng.ids[:1], _ids(10 + turn, 20)]), _ids(20 + turn, 3), _ids(30 + turn, 70)]
        out, lp = eng.score(torch.cat(new), [21, 3, 70], 2, max_tokens=64)
        eng.ids.copy_(out)
        toks.append(out)
        scores.append(tuple(lp))
    return torch.stack(toks), scores, eng


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_turns_between_captured_steps(ext, model, kv_bits):
    a, sa, ea = _talk(model, False, kv_bits)
    b, sb, eb = _talk(model, True, kv_bits)
    assert torch.equal(a, b) and torch.equal(ea.ctx_lens, eb.ctx_lens)
    for x, y in zip(sa, sb):
        assert all(torch.equal(u, v) for u, v in zip(x, y))
    for toks, s in zip(a, sa):
        if len(s[0]) == 3:  # a step: the token chosen is the likeliest
            rows = slice(None) if kv_bits == 16 else slice(0, 2)
            assert torch.equal(s[2][rows, 0], toks[rows]) and torch.equal(s[3][rows, 0], s[0][rows])
    if kv_bits == 4:
        assert ea.blocks_missing() == 0 and ea.tokens_lost() == 0


@pytest.fixture
def polls(ext):
    """Sets how often a wait looks; back to what it was afterwards, and the error word to 0."""
    before = ext.chunk_attn_wait_polls(0)
    yield ext.chunk_attn_wait_polls
    ext.chunk_attn_wait_polls(before)
    torch.cuda.synchronize()
    ext.chunk_attn_error_clear(0)


def _word(ext):
    out = torch.zeros(1, dtype=torch.int32).pin_memory()
    ext.chunk_attn_error_into(out, 0)
    torch.cuda.synchronize()
    return int(out)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("heads,lens", [((28, 4, 128), [(700, 3000), (1, 20), (0, 7), (5, 900)]), ((8, 1, 128), [(3, 9000)]), ((8, 8, 64), [(30, 700)] * 40)])
def test_a_wait_that_runs_out(ext, polls, heads, lens, q4):
    """A run that gives up says so and leaves NaN, not what stood there; a later call is as ever."""
    c = Case(heads, 16, lens, q4, seed=5)

    def run():
        if q4:
            return ops.paged_attn_chunk_q4(c.qkv, c.cache, c.table, c.cu, c.lens, *heads, c.scale)
        return ops.paged_attn_chunk(c.qkv, c.k, c.v, c.table, c.cu, c.lens, *heads, c.scale)

    polls(1 << 24)
    want = run()
    assert _word(ext) == 0 and bool(want.isfinite().all())
    polls(0)
    got = run()
    assert _word(ext) == 1 and bool(got.isnan().all())
    ext.chunk_attn_error_clear(0)
    # some look once or twice, and may be in time: a row is right or NaN, and NaN only where the word says so
    for n in (1, 2, 4):
        polls(n)
        got = run()
        bad = got.view(-1, heads[2]).isnan()
        assert torch.equal(bad.all(1), bad.any(1)) and (not bool(bad.any()) or _word(ext) == 1)
        assert torch.equal(torch.where(bad, 0, got.view(-1, heads[2])), torch.where(bad, 0, want.view(-1, heads[2])))
        ext.chunk_attn_error_clear(0)
    for n in (1 << 24, (1 << 32) - 1):
        polls(n)
        assert torch.equal(run(), want) and _word(ext) == 0


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_the_engine_says_so(ext, model, polls, kv_bits):
    eng = DecodeEngine(model, 2, 128, kv_bits=kv_bits)
    polls(1 << 24)
    eng.extend(_ids(1, 40), [30, 10])
    polls(0)
    with pytest.raises(RuntimeError, match="gave up"):
        eng.score(_ids(2, 20), [0, 20], 3)
    polls(1 << 24)
    assert eng.ctx_lens[0] == (30 if kv_bits == 4 else 31) and (kv_bits == 16 or eng.running == [True, False])
    eng.extend(_ids(2, 20), [0, 20])  # (once reported)
