# SPDX-License-Identifier: MIT
"""Serving operators on the GPU where a run leaves the ordinary (csrc/serve_kernels.cu)."""
import pytest
import torch

from barlink_sm86_b200 import ops
from test_serve_gpu import _layout_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,new,past,bs,per", [(1, 40, 0, 16, 0), (40, 60, 100, 16, 0), (64, 1, 400, 16, 1), (300, 30, 50, 32, 0),
                                                   (900, 5, 40, 16, 4)])
@pytest.mark.parametrize("spare", [None, 0, 10])
@pytest.mark.parametrize("narrow", [0, 2])
def test_lost_tokens_add_up(batch, new, past, bs, per, spare, narrow):
    """Rows of tokens without a slot, in the one block and in the kernel for many rows; a table that ends early; calls one after another."""
    args = _layout_case(batch + new, batch, new, past, bs, None)
    if spare is not None:
        args[4][1] = spare
    if narrow:
        args = (*args[:2], args[2][:, :max(1, args[2].shape[1] - narrow)].contiguous(), *args[3:])
    tokens = batch * per if per else int(args[0].clamp(min=0).sum()) + 3
    cpu, gpu = [t.clone() for t in args], [t.cuda() for t in args]
    lc, lg = torch.tensor([7], dtype=torch.int32), torch.tensor([7], dtype=torch.int32, device="cuda")
    for _ in range(2):
        a = ops.paged_layout(*cpu, tokens, bs, rows_per_request=per, lost=lc)
        b = ops.paged_layout(*gpu, tokens, bs, rows_per_request=per, lost=lg)
        assert torch.equal(lc, lg.cpu()) and torch.equal(a.slots, b.slots.cpu())
        cpu[1], gpu[1] = a.ctx_lens, b.ctx_lens
        cpu[4], gpu[4] = a.free_range, b.free_range
    with pytest.raises(RuntimeError):
        ops.paged_layout(*gpu, tokens, bs, lost=lg.long())


def test_a_captured_step_counts_its_losses():
    from barlink_sm86_b200.models import DecodeEngine, Qwen2Config, Qwen2Model
    from barlink_sm86_b200.parallel import TPComm

    cfg = Qwen2Config(hidden=512, layers=1, n_heads=4, n_kv_heads=2, head_dim=128, intermediate=1024, vocab=1000, name="test")
    eng = DecodeEngine(Qwen2Model(cfg, TPComm.single(), "cuda:0", torch.bfloat16, seed=3), 2, 64, kv_bits=4, n_blocks=3)
    eng.ids.copy_(eng.start(torch.arange(50, dtype=torch.int32, device="cuda"), [30, 20]))
    assert eng.blocks_missing() == 1 and eng.tokens_lost() == 4
    eng.capture()
    assert eng.tokens_lost() == 4  # (the warm-up's own are not counted)
    for _ in range(5):
        eng.step()
    assert eng.tokens_lost() == 4 + 5 + 3


def test_counts_at_the_end_of_32_bits():
    """As many ids as an int32 offset can name: indexes behind the last one are not taken for negative ones."""
    n = 2 ** 31 - 1
    ids = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    last = torch.tensor([3, 99, 3, 40], dtype=torch.int32, device="cuda")
    ids[-4:] = last
    for lo, reset in ((0, False), (n - 600, False), (n - 600, True)):
        r = ops.LogitRules.empty(1, 100)
        ops.count_tokens(r, ids, torch.tensor([lo, n], dtype=torch.int32, device="cuda"), reset=reset)
        want = ops.LogitRules.empty(1, 100, "cpu")
        ops.count_tokens(want, last.cpu(), torch.tensor([0, 4], dtype=torch.int32))
        assert torch.equal(r.counts.cpu(), want.counts) and torch.equal(r.seen.cpu(), want.seen)


def test_the_largest_vocabulary():
    """2^31 - 1 tokens: numbers of words and slices are those of 64-bit arithmetic; the second row's tables begin behind the first's."""
    vocab = 2 ** 31 - 1
    r = ops.LogitRules.empty(2, vocab)
    ids = torch.tensor([0, vocab - 1, vocab - 2, vocab - 2], dtype=torch.int32, device="cuda")
    for reset in (True, False):
        ops.count_tokens(r, ids, torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), reset=reset)
    assert r.counts[:, -2:].tolist() == [[0, 2], [4, 0]] and int(r.counts[0, 0]) == 2 and int(r.counts[1, 0]) == 0
    assert r.seen[:, -1].tolist() == [1 << 30, 1 << 29] and r.seen[:, 0].tolist() == [1, 0]
    r.penalties[:, 2] = 1.0
    x = torch.tensor([[5.0, 6.0, 7.0], [5.0, 9.0, 7.0]], device="cuda")
    got = ops.logits_process(x, r, offset=vocab - 3)
    assert got.tolist() == [[5.0, 6.0, 5.0], [5.0, 5.0, 7.0]]
    assert ops.logits_argmax(x, r, offset=vocab - 3)[0].tolist() == [vocab - 2, vocab - 1]
