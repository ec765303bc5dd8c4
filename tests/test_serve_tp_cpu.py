# SPDX-License-Identifier: MIT
"""The decode engine on a 4-bit cache and under rules, two gloo ranks against one."""
import os

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import DecodeEngine, Qwen2Config, Qwen2Model
from barlink_sm86_b200.parallel import TPComm


def _run(comm):
    # (an odd vocabulary: the second rank's slice ends in padding, which no rule may choose)
    cfg = Qwen2Config(hidden=128, layers=2, n_heads=4, n_kv_heads=2, head_dim=64, intermediate=256, vocab=501, name="test")
    m = Qwen2Model(cfg, comm, seed=7)
    rules = ops.LogitRules.empty(3, 501, "cpu", bias_entries=1, masked=True)
    rules.penalties.copy_(torch.tensor([1.5, 0.5, 0.25]).expand(3, 3))
    rules.mask[1, ::3] = 0
    rules.mask[2] = 0
    rules.mask[2, 15] = 1 << 20   # token 500 alone, which is the last rank's
    rules.bias_ids[0, 0], rules.bias[0, 0] = 400, 0.1
    eng = DecodeEngine(m, 3, 64, kv_bits=4, rules=rules)
    g = torch.Generator().manual_seed(1)
    lens = [20, 3, 9]
    out = eng.start(torch.randint(0, 501, (32,), generator=g, dtype=torch.int32), lens)
    toks = [out]
    eng.ids.copy_(out)
    for _ in range(10):
        toks.append(eng.step().clone())
    return torch.stack(toks, 1), rules.counts


def _rank(rank, path):
    dist.init_process_group("gloo", init_method="file://" + os.path.join(path, "meet"), rank=rank, world_size=2)
    toks, counts = _run(TPComm(dist.group.WORLD))
    torch.save((toks, counts), os.path.join(path, "out%d.pt" % rank))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_choose_the_tokens_of_one(tmp_path):
    want, counts = _run(TPComm.single())
    mp.spawn(_rank, args=(str(tmp_path),), nprocs=2)
    for rank in range(2):
        toks, c = torch.load(tmp_path / ("out%d.pt" % rank))
        assert torch.equal(toks, want) and torch.equal(c, counts)
    assert want[2].tolist() == [500] * 11
