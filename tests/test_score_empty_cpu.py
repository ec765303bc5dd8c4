# SPDX-License-Identifier: MIT
"""Log probabilities of no rows at all: empty results of the right shapes, as on the GPU (CPU path, shards, two gloo ranks, the model)."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from barlink_sm86_b200 import ops
from barlink_sm86_b200.parallel import TPComm
from test_extend_cpu import _model


def _shapes(r, ids, top):
    assert r.logprobs.shape == ids.shape and r.entropy.shape == (0,) and r.top_ids.shape == r.top_logprobs.shape == (0, top)
    assert r.top_ids.dtype == torch.int32 and r.logprobs.dtype == r.entropy.dtype == r.top_logprobs.dtype == torch.float32


IDS = [(0,), (0, 1), (0, 3), (0, 0)]


@pytest.mark.parametrize("shape", IDS)
@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("n", [50, 0])
def test_one_rank(shape, top, n):
    ids = torch.zeros(shape, dtype=torch.int32)
    _shapes(ops.token_logprobs(torch.zeros(0, n), ids, top), ids, top)
    given, parts, top_ids, top_val = ops.token_logprob_parts(torch.zeros(0, n), ids, top)
    assert given.shape == ids.shape and parts.shape == (0, 3) and top_ids.shape == top_val.shape == (0, top)
    if n:
        shards = [ops.token_logprob_parts(torch.zeros(0, n), ids, top, n * r) for r in range(2)]
        _shapes(ops.TokenLogprobs(*ops.ref.token_logprobs_of(*ops.ref.join_token_logprobs(shards))), ids, top)


@pytest.mark.parametrize("shape", [(3, 0)])
def test_rows_without_ids(shape):
    r = ops.token_logprobs(torch.zeros(3, 50), torch.zeros(shape, dtype=torch.int32), 2)
    assert r.logprobs.shape == shape and r.entropy.shape == (3,) and r.top_ids.tolist() == [[0, 1]] * 3


def _scores(comm):
    m = _model(comm, 501)
    r = [m.token_logprobs(torch.zeros(0, 128), torch.zeros(0, dtype=torch.int32), top) for top in (0, 4)]
    return r + [comm.token_logprobs_vocab_parallel(torch.zeros(0, m.w.vocab_local), torch.zeros(s, dtype=torch.int32), m.w.vocab_local, 501, 4) for s in IDS] + [
        comm.token_logprobs_vocab_parallel(torch.zeros(3, m.w.vocab_local), torch.zeros(3, 0, dtype=torch.int32), m.w.vocab_local, 501, 4)]


def _check(got):
    for r, ids, top in zip(got, [(0,), (0,)] + IDS, [0, 4] + [4] * len(IDS)):
        _shapes(ops.TokenLogprobs(*r), torch.zeros(ids), top)
    assert got[-1][0].shape == (3, 0) and got[-1][2].tolist() == [[0, 1, 2, 3]] * 3


def _rank(rank, path):
    dist.init_process_group("gloo", init_method="file://" + os.path.join(path, "meet"), rank=rank, world_size=2)
    torch.save([tuple(r) for r in _scores(TPComm(dist.group.WORLD))], os.path.join(path, "out%d.pt" % rank))
    dist.barrier()
    dist.destroy_process_group()


def test_model():
    _check(_scores(TPComm.single()))


def test_two_ranks(tmp_path):
    mp.spawn(_rank, args=(str(tmp_path),), nprocs=2)
    for rank in range(2):
        _check(torch.load(tmp_path / ("out%d.pt" % rank)))
