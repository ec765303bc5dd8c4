# SPDX-License-Identifier: MIT
"""The CPU path of token log probabilities, its refusals, and the joining of a vocabulary's shards (64-bit sums, rounded once to fp32: half
a step, 2^-24 of the value, and of the greatest logit where shards are joined from fp32 parts)."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops


def _x(rows=4, n=501):
    return torch.randn(rows, n, generator=torch.Generator().manual_seed(3)) * 3


def test_values():
    x = _x()
    ids = torch.tensor([0, 7, 500, -1], dtype=torch.int32)
    r = ops.token_logprobs(x, ids, 6)
    logp = torch.log_softmax(x.double(), -1)
    assert (r.logprobs[:3].double() - logp[[0, 1, 2], [0, 7, 500]]).abs().max() < 2e-6 and r.logprobs[3] == -math.inf
    assert (r.entropy.double() + (logp.exp() * logp).sum(-1)).abs().max() < 2e-6
    assert torch.equal(r.top_ids.long(), torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :6])
    assert (r.top_logprobs.double() - logp.sort(-1, descending=True).values[:, :6]).abs().max() < 2e-6


def test_rows_without_probabilities():
    x = _x(4, 10)
    x[0], x[1, 3], x[2, 4] = -math.inf, math.nan, math.inf
    x[3, 2:] = -math.inf
    r = ops.token_logprobs(x, torch.zeros(4, 2, dtype=torch.int32), 3)
    assert (r.logprobs[0] == -math.inf).all() and r.entropy[0] == 0 and (r.top_ids[0] == -1).all() and (r.top_logprobs[0] == -math.inf).all()
    assert torch.isnan(r.logprobs[1:3]).all() and torch.isnan(r.entropy[1:3]).all() and torch.isnan(r.top_logprobs[1:3]).all()
    assert (r.top_ids[3] >= 0).tolist() == [True, True, False] and r.top_logprobs[3, 2] == -math.inf


@pytest.mark.parametrize("world", [1, 2, 5])
def test_joined_shards(world):
    x, vocab = _x(6, 500), 497
    x[1, :110] = -math.inf
    x[2] = torch.round(x[2])  # ties, also between shards
    x[3] = -math.inf
    x[4, 3] = math.nan
    ids = torch.randint(0, vocab, (6, 3), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    per = 500 // world
    parts = [ops.token_logprob_parts(x[:, r * per:(r + 1) * per], ids, 4, r * per, vocab) for r in range(world)]
    got = ops.ref.token_logprobs_of(*ops.ref.join_token_logprobs(parts))
    want = ops.token_logprobs(x, ids, 4, 0, vocab)
    assert torch.equal(got[2][:4], want[2][:4]) and torch.equal(got[2][5], want[2][5])
    for a, b in zip(got, want):
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        fine = torch.isfinite(b)
        assert torch.equal(torch.isfinite(a), fine) and (a[fine] - b[fine]).abs().max() < 4e-6


def test_refusals():
    x, ids = _x(), torch.zeros(4, dtype=torch.int32)
    for bad in (dict(top=33), dict(top=-1), dict(offset=-1), dict(vocab=-1)):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, ids, **bad)
    for i in (ids.long(), ids[:2], ids[:, None, None]):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, i)
    with pytest.raises(ValueError):
        ops.token_logprobs(x[0], ids)
