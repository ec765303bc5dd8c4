# SPDX-License-Identifier: MIT
"""Values that are no numbers, in tokens that a new token does not see, are of no account to it (CPU path; fp32, sums of at most 60 terms below 10 in
absolute values: 60 * 10 * 2^-24 < 2^-14)."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [3, 54, 57, 59])
def test_tokens_before_it_do_without(what, at):
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(6, 2, 16, 64, generator=g) for _ in range(2))
    table = torch.tensor([[4, 0, 5, 2], [1, 3, -1, -1]], dtype=torch.int32)
    q = torch.randn(9, 6 * 64, generator=g)
    call = (table, torch.tensor([0, 5, 9], dtype=torch.int32), torch.tensor([60, 4], dtype=torch.int32), 6, 2, 64, 0.125)
    clean = ops.paged_attn_chunk(q, k, v, *call)
    v[table[0, at // 16], 1, at % 16, 7] = what
    k[table[0, 3], 0, 60 % 16:] = what  # (behind the last token)
    got = ops.paged_attn_chunk(q, k, v, *call)
    seen = torch.zeros(9, 6 * 64, dtype=torch.bool)
    seen[max(at - 55, 0):5].view(-1, 6, 64)[:, 3:, 7] = True
    assert not torch.isfinite(got[seen]).any()
    assert (got - clean)[~seen].abs().max() < 2.0 ** -14


def test_a_token_that_sees_nothing_has_zeros():
    k, v = torch.ones(1, 1, 16, 64), torch.full((1, 1, 16, 64), math.nan)
    got = ops.paged_attn_chunk(torch.ones(3, 64), k, v, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32),
                               torch.tensor([1], dtype=torch.int32), 1, 1, 64, 0.125)
    assert (got[:2] == 0).all() and torch.isnan(got[2]).all()
