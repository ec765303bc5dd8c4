# SPDX-License-Identifier: MIT
"""Alternatives on many rows, where a block has a row (or half of one) and takes many laps for it: a lap is 10240 bf16 logits, or 5120 fp32 ones, so that
152064 are 15 or 30.  The tolerances of test_score_gpu hold: a term is off by 2^-21 at most; it goes through 21 additions in its lap (fp32: 11) and through one
join a lap and 11 of threads, warps and blocks, two roundings each: 73 (93) roundings of 2^-24; and where a join changes the maximum, 2^-22 once more, which
happens to a row's large terms some five times (the k-th lap holds the largest so far with probability 1 / k: 4 of 30).  Together below
(8 + 93 + 20) 2^-24 < 2^-17."""
import math

import pytest
import torch

from barlink_sm86_b200 import ops
from test_score_gpu import _check, _g, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n", [(300, 152064), (297, 60001), (150, 152064), (160, 256000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [1, 5, 20, 32])
def test_many_laps(rows, n, dtype, top):
    x = _logits(rows + top, rows, n, dtype)
    ids = torch.randint(0, n, (rows,), generator=_g(1), device="cuda", dtype=torch.int32)
    _check(x, ids, ops.token_logprobs(x, ids, top), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_greater_ones_come_later(dtype, top):
    """Logits that rise, and ones that fall; a last lap, and a rest behind the last vector, with the greatest; equal ones throughout."""
    n, rows = 70003, 300
    up = torch.linspace(-8, 8, n, device="cuda")
    x = torch.stack([up, up.flip(0)] + [_logits(9, 1, n, torch.float32, 1.0)[0] for _ in range(3)]).to(dtype)
    x[2, -40:] = torch.arange(40, device="cuda").to(dtype) + 10
    x[3, -3:] = 50
    x[4] = torch.round(x[4].float()).to(dtype)
    x = x.repeat(rows // 5, 1)
    ids = torch.randint(0, n, (rows, 2), generator=_g(3), device="cuda", dtype=torch.int32)
    _check(x, ids, ops.token_logprobs(x, ids, top), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_rows_among_many(dtype):
    n, rows, top = 152064, 300, 24
    x = _logits(4, rows, n, dtype)
    x[::4] = torch.where(torch.rand(rows // 4, n, generator=_g(6), device="cuda") < 0.999, -math.inf, x[::4].float()).to(dtype)
    x[1::4, : n - 7000] = -math.inf   # the first laps have nothing
    x[2::4, 10:] = -math.inf          # fewer than are asked for
    x[6] = -math.inf
    ids = torch.randint(0, 10, (rows,), generator=_g(1), device="cuda", dtype=torch.int32)
    keep = torch.arange(rows, device="cuda") != 6
    got = ops.token_logprobs(x, ids, top)
    _check(x[keep], ids[keep], ops.TokenLogprobs(*(t[keep] for t in got)), top)
    assert got.logprobs[6] == -math.inf and got.entropy[6] == 0 and (got.top_ids[6] == -1).all() and (got.top_logprobs[6] == -math.inf).all()
