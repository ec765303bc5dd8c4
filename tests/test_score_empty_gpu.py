# SPDX-License-Identifier: MIT
"""Log probabilities of no rows, on the GPU: as on the CPU path."""
import pytest
import torch

from barlink_sm86_b200 import ops
from barlink_sm86_b200.models import Qwen2Config, Qwen2Model
from barlink_sm86_b200.parallel import TPComm
from test_score_empty_cpu import IDS, _shapes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", IDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_rows(shape, dtype):
    ids = torch.zeros(shape, dtype=torch.int32, device="cuda")
    for top in (0, 4):
        _shapes(ops.token_logprobs(torch.zeros(0, 50, dtype=dtype, device="cuda"), ids, top), ids, top)
        given, parts, top_ids, top_val = ops.token_logprob_parts(torch.zeros(0, 50, dtype=dtype, device="cuda"), ids, top)
        assert given.shape == ids.shape and parts.shape == (0, 3) and top_ids.shape == top_val.shape == (0, top)


def test_model(ext):
    cfg = Qwen2Config(hidden=1024, layers=1, n_heads=8, n_kv_heads=2, head_dim=128, intermediate=2816, vocab=4096, name="test")
    m = Qwen2Model(cfg, TPComm.single(), "cuda:0", torch.bfloat16, seed=3)
    ids = torch.zeros(0, dtype=torch.int32, device="cuda")
    r = m.token_logprobs(torch.zeros(0, 1024, dtype=torch.bfloat16, device="cuda"), ids, 3)
    _shapes(r, ids, 3)
    assert r.top_ids.is_cuda
