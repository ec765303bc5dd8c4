# SPDX-License-Identifier: MIT
"""The polynomial that stands in for a share of the exponentials (csrc/chunk_attn_kernels.cu, ex2_poly), from the coefficients in the source.

What tolerances of attention of new tokens allow beside the roundings of the result and of P is 2^-10 of sum p |v|: scores are off by less than 2^-11, the
polynomial by less than 2^-13 (7.5e-5; sums of at most 2^14 terms in fp32 in chains of less than 2^9: 2^-15), 2^-11 + 2^-13 + 2^-15 < 2^-10."""
import os
import re

import torch

import barlink_sm86_b200


def test_off_by_less_than_stated():
    path = os.path.join(os.path.dirname(barlink_sm86_b200.__file__), "csrc", "chunk_attn_kernels.cu")
    with open(path) as f:
        body = re.search(r"float2 ex2_poly\(float2 x\) \{(.*?)\n\}", f.read(), re.S).group(1)
    c = [float(x) for x in re.findall(r"make_float2\((0\.\d+)f, \1f\)", body)]
    assert len(c) == 4
    f = torch.linspace(-0.5, 0.5, 200001, dtype=torch.float32)
    p = torch.full_like(f, c[0])
    for x in c[1:]:
        p = (p.double() * f.double() + x).float()  # (a fused multiply-add rounds once)
    off = (p.double() / torch.exp2(f.double()) - 1).abs().max()
    assert off < 7.5e-5 < 2.0 ** -13
