"""Appending to pools of 4 bits with factors at the ends of fp32's range (needs a B200).

Rows are divided by a KV head's factor in fp32, whatever the factor is, and both of the
append's ways (16-byte pieces, and any other rows) hold what the definition says of the quotients:
exactly, as in test_gpu_fp4_append.py.
"""

import math

import pytest
import torch

import fp4_helpers as fp4
from refinekv_b200 import fp4_pool, paged_append

pytestmark = pytest.mark.gpu
DEV = "cuda"

FACTORS = [1.0, 0.3, -2.0, 1e-30, 1e30, 2.0 ** -60, 2.0 ** 60, 2.0 ** -61, 2.0 ** 61, 2.0 ** 127, 3e38,
           2.0 ** -126, 1e-40, 2.0 ** -149, 0.0, -0.0, math.inf, -math.inf, math.nan]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pieces", [True, False])
@pytest.mark.parametrize("dim", [128, 96])
def test_any_factor_divides(dim, pieces, dtype):
    gen = torch.Generator(device=DEV).manual_seed(dim)
    heads, tokens, block = len(FACTORS), 64, 16
    # blocks of 16 channels from 2^-140 to 2^126, some of the factor's own size, zeros and ones
    sizes = torch.randint(-140, 127, (tokens, heads, dim // 16), generator=gen, device=DEV)
    factor = torch.tensor(FACTORS, device=DEV)
    near = torch.frexp(factor).exponent.clamp(-140, 120).expand(tokens, heads)
    sizes[..., 0] = near + torch.randint(-12, 6, near.shape, generator=gen, device=DEV)
    rows = torch.randn(2, tokens, heads, dim, generator=gen, device=DEV)
    rows = torch.ldexp(rows, sizes.clamp(-140, 126).repeat_interleave(16, -1)).to(dtype)
    rows[:, 0] = 0
    rows[:, 1] = 1
    key, value = rows
    if not pieces:
        wide = torch.zeros(2, tokens, heads, dim + 1, device=DEV, dtype=dtype)
        wide[..., 1:] = rows
        key, value = wide[..., 1:]
    pages = tokens // block
    table = torch.randperm(pages, generator=gen, device=DEV).int()[None]
    at = torch.arange(tokens, device=DEV)
    pools = [fp4_pool(pages, heads, block, dim) for _ in "kv"]
    scales = factor, factor.flip(0).contiguous()
    want = []
    for x, by in zip(rows, scales):
        pool = fp4_pool(pages, heads, block, dim)
        for part, new in zip(fp4.parts(pool), fp4.quantise(x.float() / by[:, None])):
            part.transpose(1, 2)[table[0].long()[at // block], at % block] = new
        want.append(pool)
    paged_append(key, value, *pools, table, at, sequence_ids=torch.zeros_like(at).int(),
                 key_scale=scales[0], value_scale=scales[1])
    for pool, expected in zip(pools, want):
        wrong = (pool != expected).any(0).flatten(1).any(1)
        assert not bool(wrong.any()), [i for i, w in enumerate(wrong.tolist()) if w]
