"""Paged attention with bf16 queries is exact to its output's own rounding (needs a B200).

Bounds as in test_gpu_paged_attention.py, but for the weights: held in two bf16
terms of 2^-8 each they are off by 2^-16 at most, and the tensor cores' sums of a
tile (8 products of two terms, two roundings of 2^-23 each) with __expf's 2^-20 add
less than 2^-18:
  |out - exact| <= A (2 e + 2^-16 + 2^-18 + (rows / 32 + 32) u) + |exact| u
                   + half a unit in the result's last place.
Few rows of unlike values are where a weight's rounding shows: over many rows
it averages out.
"""

import pytest
import torch

from test_gpu_paged_attention import Served

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,hq,hk,dim,block,layout,window", [
    ([2, 3, 5, 9, 0, 1], 32, 8, 128, 32, "HND", None),
    ([4, 2, 77], 28, 4, 128, 16, "NHD", None),
    ([3, 40], 16, 2, 64, 64, "HND", None),
    ([6, 2], 16, 1, 256, 32, "HND", None),
    ([3, 7], 9, 1, 96, 32, "NHD", None),
    ([500, 4, 3000], 16, 2, 192, 16, "HND", 5),
    ([2500], 32, 8, 128, 32, "HND", None),
])
@pytest.mark.parametrize("sharp", [1.0, 4.0])
def test_bf16_queries_lose_only_the_outputs_rounding(lengths, hq, hk, dim, block, layout, window,
                                                     sharp):
    s = Served(lengths, hq, hk, dim, block, layout, seed=dim + block, window=window, sharp=sharp)
    out = s.call(return_lse=False)
    u = 2.0 ** -23
    for i, (k, v) in enumerate(zip(s.keys, s.values)):
        if len(k) == 0:
            continue
        q = s.q[i].double().view(hk, hq // hk, dim)
        k, v = k.double().transpose(0, 1), v.double().transpose(0, 1)
        scale = dim ** -0.5
        p = (q @ k.transpose(1, 2) * scale).softmax(-1)
        want, size = (p @ v).reshape(hq, dim), (p @ v.abs()).reshape(hq, dim)
        e = (q.abs() @ k.abs().transpose(1, 2) * scale).amax(-1).reshape(hq) * dim / 8 * u
        weights = 2 * e + 2 ** -16 + 2 ** -18 + (k.shape[1] / 32 + 32) * u
        half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 1 - 8)
        tol = size * weights[:, None] + want.abs() * u + half + 1e-38
        off = (out[i].double() - want).abs()
        assert bool((off <= tol).all()), (i, float((off / tol).max()))
