"""Rotation and append of more tokens than one round of CTAs takes (needs a B200).

Bounds of test_gpu_rotary.py.
"""

import pytest
import torch

from refinekv_b200 import apply_rotary, paged_append, rotary_table
from refinekv_b200.attention import device_status
from test_gpu_paged_append import make_pool, rows_of
from test_gpu_rotary import assert_rotated, rotate64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


@pytest.mark.parametrize("lead,hq,hk,dim,rotary,dtype", [
    ((3001,), 32, 8, 128, 128, torch.bfloat16),
    ((3, 1021), 28, 4, 96, 64, torch.float32),
    ((4, 2003), 14, 2, 64, 64, torch.bfloat16),
    ((2501,), 32, 0, 64, 20, torch.bfloat16),   # one element a piece
    ((2, 1501), 6, 2, 128, 50, torch.float32),
    ((30011,), 2, 1, 32, 32, torch.bfloat16),   # CTAs of one warp
    ((1201,), 200, 8, 256, 256, torch.bfloat16),  # heads over several slices
])
@pytest.mark.parametrize("interleaved", [False, True])
def test_every_round_rotates_its_own_token(lead, hq, hk, dim, rotary, dtype, interleaved):
    gen = torch.Generator(device=DEV).manual_seed(dim + rotary)
    table = rotary_table(rotary, 5000)
    q = _normal(gen, *lead, hq, dim, dtype=dtype)
    k = _normal(gen, *lead, hk, dim, dtype=dtype) if hk else None
    at = torch.randint(0, 5000, lead, generator=gen, device=DEV)
    at.view(-1)[-1] = 4999
    got_q, got_k = apply_rotary(q, k, at, table, interleaved=interleaved)
    assert_rotated(got_q, *rotate64(q, at, table, interleaved))
    if hk:
        assert_rotated(got_k, *rotate64(k, at, table, interleaved))
    # positions of another type and stride
    strided = torch.stack([at, -at], -1)[..., 0].int()
    wide = torch.zeros(*lead, 2, device=DEV, dtype=torch.int32)
    wide[..., 0] = strided
    again, _ = apply_rotary(q, None, wide[..., 0], table, interleaved=interleaved)
    assert torch.equal(again, got_q)


@pytest.mark.parametrize("hq,hk,dim,rotary,block,layout,dtype", [
    (32, 8, 128, 128, 32, "HND", torch.bfloat16),
    (0, 4, 128, 64, 16, "NHD", torch.float32),
    (7, 1, 64, 20, 64, "HND", torch.bfloat16),
])
def test_every_round_appends_its_own_token(hq, hk, dim, rotary, block, layout, dtype):
    gen = torch.Generator(device=DEV).manual_seed(dim + rotary)
    lengths = [4001, 17, 2500, 3333]
    n, blocks = len(lengths), -(-max(lengths) // block)
    pages = n * blocks + 2
    pt = torch.randperm(pages, generator=gen, device=DEV)[: n * blocks].view(n, blocks).int()
    kp, kv = make_pool(pages, hk, block, dim, layout)
    vp, vv = make_pool(pages, hk, block, dim, layout)
    at = torch.cat([torch.arange(L) for L in lengths])
    ids = torch.repeat_interleave(torch.arange(n), torch.tensor(lengths))
    order = torch.randperm(len(at), generator=torch.Generator().manual_seed(1))
    at, ids = at[order].to(DEV, torch.int32), ids[order].to(DEV, torch.int32)
    tokens = len(at)
    spoilt = torch.arange(tokens, device=DEV) % 7
    at = torch.where(spoilt == 3, -1, at)               # padding
    at = torch.where(spoilt == 5, blocks * block, at)   # past the page table
    both = _normal(gen, tokens, hq + 2 * hk, dim, dtype=dtype)
    q, k, v = both[:, :hq], both[:, hq:hq + hk], both[:, hq + hk:]
    table = rotary_table(rotary, blocks * block + 1)
    ws = {}
    got = paged_append(k, v, kp, vp, pt, at, layout=layout, query=q if hq else None,
                       cos_sin=table, sequence_ids=ids, workspace=ws)
    assert device_status(ws) == 2
    good = ((spoilt != 3) & (spoilt != 5)).nonzero()[:, 0]
    g_ids, g_at = ids[good], at[good]
    assert_rotated(rows_of(kv, pt, g_ids, g_at, block), *rotate64(k[good], g_at, table))
    assert torch.equal(rows_of(vv, pt, g_ids, g_at, block), v[good].to(torch.bfloat16))
    for view in (kv, vv):
        assert int((view != 7.0).any(-1).any(-1).sum()) == len(good)
    if hq:
        assert not bool(got[spoilt == 3].any())
        rest = (spoilt != 3).nonzero()[:, 0]
        assert_rotated(got[rest], *rotate64(q[rest], at[rest], table))
