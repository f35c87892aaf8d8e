"""Appending to a page pool against the formula in 64 bits (needs a B200).

Rotated rows have the bounds of test_gpu_rotary.py (the pool adds one bf16
rounding); copied rows and everything not written must be bit-identical.
"""

import pytest
import torch

from refinekv_b200 import apply_rotary, paged_append, rotary_table
from refinekv_b200.attention import device_status
from test_gpu_rotary import assert_rotated, rotate64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


def make_pool(pages, heads, block, dim, layout, fill=7.0):
    """A pool of sentinels and its (pages, block, heads, dim) view."""
    shape = (pages, heads, block, dim) if layout == "HND" else (pages, block, heads, dim)
    pool = torch.full(shape, fill, device=DEV, dtype=torch.bfloat16)
    return pool, pool.transpose(1, 2) if layout == "HND" else pool


def rows_of(view, table, ids, positions, block):
    """(tokens, heads, dim) rows of the tokens in a (pages, block, heads, dim) view."""
    ids, positions = ids.long(), positions.long()
    return view[table[ids, positions // block].long(), positions % block]


@pytest.mark.parametrize("lengths,chunk,hq,hk,dim,rotary,block,layout", [
    ([1, 40, 333], 1, 32, 8, 128, 128, 32, "HND"),
    ([70, 5, 16, 17], 0, 7, 1, 64, 32, 16, "NHD"),
    ([129], 50, 4, 2, 96, 96, 64, "HND"),
    ([64, 65], 64, 0, 3, 256, 64, 64, "NHD"),
    ([31, 2], 2, 5, 5, 32, 20, 32, "HND"),  # 10 pairs: no whole 16-byte pieces
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_appended_rows_match_the_formula(lengths, chunk, hq, hk, dim, rotary, block, layout,
                                         dtype, interleaved):
    gen = torch.Generator(device=DEV).manual_seed(dim + block)
    n, blocks = len(lengths), -(-max(lengths) // block)
    pages = n * blocks + 2
    pt = torch.randperm(pages, generator=gen, device=DEV)[: n * blocks].view(n, blocks).int()
    kp, kv = make_pool(pages, hk, block, dim, layout)
    vp, vv = make_pool(pages, hk, block, dim, layout)
    new = [min(L, chunk or L) for L in lengths]
    at = torch.cat([torch.arange(L - m, L) for L, m in zip(lengths, new)])
    ids = torch.repeat_interleave(torch.arange(n), torch.tensor(new))
    shuffle = torch.randperm(len(at))  # tokens in any order
    at, ids = at[shuffle].to(DEV, torch.int32), ids[shuffle].to(DEV, torch.int32)
    tokens = len(at)
    both = _normal(gen, tokens, hq + 2 * hk, dim, dtype=dtype)
    q, k, v = both[:, :hq], both[:, hq:hq + hk], both[:, hq + hk:]
    table = rotary_table(rotary, max(lengths))
    ws = {}
    implied = chunk == 1 and n == tokens
    if implied:
        order = torch.argsort(ids)
        at, ids, q, k, v = at[order], ids[order], q[order], k[order], v[order]
    got = paged_append(k, v, kp, vp, pt, at, layout=layout, query=q if hq else None, cos_sin=table,
                       sequence_ids=None if implied else ids, interleaved=interleaved,
                       workspace=ws)
    want, size = rotate64(k, at, table, interleaved)
    assert_rotated(rows_of(kv, pt, ids, at, block), want, size)
    assert torch.equal(rows_of(vv, pt, ids, at, block), v.to(torch.bfloat16))
    if hq:
        assert got.dtype == dtype
        assert_rotated(got, *rotate64(q, at, table, interleaved))
        assert torch.equal(got, apply_rotary(q, None, at, table, interleaved=interleaved)[0])
    else:
        assert got is None
    # the separate rotation and a plain append write the same bits
    kp2, kv2 = make_pool(pages, hk, block, dim, layout)
    vp2, _ = make_pool(pages, hk, block, dim, layout)
    turned, _ = apply_rotary(k, None, at, table, interleaved=interleaved)
    assert paged_append(turned, v, kp2, vp2, pt, at.long(), layout=layout, sequence_ids=ids) is None
    assert torch.equal(kp2, kp) and torch.equal(vp2, vp)
    # nothing else of the pools was written
    for view in (kv, vv):
        view[pt[ids.long(), at.long() // block].long(), at.long() % block] = 7.0
        assert bool((view == 7.0).all())
    assert device_status(ws) == 0


def test_pools_cut_out_of_one_tensor_and_unaligned_rows():
    gen = torch.Generator(device=DEV).manual_seed(8)
    block, hk, dim = 16, 2, 64
    both = torch.full((6, 2, block, hk, dim), 7.0, device=DEV, dtype=torch.bfloat16)
    pt = torch.tensor([[5, 0], [2, 3]], device=DEV, dtype=torch.int32)
    at = torch.tensor([3, 31], device=DEV, dtype=torch.int64)
    k, v = _normal(gen, 2, hk, dim), _normal(gen, 2, hk, dim)
    paged_append(k, v, both[:, 0], both[:, 1], pt, at, layout="NHD")
    assert torch.equal(both[5, 0, 3], k[0]) and torch.equal(both[3, 1, 15], v[1])
    assert int((both != 7.0).sum()) <= 4 * hk * dim
    # rows at odd elements, a strided head dim
    odd = _normal(gen, 2, hk, dim + 1)[..., 1:]
    skew = _normal(gen, 2, dim, hk).transpose(1, 2)
    paged_append(odd, skew, both[:, 0], both[:, 1], pt, at, layout="NHD")
    assert torch.equal(both[3, 0, 15], odd[1]) and torch.equal(both[5, 1, 3], skew[0])


def test_padding_and_bad_tokens_write_nothing():
    gen = torch.Generator(device=DEV).manual_seed(9)
    hk, dim, block = 2, 64, 16
    table = rotary_table(dim, 40)
    # sequence, position: good, padding, past the page table, past the rotation table, a sequence
    # that does not exist (twice), a page outside the pool (twice), good
    ids = torch.tensor([0, 0, 0, 1, 2, -1, 0, 1, 1], device=DEV, dtype=torch.int32)
    at = torch.tensor([0, -1, 48, 41, 3, 3, 16, 17, 39], device=DEV, dtype=torch.int32)
    pt = torch.tensor([[1, 9, 0], [2, -5, 3]], device=DEV, dtype=torch.int32)
    k, v, q = (_normal(gen, 9, h, dim) for h in (hk, hk, 4))
    for first, healthy in ((2, True), (9, False)):
        kp, kv = make_pool(9, hk, block, dim, "HND")
        vp, vv = make_pool(9, hk, block, dim, "HND")
        ws = {}
        got = paged_append(k[:first], v[:first], kp, vp, pt, at[:first],
                           sequence_ids=ids[:first], query=q[:first], cos_sin=table, workspace=ws)
        assert device_status(ws) == (0 if healthy else 2)
        good = [0] if healthy else [0, 8]
        g = torch.tensor(good, device=DEV)
        assert_rotated(rows_of(kv, pt, ids[g], at[g], block), *rotate64(k[g], at[g], table))
        assert int((vv != 7.0).any(-1).any(-1).sum()) == len(good)
        assert int((kv != 7.0).any(-1).any(-1).sum()) == len(good)
        assert not bool(got[1].any())  # padding: a zero query
        if not healthy:
            assert bool(got[2].isnan().all()) and bool(got[3].isnan().all())
            rest = torch.tensor([4, 5, 6, 7], device=DEV)
            assert_rotated(got[rest], *rotate64(q[rest], at[rest], table))


def test_empty_call_and_reused_buffers():
    pool, _ = make_pool(2, 1, 16, 32, "HND")
    pt = torch.zeros(1, 1, device=DEV, dtype=torch.int32)
    none = torch.empty(0, 1, 32, device=DEV)
    at = torch.empty(0, device=DEV, dtype=torch.int32)
    out = paged_append(none, none, pool, pool, pt, at, query=none)
    assert out.shape == (0, 1, 32) and bool((pool == 7.0).all())
    ws = {}
    one = torch.ones(1, 1, 32, device=DEV)
    at = torch.zeros(1, device=DEV, dtype=torch.int32)
    a = paged_append(one, one, pool, pool, pt[0], at, query=one, workspace=ws)
    b = paged_append(one, one, pool, pool, pt[0], at, query=2 * one, workspace=ws)
    assert a.data_ptr() == b.data_ptr() and float(b[0, 0, 0]) == 2.0


def test_offsets_past_32_bits():
    block, hk, dim = 64, 8, 128
    pages = 33000  # 2.16e9 elements
    kp = torch.empty(pages, hk, block, dim, device=DEV, dtype=torch.bfloat16)
    vp = torch.empty_like(kp)
    pt = torch.tensor([[pages - 1]], device=DEV, dtype=torch.int32)
    gen = torch.Generator(device=DEV).manual_seed(10)
    k, v = _normal(gen, 1, hk, dim), _normal(gen, 1, hk, dim)
    at = torch.tensor([63], device=DEV)
    paged_append(k, v, kp, vp, pt, at)
    assert torch.equal(kp[-1, :, 63], k[0]) and torch.equal(vp[-1, :, 63], v[0])


def test_graph_replay_follows_positions_and_tables():
    gen = torch.Generator(device=DEV).manual_seed(11)
    hk, dim, block = 2, 64, 16
    kp, kv = make_pool(8, hk, block, dim, "HND")
    vp, vv = make_pool(8, hk, block, dim, "HND")
    pt = torch.tensor([[0, 1], [2, 3]], device=DEV, dtype=torch.int32)
    at = torch.tensor([0, 0], device=DEV, dtype=torch.int32)
    k, v, q = _normal(gen, 2, hk, dim), _normal(gen, 2, hk, dim), _normal(gen, 2, 4, dim)
    table = rotary_table(dim, 32)
    ws = {}
    paged_append(k, v, kp, vp, pt, at, query=q, cos_sin=table, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_append(k, v, kp, vp, pt, at, query=q, cos_sin=table, workspace=ws)
    at.copy_(torch.tensor([17, -1]))
    pt.copy_(torch.tensor([[0, 6], [2, 3]]))
    kp.fill_(7.0)
    graph.replay()
    assert_rotated(kv[6, 1], *[x[0] for x in rotate64(k[:1], at[:1], table)])
    assert int((kv != 7.0).any(-1).any(-1).sum()) == 1
    assert_rotated(out[:1], *rotate64(q[:1], at[:1], table))


def test_refusals():
    pool, _ = make_pool(4, 2, 16, 64, "HND")
    k = torch.zeros(2, 2, 64, device=DEV)
    pt = torch.zeros(2, 2, device=DEV, dtype=torch.int32)
    at = torch.zeros(2, device=DEV, dtype=torch.int32)

    def call(key=k, value=None, kp=pool, vp=None, table=pt, positions=at, **kw):
        return paged_append(key, key if value is None else value, kp, kp if vp is None else vp,
                            table, positions, **kw)

    for bad, error in [
        (dict(kp=pool.float()), TypeError),
        (dict(vp=pool[:3]), ValueError),
        (dict(kp=pool[..., :48], key=k[..., :48]), ValueError),
        (dict(kp=pool[:, :, :8]), ValueError),
        (dict(layout="NHD"), ValueError),
        (dict(layout="DHN"), ValueError),
        (dict(kp=pool.transpose(2, 3)), ValueError),
        (dict(key=k[:, :1]), ValueError),
        (dict(value=k.bfloat16()), TypeError),
        (dict(key=k.half()), TypeError),
        (dict(key=k.cpu()), ValueError),
        (dict(table=pt.long()), TypeError),
        (dict(table=pt.cpu()), ValueError),
        (dict(table=pt.t()), ValueError),
        (dict(table=pt[:1]), ValueError),  # two tokens, one sequence, no ids
        (dict(positions=at[:1]), ValueError),
        (dict(positions=at.float()), TypeError),
        (dict(sequence_ids=at.long()), TypeError),
        (dict(sequence_ids=at[:1]), ValueError),
        (dict(query=k.bfloat16()), TypeError),
        (dict(query=k[:1]), ValueError),
        (dict(cos_sin=torch.zeros(4, 66, device=DEV)), ValueError),
        (dict(cos_sin=torch.zeros(4, 64, device=DEV, dtype=torch.float64)), TypeError),
    ]:
        with pytest.raises(error):
            call(**bad)
