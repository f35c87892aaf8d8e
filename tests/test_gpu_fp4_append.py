"""Appending to a page pool of 4 bits and reading rows back (needs a B200).

Everything is exact: rows that are not rotated are their definition's codes in 64
bits (ties included: bf16 rows meet them often); rotated rows are those of the
fp32 rotation that ``apply_rotary`` writes, which has its own tests.
"""

import pytest
import torch

import fp4_helpers as fp4
from refinekv_b200 import apply_rotary, fp4_pool, paged_append, paged_read, rotary_table
from refinekv_b200.attention import device_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


def _pool(pages, heads, block, dim, spare=0):
    """A pool of sentinel bytes, cut out of a wider tensor when `spare`."""
    whole = torch.full((pages, heads + spare, block, dim * 9 // 16), 0xA5, device=DEV,
                       dtype=torch.uint8)
    return whole[:, :heads]


def _expect(pool, rows, at, table, ids, factor=None):
    """The pool with the rows written as the definition says."""
    want = pool.clone().contiguous()
    block = pool.shape[2]
    codes, scales = fp4.parts(want)
    rows = rows.float()
    if factor is not None:
        rows = rows / factor[:, None]
    new = fp4.quantise(rows)
    page, row = table[ids.long(), at.long() // block].long(), at.long() % block
    for part, x in zip((codes, scales), new):
        part.transpose(1, 2)[page, row] = x
    return want


CASES = [
    # lengths, chunk, q heads, KV heads, dim, rotary, block
    ([1, 40, 333], 1, 32, 8, 128, 128, 32),
    ([70, 5, 16, 17], 0, 7, 1, 64, 32, 16),
    ([129], 50, 4, 2, 96, 96, 64),
    ([129], 50, 12, 4, 96, 48, 16),   # half of the rotary width is 24: three pieces
    ([64, 65], 64, 0, 3, 256, 64, 64),
    ([31, 2], 2, 5, 5, 32, 20, 32),   # 10 pairs: no whole pieces
    ([31, 2], 2, 5, 5, 32, 0, 16),    # not rotated
    ([700, 3], 0, 3, 2, 160, 160, 16),
    ([1], 1, 64, 32, 224, 224, 64),
]


@pytest.mark.parametrize("lengths,chunk,hq,hk,dim,rotary,block", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaled", [False, True])
def test_appended_codes_are_the_definitions(lengths, chunk, hq, hk, dim, rotary, block, dtype,
                                            interleaved, scaled):
    gen = torch.Generator(device=DEV).manual_seed(dim + block)
    n, blocks = len(lengths), -(-max(lengths) // block)
    pages = n * blocks + 2
    pt = torch.randperm(pages, generator=gen, device=DEV)[: n * blocks].view(n, blocks).int()
    kp, vp = _pool(pages, hk, block, dim), _pool(pages, hk, block, dim, spare=1)
    new = [min(L, chunk or L) for L in lengths]
    at = torch.cat([torch.arange(L - m, L) for L, m in zip(lengths, new)])
    ids = torch.repeat_interleave(torch.arange(n), torch.tensor(new))
    shuffle = torch.randperm(len(at))  # tokens in any order
    at, ids = at[shuffle].to(DEV, torch.int32), ids[shuffle].to(DEV, torch.int32)
    both = _normal(gen, len(at), hq + 2 * hk, dim, dtype=dtype)
    both *= torch.exp2(torch.randint(-6, 7, (len(at), 1, 1), generator=gen, device=DEV))
    q, k, v = both[:, :hq], both[:, hq:hq + hk], both[:, hq + hk:]
    factors = {}
    if scaled:
        factors = {name: 0.1 + torch.rand(hk, generator=gen, device=DEV)
                   for name in ("key_scale", "value_scale")}
    cs = rotary_table(rotary, max(lengths)) if rotary else None
    turned_q, turned_k = q, k.float()
    if rotary:
        turned_q = apply_rotary(q, None, at, cs, interleaved=interleaved)[0] if hq else q
        turned_k = apply_rotary(k.float(), None, at, cs, interleaved=interleaved)[0]
    want_k = _expect(kp, turned_k, at, pt, ids, factors.get("key_scale"))
    want_v = _expect(vp, v, at, pt, ids, factors.get("value_scale"))
    ws = {}
    out = paged_append(k, v, kp, vp, pt, at, sequence_ids=ids, query=q if hq else None, cos_sin=cs,
                       interleaved=interleaved, workspace=ws, **factors)
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    if hq:
        assert out.dtype == dtype and torch.equal(out, turned_q)
    # and back
    for row_type in (torch.float32, torch.bfloat16):
        rows = paged_read(kp, vp, pt, at, sequence_ids=ids, dtype=row_type, workspace=ws, **factors)
        for pool, got, name in zip((want_k, want_v), rows, ("key_scale", "value_scale")):
            page, row = pt[ids.long(), at.long() // block].long(), at.long() % block
            x = fp4.values(*(part.transpose(1, 2)[page, row] for part in fp4.parts(pool))).float()
            if scaled:
                x = x * factors[name][:, None]
            assert got.dtype == row_type and torch.equal(got, x.to(row_type))
    assert device_status(ws) == 0


def test_rows_of_views_and_of_odd_addresses():
    gen = torch.Generator(device=DEV).manual_seed(3)
    kp, vp = fp4_pool(3, 2, 16, 64), fp4_pool(3, 2, 16, 64)
    pt = torch.tensor([[2, 0]], device=DEV, dtype=torch.int32)
    at = torch.arange(20, device=DEV)  # int64
    ids = torch.zeros(20, device=DEV, dtype=torch.int32)
    cs = rotary_table(64, 20)
    flat = _normal(gen, 20 * 4 * 64 + 1)
    odd = flat[1:].view(20, 4, 64)           # rows that start 2 bytes off
    wide = _normal(gen, 64, 4, 20).permute(2, 1, 0)  # rows that are not contiguous
    for both in (odd, wide):
        k, v = both[:, :2], both[:, 2:]
        turned = apply_rotary(k.float().contiguous(), None, at, cs)[0]
        want_k, want_v = _expect(kp, turned, at, pt, ids), _expect(vp, v, at, pt, ids)
        q = both[:, 1:]
        out = paged_append(k, v, kp, vp, pt, at, sequence_ids=ids, query=q, cos_sin=cs)
        assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
        assert torch.equal(out, apply_rotary(q.contiguous(), None, at, cs)[0])


def test_extreme_blocks():
    inf, nan = float("inf"), float("nan")
    rows = torch.zeros(8, 1, 32, device=DEV)
    rows[0, 0, :16] = torch.tensor([6, 5, 3.5, 2.5, 1.75, 1.25, .75, .25] * 2)  # every tie, scale 1
    rows[0, 0, 16:] = -rows[0, 0, :16]
    rows[1, 0, 3], rows[1, 0, 20] = inf, -inf
    rows[2, 0, 5] = nan
    rows[3, 0, :16] = 2.0 ** -10 * 5.9   # below half of the smallest scale's reach
    rows[3, 0, 16:] = -(2.0 ** -9) * 6   # the smallest scale
    rows[4, 0, :16] = 1e30               # cut off at 2688
    rows[4, 0, 16:] = torch.linspace(-3000, 3000, 16)
    rows[5, 0, :] = -0.0
    rows[6, 0, :16] = torch.finfo(torch.float32).tiny
    rows[7, 0, 0] = 1e-3
    kp, vp = fp4_pool(1, 1, 16, 32), fp4_pool(1, 1, 16, 32)
    pt = torch.zeros(1, 1, device=DEV, dtype=torch.int32)
    at = torch.arange(8, device=DEV, dtype=torch.int32)
    ids = torch.zeros_like(at)
    want = _expect(kp, rows, at, pt, ids)
    paged_append(rows, rows, kp, vp, pt, at, sequence_ids=ids)
    assert torch.equal(kp, want) and torch.equal(vp, want)
    keys, _ = paged_read(kp, vp, pt, at, sequence_ids=ids, dtype=torch.float32)
    assert bool(keys[1].isnan().all()) and bool(keys[2, 0, :16].isnan().all())
    assert not bool(keys[2, 0, 16:].any()) and not bool(keys[3, 0, :16].any())
    assert bool((keys[3, 0, 16:] == -(2.0 ** -9) * 6).all())
    assert bool((keys[4, 0, :16] == 2688).all()) and float(keys[4, 0, 16:].abs().max()) == 2688
    assert not bool(keys[5:7].any())


def test_padding_and_tokens_out_of_range():
    gen = torch.Generator(device=DEV).manual_seed(5)
    kp, vp = _pool(4, 2, 16, 64), _pool(4, 2, 16, 64)
    pt = torch.tensor([[1, 9], [3, 0], [-1, 2]], device=DEV, dtype=torch.int32)
    cs = rotary_table(64, 30)
    q, k, v = (_normal(gen, 7, 2, 64) for _ in "qkv")
    #       padding  good  past the table's row  rotation table's end  bad page  bad page  bad sequence
    at = torch.tensor([-1, 3, 32, 31, 16, 0, 5], device=DEV, dtype=torch.int32)
    ids = torch.tensor([0, 1, 1, 1, 0, 2, 3], device=DEV, dtype=torch.int32)
    good = [1]
    turned = apply_rotary(k[good].float(), None, at[good], cs)[0]
    want_k, want_v = (_expect(p, x, at[good], pt, ids[good]) for p, x in ((kp, turned), (vp, v[good])))
    ws = {}
    out = paged_append(k, v, kp, vp, pt, at, sequence_ids=ids, query=q, cos_sin=cs, workspace=ws)
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    assert device_status(ws) == 2
    assert not bool(out[0].any()) and bool(out[2].isnan().all()) and bool(out[3].isnan().all())
    for i in (1, 4, 5, 6):
        assert torch.equal(out[i], apply_rotary(q[i:i + 1], None, at[i:i + 1], cs)[0][0])
    ws = {}
    keys, values = paged_read(kp, vp, pt, at, sequence_ids=ids, workspace=ws)
    assert device_status(ws) == 2
    for rows in (keys, values):
        assert not bool(rows[0].any()) and bool(rows[2].isnan().all())
        assert bool(rows[4:].isnan().all()) and not bool(rows[1].isnan().any())


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_read_of_a_bf16_pool(layout):
    gen = torch.Generator(device=DEV).manual_seed(6)
    shape = (5, 3, 32, 96) if layout == "HND" else (5, 32, 3, 96)
    kp, vp = _normal(gen, *shape), _normal(gen, *shape)
    pt = torch.tensor([[4, 0], [1, 7]], device=DEV, dtype=torch.int32)
    at = torch.tensor([0, 63, 31, 5, -4, 32], device=DEV)
    ids = torch.tensor([0, 0, 1, 1, 0, 1], device=DEV, dtype=torch.int32)
    for dtype in (torch.bfloat16, torch.float32):
        rows = paged_read(kp, vp, pt, at, sequence_ids=ids, layout=layout, dtype=dtype)
        for pool, got in zip((kp, vp), rows):
            view = pool.transpose(1, 2) if layout == "HND" else pool
            assert torch.equal(got[:2], view[[4, 0], [0, 31]].to(dtype))
            assert torch.equal(got[2:4], view[[1, 1], [31, 5]].to(dtype))
            assert not bool(got[4].any()) and bool(got[5].isnan().all())


def test_a_step_without_ids_in_a_captured_graph_and_none_at_all():
    gen = torch.Generator(device=DEV).manual_seed(7)
    kp, vp = fp4_pool(8, 4, 32, 128), fp4_pool(8, 4, 32, 128)
    pt = torch.randperm(8, generator=gen, device=DEV).view(2, 4).int()
    cs = rotary_table(128, 128)
    q, k, v = _normal(gen, 2, 16, 128), _normal(gen, 2, 4, 128), _normal(gen, 2, 4, 128)
    at, ws = torch.tensor([0, 70], device=DEV, dtype=torch.int32), {}
    out = paged_append(k, v, kp, vp, pt, at, query=q, cos_sin=cs, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_append(k, v, kp, vp, pt, at, query=q, cos_sin=cs, workspace=ws)
        keys, values = paged_read(kp, vp, pt, at)
    for step in range(3):
        at += 13
        for x in (q, k, v):
            x.copy_(_normal(gen, *x.shape))
        ids = torch.arange(2, device=DEV)
        want = _expect(kp, apply_rotary(k.float(), None, at, cs)[0], at, pt, ids)
        graph.replay()
        assert torch.equal(kp, want)
        assert torch.equal(out, apply_rotary(q, None, at, cs)[0])
        assert torch.equal(values.double(), fp4.values(*fp4.quantise(v.float())))
    none = torch.empty(0, device=DEV, dtype=torch.int32)
    assert paged_append(k[:0], v[:0], kp, vp, pt, none) is None
    assert paged_read(kp, vp, pt, none)[0].shape == (0, 4, 128)
    assert torch.equal(kp, want)


def test_the_returned_query_may_be_the_next_query():
    gen = torch.Generator(device=DEV).manual_seed(8)
    kp, vp = fp4_pool(8, 4, 32, 128), fp4_pool(8, 4, 32, 128)
    pt = torch.arange(8, device=DEV).view(2, 4).int()
    cs, ws = rotary_table(128, 128), {}
    q, k = _normal(gen, 2, 16, 128), _normal(gen, 2, 4, 128)
    at = torch.tensor([99, 70], device=DEV, dtype=torch.int32)
    once = paged_append(k, k, kp, vp, pt, at, query=q, cos_sin=cs, workspace=ws)
    want = apply_rotary(once, None, at, cs)[0]
    assert torch.equal(paged_append(k, k, kp, vp, pt, at, query=once, cos_sin=cs, workspace=ws), want)


def test_refusals():
    kp, vp = fp4_pool(4, 2, 16, 64), fp4_pool(4, 2, 16, 64)
    pt = torch.zeros(2, 2, device=DEV, dtype=torch.int32)
    k = torch.zeros(2, 2, 64, device=DEV, dtype=torch.bfloat16)
    at = torch.zeros(2, device=DEV, dtype=torch.int32)
    bf16 = torch.zeros(4, 2, 16, 64, device=DEV, dtype=torch.bfloat16)
    one = torch.ones(2, device=DEV)

    def no(error, match, *args, call=paged_append, **kw):
        with pytest.raises(error, match=match):
            call(*args, **kw)

    no(ValueError, "HND", k, k, kp, vp, pt, at, layout="NHD")
    no(TypeError, "both", k, k, kp, bf16[..., :36], pt, at)
    no(ValueError, "same 4-D shape", k, k, kp, vp[:3], pt, at)
    no(ValueError, "9 / 16", k, k, kp[..., :35], vp[..., :35], pt, at)
    no(ValueError, "9 / 16", k, k, kp[..., :9], vp[..., :9], pt, at)
    wide = torch.zeros(4, 2, 16, 72, device=DEV, dtype=torch.uint8)[..., :36]
    no(ValueError, "slab", k, k, wide, wide, pt, at)
    no(ValueError, "blocks", k, k, kp[:, :, :8], vp[:, :, :8], pt, at)
    no(ValueError, "contiguous", k, k, kp, vp, pt, at, key_scale=one[:1])
    no(ValueError, "contiguous", k, k, kp, vp, pt, at, value_scale=torch.ones(4, device=DEV)[::2])
    no(TypeError, "fp32", k, k, kp, vp, pt, at, value_scale=one.double())
    no(ValueError, "belong", k, k, bf16, bf16, pt, at, key_scale=one)
    no(ValueError, "belong", bf16, bf16, pt, at, call=paged_read, value_scale=one)
    no(TypeError, "BF16 or FP32", kp, vp, pt, at, call=paged_read, dtype=torch.float16)
    no(TypeError, "int32 or int64", kp, vp, pt, at.float(), call=paged_read)
    no(ValueError, "sequence_ids", kp, vp, pt, at.repeat(2), call=paged_read)
    flat = torch.zeros(4 * 2 * 16 * 36 + 8, device=DEV, dtype=torch.uint8)
    off = flat[8:].view(4, 2, 16, 36)
    no(ValueError, "16 bytes", k, k, off, off, pt, at)
    no(ValueError, "16 bytes", off, off, pt, at, call=paged_read)
    no(ValueError, "blocks", 1, 1, 8, 64, call=fp4_pool)
    no(ValueError, "head_dim", 1, 1, 16, 80, call=fp4_pool)
