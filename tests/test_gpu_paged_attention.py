"""Paged attention against a softmax in 64 bits (needs a B200).

Bounds, for one query row with exact weights p_j over its visible rows:
A = sum_j p_j |v_j| / sum_j p_j per channel, X = max_j scale sum_i |q_i k_ji|, u = 2^-23.
A logit adds dim / 16 tensor-core products of 16 exact terms, each rounded at
most twice: off by at most e = (dim / 8) u X, which moves each weight by e
relatively; __expf adds less than 2^-21 of the largest weight; the sums add
a tile of 32 rows at a time and then merge at most a few dozen parts, u each:
  fp32 queries:  |out - exact| <= A (2 e + 2^-20 + (rows / 32 + 32) u) + |exact| u
  bf16 queries:  weights rounded to bf16 add A 2^-8, the result half a unit
                 in its last place
  lse:           e + 2^-20 + (rows / 32 + 32) u + |lse| 2^-22.
Every row of the pool that is not visible holds NaN or infinity.
"""

import math

import pytest
import torch

from refinekv_b200 import dense_attention, page_view, paged_append, paged_attention
from refinekv_b200.attention import device_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


class Served:
    """Sequences in a pool whose every other row holds NaN or infinity, and table entries past
    the used pages hold garbage."""

    def __init__(self, lengths, hq, hk, dim, block, layout="HND", dtype=torch.bfloat16, seed=0,
                 window=None, sharp=1.0, spare=2):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.lengths, self.window, self.layout = lengths, window, layout
        n, blocks = len(lengths), max(1, -(-max(lengths) // block)) + spare
        used = [-(-L // block) for L in lengths]
        pages = sum(used) + 2
        shape = (pages, hk, block, dim) if layout == "HND" else (pages, block, hk, dim)
        self.kp = torch.full(shape, float("nan"), device=DEV, dtype=torch.bfloat16)
        self.vp = torch.full(shape, float("inf"), device=DEV, dtype=torch.bfloat16)
        kv, vv = self.views()
        order = torch.randperm(pages, generator=gen, device=DEV).int()
        self.table = torch.full((n, blocks), -7, device=DEV, dtype=torch.int32)
        self.table[:, 1::2] = 1 << 30
        self.keys, self.values, at = [], [], 0
        for i, L in enumerate(lengths):
            low = max(0, L - window) if window else 0
            self.keys.append(_normal(gen, L - low, hk, dim))
            self.values.append(_normal(gen, L - low, hk, dim))
            ids = order[at:at + used[i]]
            at += used[i]
            first = low // block  # pages before the window: garbage entries
            self.table[i, first:used[i]] = ids[first:]
            where = torch.arange(low, L, device=DEV)
            kv[ids.long()[where // block], where % block] = self.keys[-1]
            vv[ids.long()[where // block], where % block] = self.values[-1]
        self.n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
        self.q = (_normal(gen, n, hq, dim, dtype=torch.float32) * sharp).to(dtype)

    def views(self):
        if self.layout == "HND":
            return self.kp.transpose(1, 2), self.vp.transpose(1, 2)
        return self.kp, self.vp

    def call(self, **kw):
        kw = {"layout": self.layout, "window": self.window, "return_lse": True, **kw}
        return paged_attention(self.q, self.kp, self.vp, self.table, self.n, **kw)

    def check(self, out, lse, scale=None):
        hk, dim = self.views()[0].shape[2:]
        hq = self.q.shape[1]
        scale = dim ** -0.5 if scale is None else scale
        u = 2.0 ** -23
        assert out.shape == self.q.shape and out.dtype == self.q.dtype
        assert lse.shape == self.q.shape[:2] and lse.dtype == torch.float32
        for i, (k, v) in enumerate(zip(self.keys, self.values)):
            if len(k) == 0:
                assert not bool(out[i].any()) and bool((lse[i] == -math.inf).all())
                continue
            q = self.q[i].to(torch.bfloat16).double().view(hk, hq // hk, dim)
            k, v = k.double().transpose(0, 1), v.double().transpose(0, 1)
            x = q @ k.transpose(1, 2) * scale
            e = (q.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1).reshape(hq) * dim / 8 * u
            p = x.softmax(-1)
            want, size = (p @ v).reshape(hq, dim), (p @ v.abs()).reshape(hq, dim)
            want_lse = x.logsumexp(-1).reshape(hq)
            sums = 2 ** -20 + (x.shape[-1] / 32 + 32) * u
            tol = size * (2 * e + sums)[:, None] + want.abs() * u
            if out.dtype == torch.bfloat16:
                half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 1 - 8)
                tol = tol * 1.01 + size * 2 ** -8 + half + 1e-38
            off = (out[i].double() - want).abs()
            assert bool((off <= tol).all()), (i, float((off - tol).max()), float(off.max()))
            off = (lse[i].double() - want_lse).abs()
            assert bool((off <= e + sums + want_lse.abs() * 2 ** -22).all()), (i, float(off.max()))


CASES = [
    # lengths, q heads, KV heads, dim, block, layout, window
    ([1], 32, 8, 128, 32, "HND", None),
    ([333], 32, 8, 128, 32, "HND", None),
    ([31, 32, 33, 0, 1, 64, 65], 28, 4, 128, 16, "NHD", None),
    ([0, 0, 0], 4, 2, 64, 64, "HND", None),
    ([4097, 0, 17, 1000], 16, 1, 128, 64, "HND", None),
    ([5000], 2, 2, 64, 16, "HND", None),
    ([100, 2100], 9, 1, 96, 32, "NHD", None),
    ([777, 1], 32, 2, 256, 32, "HND", None),
    ([513, 48, 15], 6, 3, 32, 16, "NHD", None),
    ([1500], 8, 8, 160, 64, "NHD", None),
    ([300, 299], 12, 1, 192, 16, "HND", None),
    ([65], 10, 2, 224, 64, "HND", None),
    ([20000, 3], 8, 1, 128, 32, "HND", None),
    ([1 + 7 * (i % 41) for i in range(300)], 8, 2, 64, 16, "HND", None),
    # rows over so many CTAs that their parts are joined in groups
    ([70000, 3], 8, 1, 128, 32, "HND", None),
    ([150000], 16, 1, 64, 16, "NHD", None),
    ([66000, 68000], 4, 1, 256, 64, "HND", None),
    ([1000, 5, 64, 0, 33], 32, 8, 128, 32, "HND", 1),
    ([1000, 5, 64, 0, 33, 130], 28, 4, 128, 16, "NHD", 20),
    ([1000, 555, 64, 63], 8, 8, 64, 64, "HND", 64),
    ([9999, 4096, 4097], 16, 2, 128, 32, "NHD", 4096),
]


@pytest.mark.parametrize("lengths,hq,hk,dim,block,layout,window", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_matches_the_formula(lengths, hq, hk, dim, block, layout, window, dtype):
    s = Served(lengths, hq, hk, dim, block, layout, dtype, seed=dim + block, window=window)
    ws = {}
    out, lse = s.call(workspace=ws)
    s.check(out, lse)
    assert device_status(ws) == 0
    # a second call on the used workspace, and one without the sums, repeat the bits
    out, lse = out.clone(), lse.clone()
    again = s.call(workspace=ws)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert torch.equal(s.call(return_lse=False), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sharp_softmax_and_scale(dtype):
    s = Served([3000, 40, 1], 8, 2, 128, 32, dtype=dtype, seed=3, sharp=12.0)
    s.check(*s.call())
    s.check(*s.call(scale=0.3), scale=0.3)
    s.check(*s.call(scale=-0.05), scale=-0.05)
    s.check(*s.call(scale=0.0), scale=0.0)


def test_workspace_serves_other_shapes_and_the_results_repeat():
    ws = {}
    shapes = [([9000, 12], 32, 8, 128, 32), ([40] * 200, 4, 4, 64, 16), ([9000], 4, 1, 128, 32),
              ([3, 5000, 0], 32, 2, 256, 64)]
    first = {}
    for turn in range(2):
        for i, (lengths, *shape) in enumerate(shapes):
            s = Served(lengths, *shape, seed=i)
            out, lse = s.call(workspace=ws)
            s.check(out, lse)
            if turn:
                assert torch.equal(out, first[i])
            first[i] = out.clone()
    assert device_status(ws) == 0


def test_parts_join_by_their_sums():
    s = Served([1000], 8, 2, 128, 16, dtype=torch.float32, seed=5)
    whole, total = s.call()
    whole, total = whole.clone(), total.clone()
    cut = 400  # a whole number of pages
    head = paged_attention(s.q, s.kp, s.vp, s.table, s.n * 0 + cut, return_lse=True)
    tail = paged_attention(s.q, s.kp, s.vp, s.table[:, cut // 16:], s.n - cut, return_lse=True)
    joined = sum((lse - total).exp()[..., None] * out for out, lse in (head, tail))
    # both sides carry the fp32 bound above with e near 2^-17
    assert float((joined - whole).abs().max()) <= 2 ** -14


def test_infinities_and_nans_in_visible_rows_follow_the_formula():
    s = Served([100, 100, 100, 100, 100], 4, 1, 64, 32, dtype=torch.float32, seed=6)
    s.q[:] = s.q.abs() + 0.5
    kv, vv = s.views()
    put = lambda view, i, j, x: view.__setitem__((int(s.table[i, j // 32]), j % 32), x)  # noqa: E731
    put(kv, 0, 70, float("nan"))   # a NaN logit: the whole row is NaN
    put(kv, 1, 70, float("-inf"))  # a logit of -inf: that row weighs nothing
    put(vv, 2, 33, float("inf"))   # an infinite value: infinite results
    for j in range(100):
        put(kv, 3, j, float("-inf"))  # every logit -inf: 0 / 0, as the softmax has it
    put(kv, 4, 2, float("inf"))    # a logit of +inf: inf - inf
    out, lse = s.call()
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    keep = torch.arange(100, device=DEV) != 70
    s.keys, s.values = [s.keys[1][keep]], [s.values[1][keep]]
    s.q, s.lengths = s.q[1:2], [99]
    s.check(out[1:2], lse[1:2])
    assert bool((out[2] == float("inf")).all())
    assert bool(out[3].isnan().all()) and bool((lse[3] == -math.inf).all())
    assert bool(out[4].isnan().all())


def test_strides_and_alignments():
    s = Served([70, 33], 8, 2, 64, 32, "NHD", seed=7)
    want = s.call()[0].clone()
    fused = torch.zeros(2, 12, 64, device=DEV, dtype=torch.bfloat16)
    fused[:, 2:10] = s.q
    assert torch.equal(paged_attention(fused[:, 2:10], s.kp, s.vp, s.table, s.n, layout="NHD"), want)
    odd = torch.zeros(2, 8, 65, device=DEV, dtype=torch.bfloat16)
    odd[..., 1:] = s.q
    assert torch.equal(paged_attention(odd[..., 1:], s.kp, s.vp, s.table, s.n, layout="NHD"), want)
    skew = s.q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(paged_attention(skew, s.kp, s.vp, s.table, s.n, layout="NHD"), want)
    both = torch.stack([s.kp, s.vp], 1)  # pools cut out of one tensor
    assert torch.equal(paged_attention(s.q, both[:, 0], both[:, 1], s.table, s.n, layout="NHD"),
                       want)
    hnd = [x.transpose(1, 2).contiguous() for x in (s.kp, s.vp)]
    assert torch.equal(paged_attention(s.q, *hnd, s.table, s.n), want)
    wide = torch.full((2, 9), -1, device=DEV, dtype=torch.int32)
    wide[:, 1:1 + s.table.shape[1]] = s.table
    lengths = torch.stack([s.n, s.n], 1)[:, 0]
    assert torch.equal(paged_attention(s.q, s.kp, s.vp, wide[:, 1:1 + s.table.shape[1]], lengths,
                                       layout="NHD"), want)
    one = paged_attention(s.q[:1], s.kp, s.vp, s.table[0], s.n[:1], layout="NHD")
    assert torch.equal(one, paged_attention(s.q[:1], s.kp, s.vp, s.table[:1], s.n[:1],
                                            layout="NHD"))


def test_bad_lengths_and_pages_are_flagged():
    s = Served([40, 40], 4, 2, 64, 32, seed=8, spare=0)
    ws = {}
    s.n.copy_(torch.tensor([40, 65]))  # two pages of 32 hold 64
    out, lse = s.call(workspace=ws)
    assert device_status(ws) == 2
    good = Served([40, 40], 4, 2, 64, 32, seed=8, spare=0)
    want = good.call()[0]
    assert torch.equal(out[0], want[0])
    ws = {}
    s.n.copy_(torch.tensor([40, -1]))
    out, lse = s.call(workspace=ws)
    assert device_status(ws) == 2 and torch.equal(out[0], want[0]) and not bool(out[1].any())
    for bad in (-1, s.kp.shape[0]):
        ws = {}
        s.n.copy_(torch.tensor([40, 40]))
        s.table[1, 1] = bad
        out, _ = s.call(workspace=ws)
        assert device_status(ws) == 2 and torch.equal(out[0], want[0])


def test_offsets_past_32_bits():
    pages, heads, block, dim = 33000, 8, 64, 128  # 2.16e9 elements a pool
    gen = torch.Generator(device=DEV).manual_seed(9)
    kp = torch.empty(pages, heads, block, dim, device=DEV, dtype=torch.bfloat16)
    vp = torch.empty_like(kp)
    keys, values = _normal(gen, 2, heads, block, dim), _normal(gen, 2, heads, block, dim)
    for i, page in enumerate((pages - 1, pages - 3)):
        kp[page], vp[page] = keys[i], values[i]
    table = torch.tensor([[pages - 1, pages - 3]], device=DEV, dtype=torch.int32)
    n = torch.tensor([100], device=DEV, dtype=torch.int32)
    q = _normal(gen, 1, 32, dim)
    got = paged_attention(q, kp, vp, table, n)
    small = torch.tensor([[0, 1]], device=DEV, dtype=torch.int32)
    assert torch.equal(got, paged_attention(q, keys, values, small, n))


def test_agrees_with_dense_attention_over_one_cache():
    gen = torch.Generator(device=DEV).manual_seed(10)
    heads, group, dim, tokens, suffix = 8, 4, 128, 2048, 33
    kc, vc = _normal(gen, heads, 2112, dim), _normal(gen, heads, 2112, dim)
    q = _normal(gen, heads, group, 1, dim)
    want = dense_attention(q, page_view(kc, vc, tokens), kc[:, tokens:tokens + suffix],
                           vc[:, tokens:tokens + suffix])
    pages = [c.view(heads, 66, 32, dim).transpose(0, 1) for c in (kc, vc)]  # strided pool views
    got = paged_attention(q.view(1, heads * group, dim), *pages,
                          torch.arange(66, device=DEV, dtype=torch.int32)[None],
                          torch.tensor([tokens + suffix], device=DEV, dtype=torch.int32))
    # each side within A 2^-8 and half a bf16 unit of the softmax, A below 1 and outputs below 0.25
    assert float((got.view_as(want).float() - want.float()).abs().max()) <= 2 * (2 ** -8 + 2 ** -11)


def test_graph_replay_follows_growing_sequences():
    s = Served([500, 70, 0], 8, 2, 64, 16, seed=11, spare=4)
    kv, vv = s.views()
    ws = {}
    s.call(workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = s.call(workspace=ws)
    gen = torch.Generator(device=DEV).manual_seed(12)
    for lengths in ([500, 70, 0], [501, 71, 0], [3, 0, 0]):
        for i, L in enumerate(lengths):
            if L > len(s.keys[i]):
                k, v = _normal(gen, 1, 2, 64), _normal(gen, 1, 2, 64)
                page = int(s.table[i, (L - 1) // 16])
                assert 0 <= page < s.kp.shape[0]  # 500 and 70 end inside a page
                kv[page, (L - 1) % 16], vv[page, (L - 1) % 16] = k[0], v[0]
                s.keys[i], s.values[i] = torch.cat([s.keys[i], k]), torch.cat([s.values[i], v])
            s.keys[i], s.values[i] = s.keys[i][:L], s.values[i][:L]
        s.n.copy_(torch.tensor(lengths))
        graph.replay()
        s.check(out, lse)


def test_other_stream_after_an_append():
    s = Served([64, 20], 8, 2, 64, 16, seed=13, spare=1)
    pages = s.kp.shape[0]
    spare = sorted(set(range(pages)) - set(s.table[s.table >= 0].unique().tolist()))
    s.table[0, 4] = spare[0]
    gen = torch.Generator(device=DEV).manual_seed(14)
    k, v = _normal(gen, 2, 2, 64), _normal(gen, 2, 2, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ws = {}
        paged_append(k, v, s.kp, s.vp, s.table, s.n, workspace=ws)
        s.n += 1
        out, lse = s.call(workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(2):
        s.keys[i] = torch.cat([s.keys[i], k[i:i + 1]])
        s.values[i] = torch.cat([s.values[i], v[i:i + 1]])
    s.check(out, lse)
    assert device_status(ws) == 0


@pytest.mark.parametrize("dim,hq,hk", [(192, 16, 1), (128, 2, 2)])
def test_as_many_sequences_as_the_kernel_takes(dim, hq, hk):
    lengths = [(7 * i) % 5 for i in range(4095)] + [900]
    s = Served(lengths, hq, hk, dim, 16, seed=dim)
    out, lse = s.call()
    some = [0, 1, 2, 3, 4, 2047, 4094, 4095]
    for i in some:
        one = paged_attention(s.q[i:i + 1], s.kp, s.vp, s.table[i:i + 1], s.n[i:i + 1],
                              return_lse=True)
        part = Served.__new__(Served)
        part.__dict__.update(s.__dict__)
        part.keys, part.values, part.q = s.keys[i:i + 1], s.values[i:i + 1], s.q[i:i + 1]
        part.check(*one)
        part.check(out[i:i + 1], lse[i:i + 1])
    empty = s.n == 0
    assert not bool(out[empty].any()) and bool((lse[empty] == -math.inf).all())
    assert bool(out[~empty].isfinite().all())
    more = torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="4096 sequences"):
        paged_attention(torch.cat([s.q, s.q[:1]]), s.kp, s.vp, torch.cat([s.table, s.table[:1]]),
                        torch.cat([s.n, more]))


def test_no_sequences():
    s = Served([5], 4, 2, 64, 16)
    out, lse = paged_attention(s.q[:0], s.kp, s.vp, s.table[:0], s.n[:0], return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_refusals():
    s = Served([5, 6], 4, 2, 64, 16)

    def call(q=s.q, kp=s.kp, vp=s.vp, table=s.table, n=s.n, **kw):
        return paged_attention(q, kp, vp, table, n, **kw)

    for bad, error in [
        (dict(q=s.q.half()), TypeError),
        (dict(q=s.q[:1]), ValueError),
        (dict(q=s.q[:, :3]), ValueError),
        (dict(q=s.q[..., :32]), ValueError),
        (dict(q=s.q.repeat(1, 9, 1)), ValueError),  # 18 query heads a KV head
        (dict(q=s.q.cpu()), ValueError),
        (dict(kp=s.kp.float()), TypeError),
        (dict(kp=s.kp.cpu(), vp=s.vp.cpu()), RuntimeError),
        (dict(vp=s.vp[:1]), ValueError),
        (dict(layout="NHD"), ValueError),
        (dict(layout="nhd"), ValueError),
        (dict(kp=s.kp.transpose(2, 3), vp=s.vp.transpose(2, 3)), ValueError),
        (dict(kp=s.kp[:, :, :8], vp=s.vp[:, :, :8]), ValueError),
        (dict(table=s.table.long()), TypeError),
        (dict(table=s.table.cpu()), ValueError),
        (dict(table=s.table[0]), ValueError),
        (dict(n=s.n.long()), TypeError),
        (dict(n=s.n[:1]), ValueError),
        (dict(n=s.n.cpu()), ValueError),
        (dict(window=0), ValueError),
    ]:
        with pytest.raises(error):
            call(**bad)
    skewed = torch.zeros(3 * 2 * 16 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(3, 2, 16, 64)
    with pytest.raises(ValueError, match="aligned"):
        call(kp=skewed, vp=skewed)
