"""Attention over a page pool with a cap, a bias, a prefix, weights' sums, and over 4 bits, against
the formula in 64 bits (needs a B200).

Bounds, for one query row with exact weights p_j over its visible rows (as in
test_gpu_paged_attention.py): A = sum_j p_j |v_j| per channel, X = max_j scale sum_i |q_i
k_ji|, u = 2^-23.  A product q.k adds dim / 16 tensor-core products of 16 exact terms,
each rounded at most twice: it is off by at most (dim / 8) u X, and by 3 u X for the
factors it is multiplied by.  A cap c divides, takes a tanh (2 ulp) and multiplies: at most 4
u |x| more, |x| <= c, and its slope is at most 1, so that the product's error does not grow.  A
bias adds its own rounding and the sum's, u (|slope| L + |x|).  Together e; a weight
moves by e relatively, and by 2^-20 for its exponential; the sums add a tile of 32 or 64 rows
at a time and then merge at most a few dozen parts, u each:
  fp32 queries:  |out - exact| <= A (2 e + 2^-20 + (rows / 32 + 32) u) + |exact| 2 u
  bf16 queries:  weights rounded add A 2^-8 (bf16 terms) at most, the result half a unit in its
                 last place
  lse:           e + 2^-20 + (rows / 32 + 32) u + |lse| 2^-22
  weights:       sum over the group of p (e + the lse's error + 2^-20) + (group + 1) u (W + sum).
For 4 bits the weights' fp16 terms (11 significant bits: half a step is 2^-11 of the value) are off
by 2^-11 (bf16 queries) or 2^-22 (fp32) of the weight, and at least 2^-40 of the greatest: rows
2^-40 A' more, A' = sum |v_j| / sum e^(x_j - max), far below.
Every row of the pool that is not visible holds NaN.
"""

import math

import pytest
import torch

import fp4_helpers as fp4
from refinekv_b200 import fp4_pool, paged_attention
from refinekv_b200.attention import device_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


class Served:
    """Sequences in a pool whose other rows hold NaN; table entries of pages that are not used
    hold garbage."""

    def __init__(self, lengths, hq, hk, dim, block, layout="HND", bits=16, dtype=torch.bfloat16,
                 window=None, prefix=0, softcap=None, slopes=False, weights=False, scaled=False,
                 seed=0, sharp=1.0, spare=2):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.lengths, self.hk, self.dim, self.bits = lengths, hk, dim, bits
        n, blocks = len(lengths), max(1, -(-max(lengths) // block)) + spare
        used = [-(-L // block) for L in lengths]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=gen, device=DEV).int()
        self.table = torch.full((n, blocks), -7, device=DEV, dtype=torch.int32)
        self.table[:, 1::2] = 1 << 30
        if bits == 4:
            self.kp, self.vp = fp4_pool(pages, hk, block, dim), fp4_pool(pages, hk, block, dim)
            for pool in (self.kp, self.vp):
                fp4.parts(pool)[0].random_(0, 256, generator=gen)
                fp4.parts(pool)[1].fill_(fp4.NAN_SCALE)
        else:
            shape = (pages, hk, block, dim) if layout == "HND" else (pages, block, hk, dim)
            self.kp, self.vp = (torch.full(shape, math.nan, device=DEV, dtype=torch.bfloat16)
                                for _ in "kv")
        self.args = dict(layout=layout, window=window, prefix=prefix, softcap=softcap)
        factor = [torch.ones(hk, device=DEV)] * 2
        if scaled:
            factor = [0.2 + torch.rand(hk, generator=gen, device=DEV) for _ in "kv"]
            self.args.update(key_scale=factor[0], value_scale=factor[1])
        self.rows, self.at, at = [], [], 0
        for i, L in enumerate(lengths):
            seen = torch.arange(L, device=DEV)
            if window is not None:
                seen = seen[(seen >= L - window) | (seen < prefix)]
            ids = order[at:at + used[i]]
            at += used[i]
            need = torch.unique(seen // block)
            self.table[i, need] = ids[need]
            page, row = ids.long()[seen // block], seen % block
            both = []
            for pool, by in zip((self.kp, self.vp), factor):
                x = _normal(gen, len(seen), hk, dim)
                if bits == 4:
                    held = fp4.quantise(x.float())
                    for part, new in zip(fp4.parts(pool), held):
                        part.transpose(1, 2)[page, row] = new
                    x = fp4.values(*held) * by.double()[:, None]
                elif layout == "HND":
                    pool.transpose(1, 2)[page, row] = x
                else:
                    pool[page, row] = x
                both.append(x.double())
            self.rows.append(both)
            self.at.append(seen)
        self.n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
        self.q = (_normal(gen, n, hq, dim, dtype=torch.float32) * sharp).to(dtype)
        if slopes:
            self.args["slopes"] = -torch.rand(hq, generator=gen, device=DEV) / 16
        self.before = None
        if weights:
            self.before = torch.rand(n, hk, blocks * block + 3, generator=gen, device=DEV)
            self.args["weights"] = self.before.clone()

    def call(self, **kw):
        return paged_attention(self.q, self.kp, self.vp, self.table, self.n,
                               **{"return_lse": True, **self.args, **kw})

    def check(self, out, lse, scale=None):
        hq, hk, dim = self.q.shape[1], self.hk, self.dim
        scale = dim ** -0.5 if scale is None else scale
        u, cap, slopes = 2.0 ** -23, self.args["softcap"], self.args.get("slopes")
        assert out.shape == self.q.shape and out.dtype == self.q.dtype
        assert lse.shape == self.q.shape[:2] and lse.dtype == torch.float32
        got_weights = self.args.get("weights")
        rest = None if got_weights is None else got_weights - self.before
        for i, ((k, v), L, seen) in enumerate(zip(self.rows, self.lengths, self.at)):
            if len(k) == 0:
                assert not bool(out[i].any()) and bool((lse[i] == -math.inf).all())
                assert rest is None or not bool(rest[i].any())
                continue
            q = self.q[i].to(torch.bfloat16).double().view(hk, hq // hk, dim)
            k, v = k.transpose(0, 1), v.transpose(0, 1)
            x = q @ k.transpose(1, 2) * scale
            top = (q.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1)
            e = (dim / 8 + 3) * u * top
            if cap:
                x = cap * torch.tanh(x / cap)
                e = e + 4 * u * x.abs().amax(-1)
            if slopes is not None:
                bias = slopes.double().view(hk, -1, 1) * (seen - (L - 1))
                e = e + u * (bias.abs().amax(-1) + (x + bias).abs().amax(-1))
                x = x + bias
            p = x.softmax(-1)
            want, size = (p @ v).reshape(hq, dim), (p @ v.abs()).reshape(hq, dim)
            want_lse = x.logsumexp(-1)
            sums = 2 ** -20 + (x.shape[-1] / 32 + 32) * u
            flat = e.reshape(hq)
            tol = size * (2 * flat + sums)[:, None] + want.abs() * 2 * u + 1e-30
            if self.bits == 4:  # the fp16 terms
                tail = v.abs().sum(1, keepdim=True) / (x - x.amax(-1, keepdim=True)).exp().sum(
                    -1, keepdim=True)
                tol = tol + size * 2 ** -21 + (tail * 2 ** -40).reshape(hq, dim)
            if out.dtype == torch.bfloat16:
                half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 1 - 8)
                term = 2 ** -11 if self.bits == 4 else 2 ** -8
                tol = tol * 1.01 + size * term + half + 1e-38
            off = (out[i].double() - want).abs()
            assert bool((off <= tol).all()), (i, float((off - tol).max()), float(off.max()))
            off = (lse[i].double().view(hk, -1) - want_lse).abs()
            lse_tol = e + sums + want_lse.abs() * 2 ** -22
            assert bool((off <= lse_tol).all()), (i, float(off.max()))
            if rest is not None:
                added = p.sum(1)
                tol = ((p * (e + lse_tol + 2 ** -20)[..., None]).sum(1)
                       + (hq // hk + 1) * u * (self.before[i][:, seen].double() + added))
                off = (got_weights[i][:, seen].double() - self.before[i][:, seen].double() - added)
                assert bool((off.abs() <= tol).all()), (i, float((off.abs() - tol).max()))
                hidden = torch.ones(rest.shape[2], device=DEV, dtype=torch.bool)
                hidden[seen] = False
                assert not bool(rest[i][:, hidden].any())


LENGTHS = [
    # lengths, q heads, KV heads, dim, block, layout of a bf16 pool
    ([1], 32, 8, 128, 32, "HND"),
    ([333], 32, 8, 128, 32, "NHD"),
    ([31, 32, 33, 0, 1, 64, 65], 28, 4, 128, 16, "NHD"),
    ([0, 0, 0], 4, 2, 64, 64, "HND"),
    ([4097, 0, 17, 1000], 16, 1, 128, 64, "HND"),
    ([100, 2100], 9, 1, 96, 32, "NHD"),
    ([777, 1], 32, 2, 256, 32, "HND"),
    ([513, 48, 15], 6, 3, 32, 16, "NHD"),
    ([1500, 63], 8, 8, 160, 64, "NHD"),
    ([300, 299], 12, 1, 192, 16, "HND"),
    ([65, 1030], 10, 2, 224, 64, "HND"),
    ([20000, 3], 8, 1, 128, 32, "HND"),
    ([1 + 7 * (i % 41) for i in range(300)], 8, 2, 64, 16, "HND"),
    ([70000, 3], 8, 1, 128, 32, "HND"),  # parts joined in groups
    ([40000, 900], 16, 1, 32, 16, "HND"),
]
FORMS = [
    dict(softcap=30.0),
    dict(softcap=0.5, weights=True),
    dict(slopes=True),
    dict(window=40, prefix=4),
    dict(window=700, prefix=333, slopes=True, softcap=5.0, weights=True),
    dict(window=1, prefix=1, weights=True),
    dict(prefix=7),  # without a window everything is visible
    dict(weights=True),
]


@pytest.mark.parametrize("lengths,hq,hk,dim,block,layout", LENGTHS)
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bf16_pools_match_the_formula(lengths, hq, hk, dim, block, layout, form, dtype):
    s = Served(lengths, hq, hk, dim, block, layout, dtype=dtype, seed=dim + form, **FORMS[form])
    ws = {}
    out, lse = s.call(workspace=ws)
    s.check(out, lse)
    assert device_status(ws) == 0
    out, lse = out.clone(), lse.clone()
    again = s.call(workspace=ws)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert torch.equal(s.call(return_lse=False), out)


@pytest.mark.parametrize("lengths,hq,hk,dim,block,layout", LENGTHS)
@pytest.mark.parametrize("form", [None, 1, 4, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pools_of_4_bits_match_the_formula(lengths, hq, hk, dim, block, layout, form, dtype):
    more = {} if form is None else FORMS[form]
    s = Served(lengths, hq, hk, dim, block, bits=4, dtype=dtype, seed=dim, scaled=form != 4, **more)
    ws = {}
    out, lse = s.call(workspace=ws)
    s.check(out, lse)
    assert device_status(ws) == 0
    out, lse = out.clone(), lse.clone()
    again = s.call(workspace=ws)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert torch.equal(s.call(return_lse=False), out)


@pytest.mark.parametrize("dim", range(32, 257, 32))
@pytest.mark.parametrize("group", [1, 5, 8, 9, 16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_head_dim_and_group_over_4_bits(dim, group, dtype):
    """Every instance, with pages that are a quarter, a half and the whole of a tile."""
    for block in (16, 32, 64):
        s = Served([1000, 1, 64, 0, 129], 2 * group, 2, dim, block, bits=4, dtype=dtype,
                   seed=dim + group, scaled=True, weights=block == 32)
        s.check(*s.call())


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sharp_softmax_scale_and_small_queries(bits, dtype):
    for sharp, scale in ((12.0, None), (12.0, -0.05), (1.0, 0.0), (2.0 ** -60, 2.0 ** 57),
                         (2.0 ** 40, 2.0 ** -43), (2.0 ** -130, 1.0)):
        s = Served([3000, 40, 1], 8, 2, 128, 32, bits=bits, dtype=dtype, seed=3, sharp=sharp,
                   softcap=20.0 if scale is None else None, weights=True)
        s.check(*s.call(scale=scale), scale=scale)


def test_queries_with_channels_of_very_different_size():
    """2^20 between a query's channels: the small ones still count where the keys are zero
    elsewhere."""
    s = Served([64], 4, 1, 64, 16, bits=4, dtype=torch.float32, seed=4)
    s.q[:, :, :32] *= 2.0 ** 20
    codes, scales = fp4.parts(s.kp)
    codes[..., :16] = 0
    k, v = s.rows[0]
    k[..., :32] = 0
    s.check(*s.call())


def test_a_cap_without_effect_and_no_cap_agree():
    s = Served([500, 77], 8, 2, 128, 32, dtype=torch.float32, seed=5, softcap=1e30)
    plain = paged_attention(s.q, s.kp, s.vp, s.table, s.n, return_lse=True)
    for a, b in zip(s.call(), plain):
        # c tanh(x / c) with x / c far below 1 is x but for three roundings
        assert float((a - b).abs().max()) <= 2 ** -18


def test_infinities_and_nans_follow_the_formula():
    s = Served([100, 100, 100, 100], 4, 1, 64, 32, dtype=torch.float32, seed=6, softcap=10.0,
               weights=True)
    s.q[:] = s.q.abs() + 0.5
    put = lambda pool, i, j, x: pool.transpose(1, 2).__setitem__(  # noqa: E731
        (int(s.table[i, j // 32]), j % 32), x)
    put(s.kp, 0, 70, math.nan)   # a NaN logit: the whole row is NaN
    put(s.kp, 1, 70, -math.inf)  # capped: -10
    put(s.kp, 2, 70, math.inf)   # capped: 10
    put(s.vp, 3, 33, math.inf)   # an infinite value
    out, lse = s.call()
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    assert torch.equal(s.args["weights"][0], s.before[0])  # adds nothing
    for i, x in ((1, -10.0), (2, 10.0)):
        assert bool(out[i].isfinite().all()) and bool(lse[i].isfinite().all())
        gain = (s.args["weights"] - s.before)[i, 0, 70]
        want = float((x - lse[i].double()).exp().sum())
        assert abs(float(gain) - want) <= 2 ** -20 * (1 + want)
    assert bool((out[3] == math.inf).all())


def test_nan_blocks_of_4_bits_make_their_rows_nan():
    s = Served([100, 100, 100], 4, 1, 64, 32, bits=4, dtype=torch.float32, seed=7, weights=True)
    page = int(s.table[0, 1])
    fp4.parts(s.kp)[1][page, 0, 3, 2] = fp4.NAN_SCALE
    page = int(s.table[1, 1])
    fp4.parts(s.vp)[1][page, 0, 3, 2] = fp4.NAN_SCALE
    out, lse = s.call()
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    nan = out[1].isnan()
    assert bool(nan[:, 32:48].all()) and not bool(nan[:, :32].any()) and not bool(nan[:, 48:].any())
    assert bool(lse[1].isfinite().all()) and bool(out[2].isfinite().all())


@pytest.mark.parametrize("bits", [4, 16])
def test_bad_pages_and_lengths(bits):
    s = Served([100, 200, 64, 70], 8, 2, 64, 32, bits=bits, seed=8, weights=True, softcap=9.0)
    good = [x.clone() for x in s.call(workspace={})]
    s.args["weights"].copy_(s.before)
    s.table[1, 2] = 10 ** 6           # a visible page outside the pool
    s.n[2] = s.table.shape[1] * 32 + 1  # past the table
    s.n[3] = -5                       # counts as 0
    ws = {}
    out, lse = s.call(workspace=ws)
    assert device_status(ws) == 2
    assert torch.equal(out[0], good[0][0]) and torch.equal(lse[0], good[1][0])
    assert bool(out[1:3].isnan().all()) and bool(lse[1:3].isnan().all())
    assert not bool(out[3].any()) and bool((lse[3] == -math.inf).all())
    rest = s.args["weights"] - s.before
    assert bool(rest[0].any()) and not bool(rest[1:].any())


@pytest.mark.parametrize("bits", [4, 16])
def test_a_captured_step_of_growing_sequences(bits):
    """Lengths, tables and slopes are read on the device; the weights add up over replays."""
    s = Served([40, 65, 0, 300], 8, 2, 64, 16, bits=bits, seed=9, weights=True, slopes=True,
               window=50, prefix=8, dtype=torch.float32)
    # all rows of the tables' pages visible from here on
    full = Served([336] * 4, 8, 2, 64, 16, bits=bits, seed=10, spare=0, slopes=True)
    s.kp, s.vp, s.table = full.kp, full.vp, full.table
    ws, total = {}, s.before.clone()
    s.call(workspace=ws)
    s.args["weights"].copy_(s.before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = s.call(workspace=ws)
    for step in range(3):
        s.n.copy_(torch.tensor([40, 65, 2, 300], device=DEV) + 11 * step)
        s.args["slopes"].mul_(0.5)
        graph.replay()
        eager = {**s.args, "weights": total}
        want = paged_attention(s.q, s.kp, s.vp, s.table, s.n, return_lse=True, **eager)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert torch.equal(s.args["weights"], total)
    assert device_status(ws) == 0


def test_one_workspace_for_every_form_and_pool():
    ws, first = {}, {}
    shapes = [dict(bits=4, softcap=8.0), dict(bits=16, slopes=True), dict(bits=4, weights=True),
              dict(bits=16, weights=True), dict(bits=16)]
    for turn in range(2):
        for i, form in enumerate(shapes):
            for j, (lengths, hq, hk, dim, block) in enumerate(
                    [([9000, 12], 32, 8, 128, 32), ([40] * 100, 4, 4, 64, 16), ([3, 2000, 0], 32, 2, 256, 64)]):
                s = Served(lengths, hq, hk, dim, block, seed=j, **form)
                out, lse = s.call(workspace=ws)
                s.check(out, lse)
                if turn:
                    assert torch.equal(out, first[i, j])
                first[i, j] = out.clone()
    assert device_status(ws) == 0


def test_two_calls_at_once_on_streams_of_their_own():
    a = Served([9000, 12, 500], 32, 8, 128, 32, bits=4, seed=1, weights=True)
    b = Served([5000, 3], 28, 4, 128, 16, seed=2, weights=True, softcap=30.0)
    want = []
    for s in (a, b):
        out, lse = s.call()
        want.append((out.clone(), lse.clone(), s.args["weights"].clone()))
    streams = [torch.cuda.Stream() for _ in "ab"]
    spaces = [{}, {}]
    for s, space in zip((a, b), spaces):
        s.call(workspace=space)
    torch.cuda.synchronize()
    for turn in range(20):
        got = []
        for s, stream, space in zip((a, b), streams, spaces):
            s.args["weights"].copy_(s.before)
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(s.call(workspace=space))
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        for s, (out, lse), w in zip((a, b), got, want):
            assert torch.equal(out, w[0]) and torch.equal(lse, w[1])
            assert torch.equal(s.args["weights"], w[2])


def test_views_of_pools_weights_and_slopes():
    s = Served([100, 31], 8, 2, 64, 16, bits=4, seed=11, weights=True, slopes=True)
    out, lse = (x.clone() for x in s.call())
    added = s.args["weights"] - s.before
    # pools cut out of a wider tensor, pages and heads further apart
    wide = torch.full((s.kp.shape[0], 5, 16, 36), 0xFF, device=DEV, dtype=torch.uint8)
    wide[:, 1:3], wide[:, 3:5] = s.kp, s.vp
    s.kp, s.vp = wide[:, 1:3], wide[:, 3:5]
    # weights cut out of a wider tensor, at an odd place
    held = torch.zeros(2, 3, 400, device=DEV)
    s.args["weights"] = held[:, 1:, 5:5 + s.table.shape[1] * 16]
    s.args["slopes"] = torch.stack([s.args["slopes"], s.args["slopes"]], 1)[:, 0]
    got = s.call()
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)
    # 0 + p against w + p - w: a rounding of w + p, below 2
    assert float((s.args["weights"] - added[..., :s.table.shape[1] * 16]).abs().max()) <= 2 ** -23
    assert not bool(held[:, 0].any())


def test_refusals():
    s = Served([40], 8, 2, 64, 16, seed=12)
    four = Served([40], 8, 2, 64, 16, bits=4, seed=12)
    w = torch.zeros(1, 2, s.table.shape[1] * 16, device=DEV)

    def no(error, match, served=s, **kw):
        with pytest.raises(error, match=match):
            served.call(**kw)

    for cap in (0.0, -1.0, math.inf, math.nan):
        no(ValueError, "softcap", softcap=cap)
    no(ValueError, "softcap", softcap=1e-60)  # nothing is left of it in fp32
    no(ValueError, "prefix", prefix=-1)
    no(ValueError, "slopes", slopes=torch.zeros(2, device=DEV))
    no(TypeError, "slopes", slopes=torch.zeros(8, device=DEV, dtype=torch.float64))
    no(ValueError, "slopes", slopes=torch.zeros(8))
    no(ValueError, "belong", key_scale=torch.ones(2, device=DEV))
    no(ValueError, "key_scale", four, key_scale=torch.ones(3, device=DEV))
    no(ValueError, "weights", weights=w[..., :-1])
    no(ValueError, "weights", weights=w[:, :1])
    no(TypeError, "weights", weights=w.double())
    no(ValueError, "overlap", weights=w[:, :1].expand(1, 2, -1))
    no(ValueError, "contiguous", weights=torch.zeros(1, 2, 2 * w.shape[2], device=DEV)[..., ::2])
    no(ValueError, "HND", four, layout="NHD")
