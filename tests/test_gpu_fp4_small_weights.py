"""Attention over pools of 4 bits where the tokens of greatest weight have values of zero: the
output is what the tokens of small weight say (needs a B200).

Bounds, with the formula of test_gpu_paged_more.py's: p_j exact weights, A = sum_j p_j |v_j| per
channel, X = max_j scale sum_i |q_i k_ji|, u = 2^-23, e = (dim / 8 + 3) u X for a logit, and D the
distance of the greatest logit from the least.  A weight that lies d <= D below the greatest comes
from exponentials whose arguments add up to -d: an argument's difference is rounded once, its factor
log2(e) is off by 2^-25 at most, the product (with a constant up to 16 added to it) is rounded
once more, 2^-24 each, so that all of them are off by 2.5 d 2^-24 + 2^-20, and by 2^-22 for each of four
exponentials (in the tile, over the warps, the CTAs, groups of CTAs): 2^-19 + D 2^-22 is more than
that.  A weight is held in fp16 terms with 2^-11 (bf16 queries) or 2^-22 (fp32 queries) of itself,
however small it is.  The sums add 16 rows at a time, for four sizes of weights at most here,
half a u each, and merge a few dozen parts:
  fp32 queries:  |out - exact| <= A (2 e + 2^-19 + D 2^-22 + 2^-22 + (rows / 8 + 64) u) + |exact| 2 u
  bf16 queries:  A 2^-11 more, and half a unit in the result's last place.
What the kernel leaves out of small weights, 2^-18 of A for bf16 queries and 2^-21 for fp32 ones, is
within this: it leaves none out but 35 and 18 nats below the greatest, where D (2^-22 - 2.5 2^-24)
is 2^-18.3 and 2^-19.3, and for bf16 queries half of the sums' part is unused, 2^-18 at least.
"""

import pytest
import torch

import fp4_helpers as fp4
from refinekv_b200 import fp4_pool, paged_attention
from refinekv_b200.attention import device_status

pytestmark = pytest.mark.gpu
DEV = "cuda"

#: How far, in nats, the greatest logit of a query lies above the others.
DISTANCES = (0.0, 6.0, 12.0, 15.0, 18.0, 22.0, 30.0, 45.0, 60.0, 80.0)


class Above:
    """Sequences whose token j has a logit of about ``distance * heights[j]`` (a query head's own
    distance), and a row of zeros for a value where that height is not 0."""

    def __init__(self, heights, hq, hk, dim, block, dtype, seed=0, noise=1.0, values_up_to=0.0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        n, lengths = len(heights), [len(h) for h in heights]
        blocks = -(-max(lengths) // block) + 1
        self.table = torch.randperm(n * blocks, generator=gen, device=DEV).int().view(n, blocks)
        self.n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
        self.pools = [fp4_pool(n * blocks, hk, block, dim) for _ in "kv"]
        for pool in self.pools:
            fp4.parts(pool)[1].fill_(fp4.NAN_SCALE)  # rows that are not visible
        self.rows = []
        for i, height in enumerate(heights):
            height = torch.tensor(height, device=DEV)[:, None, None]
            at = torch.arange(len(height), device=DEV)
            page, row = self.table[i].long()[at // block], at % block
            k, v = (torch.randn(len(height), hk, dim, generator=gen, device=DEV) for _ in "kv")
            k[..., :16] = 6 * height
            k[..., 16:] *= noise * (height == 0)
            v *= height <= values_up_to
            both = []
            for pool, x in zip(self.pools, (k, v)):
                held = fp4.quantise(x)
                for part, new in zip(fp4.parts(pool), held):
                    part.transpose(1, 2)[page, row] = new
                both.append(fp4.values(*held))
            self.rows.append(both)
        self.q = torch.randn(n, hq, dim, generator=gen, device=DEV)
        above = torch.tensor(DISTANCES, device=DEV)[torch.arange(hq, device=DEV) % len(DISTANCES)]
        self.q[..., :16] = (above * dim ** 0.5 / 96)[:, None]
        self.q = self.q.to(dtype)

    def check(self, **more):
        workspace = {}
        out = paged_attention(self.q, *self.pools, self.table, self.n, workspace=workspace, **more)
        assert device_status(workspace) == 0 and out.dtype == self.q.dtype
        u, slopes = 2.0 ** -23, more.get("slopes")
        hq, dim = self.q.shape[1:]
        for i, (k, v) in enumerate(self.rows):
            hk = k.shape[1]
            q = self.q[i].to(torch.bfloat16).double().view(hk, hq // hk, dim)
            k, v = k.transpose(0, 1), v.transpose(0, 1)
            x = q @ k.transpose(1, 2) * dim ** -0.5
            e = (dim / 8 + 3) * u * (q.abs() @ k.abs().transpose(1, 2)).amax(-1) * dim ** -0.5
            if slopes is not None:  # its own rounding and the sum's
                bias = slopes.double().view(hk, -1, 1) * (torch.arange(x.shape[-1], device=DEV)
                                                          - (x.shape[-1] - 1))
                e = e + u * (bias.abs().amax(-1) + (x + bias).abs().amax(-1))
                x = x + bias
            p = x.softmax(-1)
            want, size = (p @ v).reshape(hq, dim), (p @ v.abs()).reshape(hq, dim)
            far = x.amax(-1) - x.amin(-1)
            part = 2 * e + 2.0 ** -19 + far * 2.0 ** -22 + 2.0 ** -22 + (x.shape[-1] / 8 + 64) * u
            tol = size * part.reshape(hq, 1) + want.abs() * 2 * u + 1e-37
            if out.dtype == torch.bfloat16:
                half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 1 - 8)
                tol = tol * 1.01 + size * 2.0 ** -11 + half
            off = (out[i].double() - want).abs()
            worst = (off / tol).amax(-1)
            assert bool((off <= tol).all()), (i, [round(w, 2) for w in worst.tolist()])


def _one_above(length, at):
    return [float(j == at % length) for j in range(length)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("at", [0, -1, 777])
@pytest.mark.parametrize("hq,hk,dim,block", [
    (10, 1, 128, 32), (8, 1, 128, 64), (20, 2, 64, 16), (10, 2, 96, 32), (16, 1, 32, 16),
    (5, 1, 256, 64), (16, 1, 256, 16), (10, 1, 160, 32), (10, 1, 192, 16), (7, 1, 224, 32)])
def test_what_lies_below_one_great_token_counts(hq, hk, dim, block, at, dtype):
    """In its tile and in others, before it and behind it, over one CTA and over many."""
    lengths = (3000, 64, 2, 17, 100, 40000) if dim == 128 else (3000, 64, 2, 17)
    Above([_one_above(n, at) for n in lengths], hq, hk, dim, block, dtype, seed=dim + hq).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,dim", [(8, 128), (16, 64), (10, 96)])
@pytest.mark.parametrize("way", [1, -1])
def test_weights_of_every_size_in_a_tile(hq, dim, way, dtype):
    """Logits that rise or fall by steps; only the lowest, then the lower half, have values."""
    steps = (6.0, 4.0, 3.0, 2.0, 1.5, 1.0, 0.5, 0.0)[::way]
    heights = [[steps[j * 8 // n] / 6 for j in range(n)] for n in (64, 8, 23, 700, 5000)]
    for most in (0.0, 0.3):
        Above(heights, hq, 1, dim, 32, dtype, seed=dim, values_up_to=most).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("slope", [1.0, -1.0, 0.25])
def test_steep_biases(slope, dtype):
    """A bias of a nat a token: the newest (or the first) have nearly all of the weight and no value."""
    for n in (60, 130, 400):
        near = [float(n - 1 - j < 20 or j < 20) / 1e3 for j in range(n)]
        s = Above([near, near[20:]], 8, 2, 128, 32, dtype, seed=n, noise=0.1)
        s.check(slopes=torch.full((8,), slope, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_small_weights_and_nan(dtype):
    """A NaN logit makes its row NaN, a NaN value its channels, next to weights of every size."""
    s = Above([_one_above(64, 0)] * 3, 10, 1, 128, 32, dtype)
    page = int(s.table[1, 1])
    fp4.parts(s.pools[0])[1][page, 0, 5, 3] = fp4.NAN_SCALE
    page = int(s.table[2, 1])
    fp4.parts(s.pools[1])[1][page, 0, 5, 3] = fp4.NAN_SCALE
    out = paged_attention(s.q, *s.pools, s.table, s.n)
    assert bool(out[0].isfinite().all()) and bool(out[1].isnan().all())
    nan = out[2].isnan()
    assert bool(nan[:, 48:64].all()) and not bool(nan[:, :48].any()) and not bool(nan[:, 64:].any())
