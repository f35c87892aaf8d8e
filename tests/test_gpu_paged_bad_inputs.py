"""What a bad length or page does to paged attention's results and to the status (needs a B200).

A row whose tokens cannot be had is NaN, in the output and in its sum: never
the page of another sequence, and never the part of the row that could be had.
The status of a workspace outlives the scratch it was first written to.
"""

import math

import pytest
import torch

from refinekv_b200 import paged_attention
from refinekv_b200.attention import device_status
from test_gpu_paged_attention import Served

pytestmark = pytest.mark.gpu


def _harmless(s):
    """Zeros in place of the NaN and infinity of the rows that are not visible: what is read of
    them by mistake then leaves a plausible result."""
    for pool in (s.kp, s.vp):
        pool.nan_to_num_(nan=0.0, posinf=0.0, neginf=0.0)


def _only(bad, out, lse, want, want_lse):
    """Rows `bad` are NaN throughout, the others have the bits of the healthy call."""
    for i in range(len(out)):
        if i in bad:
            assert bool(out[i].isnan().all()) and bool(lse[i].isnan().all()), i
        else:
            assert torch.equal(out[i], want[i]) and torch.equal(lse[i], want_lse[i]), i


@pytest.mark.parametrize("lengths,hq,hk,dim,block,layout,row", [
    ([40, 40, 7], 4, 2, 64, 32, "HND", 1),         # tiles of two pages
    ([100, 130], 8, 1, 64, 64, "NHD", 0),          # pages of a whole tile
    ([100, 333, 20], 28, 4, 128, 16, "NHD", 1),    # two pages a tile, two tiles a page
    ([70, 200], 16, 1, 256, 64, "HND", 1),
    ([9000, 12], 32, 8, 128, 32, "HND", 0),        # rows cut over CTAs
    ([70000, 3], 8, 1, 128, 32, "HND", 0),         # and joined in groups
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_a_page_outside_the_pool_makes_its_row_nan(lengths, hq, hk, dim, block, layout, row, dtype,
                                                   where):
    s = Served(lengths, hq, hk, dim, block, layout, dtype, seed=dim)
    _harmless(s)
    ws = {}
    want, want_lse = (x.clone() for x in s.call(workspace=ws))
    blocks = -(-lengths[row] // block)
    at = {"first": 0, "middle": blocks // 2, "last": blocks - 1}[where]
    good = int(s.table[row, at])
    for bad in (-1, s.kp.shape[0], -2 ** 31, 2 ** 31 - 1):
        s.table[row, at] = bad
        mine = {}
        _only({row}, *s.call(workspace=mine), want, want_lse)
        assert device_status(mine) == 2
        _only({row}, *s.call(), want, want_lse)  # without a workspace there is no other sign
    s.table[row, at] = good
    again = s.call(workspace=ws)
    assert torch.equal(again[0], want) and torch.equal(again[1], want_lse)
    assert device_status(ws) == 0


def test_every_page_of_a_tile_outside_the_pool():
    s = Served([64, 64], 4, 2, 64, 16, seed=1)
    _harmless(s)
    want, want_lse = (x.clone() for x in s.call())
    s.table[0, :4] = -3  # nothing of the row's only tile can be loaded
    _only({0}, *s.call(), want, want_lse)


@pytest.mark.parametrize("window", [None, 24])
def test_a_length_past_the_table_makes_its_row_nan(window):
    s = Served([40, 50, 64, 3], 4, 2, 64, 32, seed=2, spare=0, window=window)
    _harmless(s)
    want, want_lse = (x.clone() for x in s.call())
    for bad in (65, 1 << 30, 2 ** 31 - 1):
        s.n.copy_(torch.tensor([40, bad, 64, 3]))
        ws = {}
        _only({1}, *s.call(workspace=ws), want, want_lse)
        assert device_status(ws) == 2
    s.n.copy_(torch.tensor([40, -5, 64, 3]))  # the nearest length: an empty row
    ws = {}
    out, lse = s.call(workspace=ws)
    assert device_status(ws) == 2
    assert not bool(out[1].any()) and bool((lse[1] == -math.inf).all())
    keep = torch.tensor([0, 2, 3], device="cuda")
    assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])


def test_only_bad_lengths():
    s = Served([5, 9], 16, 1, 128, 32, seed=3, spare=0)
    _harmless(s)
    s.n.copy_(torch.tensor([33, 100]))
    out, lse = s.call()
    assert bool(out.isnan().all()) and bool(lse.isnan().all())
