"""Eviction from a page pool against its definition, row by row (needs a B200).  Everything is
exact: rows, weights and positions are moved, never computed."""

import math

import pytest
import torch

import fp4_helpers as fp4
from refinekv_b200 import (apply_rotary, fp4_pool, paged_append, paged_attention, paged_evict,
                           rotary_table)
from refinekv_b200.attention import device_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Full:
    """Pools of random bytes (each row its own), weights, and positions when `aged`."""

    def __init__(self, lengths, hk, dim, block, layout="HND", bits=16, aged=False, seed=0, spare=1):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.lengths, self.block, self.layout, self.bits = lengths, block, layout, bits
        n, blocks = len(lengths), max(1, -(-max(lengths) // block)) + spare
        pages = n * blocks + 1
        if bits == 4:
            self.pools = [fp4_pool(pages, hk, block, dim) for _ in "kv"]
            for pool in self.pools:
                pool.random_(0, 256, generator=gen)
        else:
            shape = (pages, hk, block, dim) if layout == "HND" else (pages, block, hk, dim)
            self.pools = [torch.randint(-2 ** 15, 2 ** 15, shape, generator=gen, device=DEV,
                                        dtype=torch.int16).view(torch.bfloat16) for _ in "kv"]
        order = torch.randperm(pages, generator=gen, device=DEV)[: n * blocks]
        self.table = order.view(n, blocks).int()
        self.n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
        self.w = torch.rand(n, hk, blocks * block, generator=gen, device=DEV)
        self.at = None
        if aged:
            self.at = torch.rand(n, hk, blocks * block, generator=gen, device=DEV).argsort(-1).int() - 50

    def rows(self, pools, i, h):
        """Sequence i's rows of KV head h as bytes: (tokens, bytes) of keys and values together."""
        at = torch.arange(self.table.shape[1] * self.block, device=DEV)
        page, row = self.table[i].long()[at // self.block], at % self.block
        out = []
        for pool in pools:
            if self.bits == 4:
                out += [part[page, h, row] for part in fp4.parts(pool)]
            else:
                x = pool[page, h, row] if self.layout == "HND" else pool[page, row, h]
                out.append(x.view(torch.uint8))
        return torch.cat(out, -1)

    def evict(self, budget, recent, **kw):
        return paged_evict(*self.pools, self.table, self.n, self.w, budget, recent=recent,
                           positions=self.at, layout=self.layout, **kw)

    def check(self, budget, recent, **kw):
        pools, w = [p.clone() for p in self.pools], self.w.clone()
        at = None if self.at is None else self.at.clone()
        lengths = self.n.tolist()
        new = self.evict(budget, recent, **kw)
        assert new.tolist() == [min(max(n, 0), budget) for n in lengths]
        for i, n in enumerate(lengths):
            for h in range(w.shape[1]):
                want_rows, want_w = self.rows(pools, i, h), w[i, h].clone()
                want_at = None if at is None else at[i, h].clone()
                if n > budget:
                    age = torch.arange(n) if at is None else at[i, h, :n].cpu()
                    newest = int(age.max())
                    worth = w[i, h, :n].tolist()
                    key = [(0 if recent and int(a) > newest - recent else 1,
                            math.inf if math.isnan(x) else -x) for a, x in zip(age, worth)]
                    # NaN after -inf
                    key = [(a, 1 if math.isnan(x) else 0, b) for (a, b), x in zip(key, worth)]
                    key = [(0, 0, 0) if k[0] == 0 else k for k in key]
                    kept = sorted(sorted(range(n), key=lambda j: key[j])[:budget])
                    holes = torch.tensor(sorted(set(range(budget)) - set(kept)), device=DEV).long()
                    movers = torch.tensor([j for j in kept if j >= budget], device=DEV).long()
                    want_rows[holes] = want_rows[movers]
                    want_w[holes] = want_w[movers]
                    want_w[budget:n] = 0
                    if at is not None:
                        want_at[holes] = want_at[movers]
                assert torch.equal(self.rows(self.pools, i, h), want_rows), (i, h)
                assert torch.equal(self.w[i, h].view(torch.int32), want_w.view(torch.int32)), (i, h)
                assert at is None or torch.equal(self.at[i, h], want_at)
        # pages that no table names keep their bytes
        free = torch.ones(len(pools[0]), device=DEV, dtype=torch.bool)
        free[self.table.long().flatten()] = False
        for a, b in zip(pools, self.pools):
            assert torch.equal(a[free].view(torch.uint8), b[free].view(torch.uint8))
        return new


CASES = [
    # lengths, KV heads, dim, block, layout, budget, recent
    ([5, 4, 3, 0], 2, 32, 16, "HND", 4, 0),
    ([5, 4, 3, 0], 2, 32, 16, "NHD", 4, 4),
    ([2, 1], 1, 64, 16, "HND", 1, 0),
    ([2, 100], 1, 64, 16, "HND", 1, 1),
    ([100, 31, 32, 33, 65], 3, 128, 32, "NHD", 32, 7),
    ([1000, 517, 1], 4, 96, 64, "HND", 500, 100),
    ([1000, 999], 2, 256, 16, "NHD", 999, 1),
    ([513, 512, 511], 2, 160, 32, "HND", 256, 256),
    ([4097] * 5, 4, 64, 32, "HND", 4096, 256),
    ([300], 1, 224, 64, "HND", 1000, 3),       # nothing to do
    ([9000, 20000], 2, 32, 32, "HND", 700, 50),  # rows shared by clusters
    ([70001], 1, 32, 64, "NHD", 30000, 512),
]


@pytest.mark.parametrize("lengths,hk,dim,block,layout,budget,recent", CASES)
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("aged", [False, True])
def test_the_rows_of_greatest_weight_stay(lengths, hk, dim, block, layout, budget, recent, bits, aged):
    if bits == 4:
        layout = "HND"
    f = Full(lengths, hk, dim, block, layout, bits, aged, seed=dim)
    ws = {}
    f.check(budget, recent, workspace=ws)
    assert device_status(ws) == 0
    f.n.copy_(torch.tensor(lengths, device=DEV))  # once more: the same lengths, other weights
    f.w.uniform_()
    f.check(budget, recent, workspace=ws)


@pytest.mark.parametrize("kind", ["equal", "few", "zero", "special", "negative"])
def test_ties_and_special_weights(kind):
    f = Full([600, 257, 5000], 2, 32, 32, seed=1)
    if kind == "equal":
        f.w.fill_(0.5)
    elif kind == "few":
        f.w.copy_((f.w * 5).floor())
    elif kind == "zero":
        f.w.copy_(torch.where(f.w < 0.5, -0.0, 0.0))
    elif kind == "negative":
        f.w.sub_(0.5)
    else:
        for at, x in ((0.2, math.nan), (0.4, -math.inf), (0.6, math.inf), (0.7, -1e38)):
            f.w.masked_fill_((f.w > at) & (f.w < at + 0.15), x)
    f.check(256, 0)


def test_duplicate_positions_of_the_newest():
    """More rows among the newest than the budget: the first of them stay."""
    f = Full([200], 1, 32, 16, aged=True, seed=2)
    f.at.fill_(7)
    f.check(50, 20)


def test_extreme_positions():
    f = Full([200], 1, 32, 16, aged=True, seed=3)
    f.at[..., ::2] -= 2 ** 31 - 300
    f.at[..., 5] = 2 ** 31 - 1
    f.check(50, 20)


def test_rows_longer_than_shared_memory_holds():
    f = Full([400000], 1, 32, 64, seed=4)
    f.w.copy_((f.w * 4096).floor())
    f.check(1000, 300)
    f = Full([350000], 1, 32, 64, aged=True, seed=5)
    f.check(340000, 300)


def test_weights_and_positions_of_wider_tensors_and_strided_pools():
    f = Full([100, 90], 2, 64, 32, bits=4, aged=True, seed=6)
    width = f.w.shape[2]
    wide = torch.zeros(3, 2, width + 9, device=DEV)
    wide[1:, :, 5:5 + width] = f.w
    at = torch.zeros(2, 4, width + 1, device=DEV, dtype=torch.int32)
    at[:, ::2, :width] = f.at
    f.w, f.at = wide[1:, :, 5:], at[:, ::2]
    both = torch.zeros(f.pools[0].shape[0], 5, 32, 36, device=DEV, dtype=torch.uint8)
    both[:, :2], both[:, 3:] = f.pools
    f.pools = [both[:, :2], both[:, 3:]]
    f.check(64, 9)
    assert not bool(both[:, 2].any()) and not bool(wide[0].any()) and not bool(at[:, 1::2].any())


def test_the_returned_lengths_may_be_the_next_lengths():
    f = Full([100, 90, 20], 8, 64, 32, seed=7)
    ws = {}
    f.n = f.check(64, 0, workspace=ws)
    f.n = f.check(32, 0, workspace=ws)
    assert f.n.tolist() == [32, 32, 20]
    assert f.check(33, 0, workspace=ws).tolist() == [32, 32, 20]


def test_the_buffers_of_returned_lengths_stay():
    """A captured eviction writes its lengths into the workspace's buffer on every replay, so
    calls that are given that buffer as their lengths must not have it replaced."""
    pools = [torch.zeros(2, 1, 16, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    table = torch.arange(2, device="cuda", dtype=torch.int32).view(1, 2)
    weights, ws = torch.rand(1, 1, 32, device="cuda"), {}
    lengths = torch.tensor([32], device="cuda", dtype=torch.int32)
    buffers = []
    for budget in (20, 16, 9, 4):
        lengths = paged_evict(*pools, table, lengths, weights, budget, workspace=ws)
        assert lengths.item() == budget
        buffers.append(lengths.data_ptr())
    assert buffers[0] == buffers[2] and buffers[1] == buffers[3] and buffers[0] != buffers[1]
    kept = {t.data_ptr() for name, t in ws.items() if name.startswith("evict_lengths")}
    assert kept == set(buffers)


@pytest.mark.parametrize("bits", [4, 16])
def test_bad_lengths_and_pages(bits):
    f = Full([100, 100, 100, 100], 2, 32, 32, bits=bits, seed=8)
    f.w[:, :, :64] = 0
    f.w[:, :, 64:] += 1
    f.n[1] = f.table.shape[1] * 32 + 1
    f.n[2] = -3
    before, w = [f.rows(f.pools, i, 0) for i in range(4)], f.w.clone()
    f.table[0, 2], f.table[3, 0] = 10 ** 6, -1   # a source page, a target page
    ws = {}
    assert f.evict(64, 0, workspace=ws).tolist() == [64, f.table.shape[1] * 32 + 1, 0, 64]
    assert device_status(ws) == 2
    for i in (1, 2):
        assert torch.equal(f.rows(f.pools, i, 0), before[i]) and torch.equal(f.w[i], w[i])
    f.table[0, 2] = f.table[0, 1]
    got = f.rows(f.pools, 0, 0)
    # kept are rows 64..99 and, of those without weight, the first 28: rows 64..95, in the bad page, go
    # to rows 28..59 and rows 96..99 behind them
    assert torch.equal(got[:28], before[0][:28]) and torch.equal(got[60:64], before[0][96:100])
    if bits == 16:
        assert bool(got[28:60].reshape(32, -1).view(torch.bfloat16).isnan().all())
    else:
        at = torch.arange(28, 60, device=DEV)
        for pool in f.pools:
            assert bool((fp4.parts(pool)[1][f.table[0].long()[at // 32], 0, at % 32] == fp4.NAN_SCALE).all())


def test_a_captured_step_that_keeps_a_budget():
    """A decode loop in a graph: rotate by the token's own position, append behind the kept rows,
    attend and add up the weights, evict.  Against the same steps on plain rows."""
    hq, hk, dim, block, budget, recent, n, steps = 8, 2, 64, 16, 24, 6, 3, 40
    gen = torch.Generator(device=DEV).manual_seed(9)
    blocks = -(-(budget + 1) // block)
    pages = torch.randperm(n * blocks, generator=gen, device=DEV).view(n, blocks).int()
    kp, vp = (torch.zeros(n * blocks, hk, block, dim, device=DEV, dtype=torch.bfloat16) for _ in "kv")
    cs = rotary_table(dim, steps + 8)
    lengths = torch.zeros(n, device=DEV, dtype=torch.int32)
    now = torch.tensor([0, 3, 7], device=DEV, dtype=torch.int32)
    start = now.clone()
    w = torch.zeros(n, hk, blocks * block, device=DEV)
    at = torch.zeros(n, hk, blocks * block, device=DEV, dtype=torch.int32)
    x = torch.zeros(n, hq + 2 * hk, dim, device=DEV, dtype=torch.bfloat16)
    ws = {}

    def step():
        q, k, v = x.split([hq, hk, hk], 1)
        q, k = apply_rotary(q, k, now, cs)
        paged_append(k, v, kp, vp, pages, lengths, workspace=ws)
        at.scatter_(2, lengths.long().view(n, 1, 1).expand(n, hk, 1),
                    now.view(n, 1, 1).expand(n, hk, 1))
        out = paged_attention(q, kp, vp, pages, lengths + 1, weights=w, workspace=ws)
        lengths.copy_(paged_evict(kp, vp, pages, lengths + 1, w, budget, recent=recent, positions=at,
                                  workspace=ws))
        now.add_(1)
        return out

    step()
    for t in (lengths, w, at):
        t.zero_()
    now.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in (lengths, w, at):
        t.zero_()
    now.copy_(start)
    held = [[dict(k=[], v=[], w=[], at=[]) for _ in range(hk)] for _ in range(n)]

    def off(x):
        """How far a sum x of weights may be: e <= 11 2^-23 X with X = max scale |q|.|k| < 12 (64
        channels), the sum's error e + 2^-20 + 33 2^-23, 2^-20 for the exponential: 2^-14.3 of
        every weight; `steps` additions of 2^-24 x each."""
        return x * 2 ** -14 + 1e-6

    for j in range(steps):
        x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
        q, k, v = x.split([hq, hk, hk], 1)
        q, k = apply_rotary(q, k, start + j, cs)
        graph.replay()
        for i in range(n):
            for h in range(hk):
                row = held[i][h]
                row["k"].append(k[i, h].double())
                row["v"].append(v[i, h].double())
                row["w"].append(0.0)
                row["at"].append(int(start[i]) + j)
                keys, values = torch.stack(row["k"]), torch.stack(row["v"])
                p = (q[i, h * 4:h * 4 + 4].double() @ keys.T * dim ** -0.5).softmax(-1)
                want = p @ values
                # bf16 weights and output: 2^-8 of sum p |v| and of the output each
                bound = (p @ values.abs()) * 2 ** -8 + want.abs() * 2 ** -8 + 1e-6
                assert bool(((out[i, h * 4:h * 4 + 4].double() - want).abs() <= bound).all())
                row["w"] = [a + b for a, b in zip(row["w"], p.sum(0).tolist())]
                got = w[i, h, :len(row["w"])].tolist()
                if len(row["w"]) > budget:  # one goes: not one of the newest, the least weight
                    left = at[i, h, :budget].tolist()
                    (gone,) = [r for r in range(budget + 1) if row["at"][r] not in left]
                    assert row["at"][gone] <= int(start[i]) + j - recent
                    least = min(x for r, x in enumerate(row["w"])
                                if row["at"][r] <= int(start[i]) + j - recent)
                    assert row["w"][gone] - least <= off(row["w"][gone]) + off(least)
                    # the last row takes its place
                    for values_of in row.values():
                        if gone < budget:
                            values_of[gone] = values_of[budget]
                        values_of.pop()
                    got = w[i, h, :budget].tolist()
                assert at[i, h, :len(row["at"])].tolist() == row["at"]
                assert all(abs(a - b) <= off(b) for a, b in zip(got, row["w"]))
    assert lengths.tolist() == [budget] * n and device_status(ws) == 0
    assert not bool(w[:, :, budget:].any())


def test_two_evictions_at_once_on_streams_of_their_own():
    a, b = Full([3000, 40], 2, 64, 32, seed=10), Full([20000], 1, 32, 32, aged=True, seed=11)
    streams = [torch.cuda.Stream() for _ in "ab"]
    copies = []
    for f in (a, b):
        g = Full.__new__(Full)
        g.__dict__.update(f.__dict__)
        g.pools, g.w = [p.clone() for p in f.pools], f.w.clone()
        g.at = None if f.at is None else f.at.clone()
        g.evict(1000, 30)
        copies.append(g)
    torch.cuda.synchronize()
    for f, stream in zip((a, b), streams):
        with torch.cuda.stream(stream):
            f.evict(1000, 30)
    torch.cuda.synchronize()
    for f, g in zip((a, b), copies):
        assert torch.equal(f.w, g.w)
        for p, q in zip(f.pools, g.pools):
            assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))


def test_refusals():
    f = Full([40], 2, 64, 16, seed=12)

    def no(error, match, budget=8, recent=2, **kw):
        args = dict(positions=None, layout="HND", weights=f.w, lengths=f.n) | kw
        with pytest.raises(error, match=match):
            paged_evict(*f.pools, f.table, args.pop("lengths"), args.pop("weights"), budget,
                        recent=recent, **args)

    no(ValueError, "budget", budget=0)
    no(ValueError, "recent", recent=9)
    no(ValueError, "recent", recent=-1)
    no(ValueError, "weights", weights=f.w[..., :-1])
    no(ValueError, "weights", weights=f.w.cpu())
    no(TypeError, "weights", weights=f.w.half())
    no(ValueError, "overlap", weights=f.w[:, :1].expand(-1, 2, -1))
    no(TypeError, "positions", positions=f.w.long())
    no(ValueError, "positions", positions=f.w.int()[:, :1])
    no(TypeError, "lengths", lengths=f.n.long())
    no(ValueError, "lengths", lengths=f.n.repeat(2))
    no(ValueError, "layout", layout="DHN")
