"""The page-pool serving example with pools of 4 bits and with a budget: its operators together, as
a server uses them.

The reference is one step of a one-layer decoder in 64 bits over what the pool holds before the
step (``paged_read``, tested by itself) and the new token's row.  The example keeps activations in
bf16, so its logits must agree to 2 % of their scale, as in test_gpu_serving_example.py.
"""

import pytest
import torch

import fp4_helpers as fp4
from refinekv_b200 import apply_rotary, paged_read
from test_gpu_serving_example import _example

pytestmark = pytest.mark.gpu


def _prompts(*lengths):
    gen = torch.Generator().manual_seed(5)
    return [torch.randint(0, 512, (n,), generator=gen) for n in lengths]


def _held(server, i, rows):
    """(rows, KV heads, dim) fp64 keys and values of sequence i."""
    at = torch.arange(rows, device="cuda", dtype=torch.int32)
    return [x.double() for x in paged_read(*server.pools[0], server.table, at,
                                           sequence_ids=torch.full_like(at, i),
                                           dtype=torch.float32)]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("budget", [None, 40, 1000])
def test_a_step_attends_over_what_the_pool_holds(bits, budget):
    ex = _example()
    model = ex.Decoder(layers=1, dense=1)
    prompts = _prompts(61, 1, 200, 32)
    server = ex.Server(model, prompts, 12, bits=bits, budget=budget, recent=8)
    groups = model.hq // model.hk
    for step in range(8):
        rows = server.lengths if budget is None else server.rows
        counts = rows.tolist()
        x = model.embed[server.tokens]
        q, k, v = model.project(0, x)
        if bits == 4 and budget is None:  # rotated in fp32 on the way
            q = apply_rotary(q, None, server.lengths, server.cos_sin)[0]
            k = apply_rotary(k.float(), None, server.lengths, server.cos_sin)[0]
        else:
            q, k = apply_rotary(q, k, server.lengths, server.cos_sin)
        if bits == 4:
            k, v = (fp4.values(*fp4.quantise(t.float())) for t in (k, v))
        before = [_held(server, i, n) for i, n in enumerate(counts)]
        kept = None if budget is None else server.held[0].clone()
        logits = server.step()
        for i, (keys, values) in enumerate(before):
            keys = torch.cat([keys, k[i:i + 1].double()])
            values = torch.cat([values, v[i:i + 1].double()])
            heads = q[i].double().view(model.hk, groups, model.dim)
            p = torch.einsum("hgd,thd->hgt", heads, keys).mul(model.dim ** -0.5).softmax(-1)
            y = torch.einsum("hgt,thd->hgd", p, values).flatten()
            want = model.logits((x[i].double() + y @ model.out[0].double()).float())
            assert float((logits[i] - want).abs().max()) <= 0.02 * float(want.abs().max())
            if budget is None:
                continue
            now = len(prompts[i]) + step
            new = min(counts[i] + 1, budget)
            assert int(server.rows[i]) == new
            for h in range(model.hk):
                left = server.held[0][i, h, :new].tolist()
                had = kept[i, h, :counts[i]].tolist() + [now]
                assert len(set(left)) == new and set(left) <= set(had)
                assert set(had[-8:]) <= set(left) if step == 0 else now in left
                stay = server.weights[0][i, h, :new]
                assert bool((stay >= 0).all()) and not bool(server.weights[0][i, h, new:].any())
    assert server.healthy()


def test_a_budget_that_is_never_reached_changes_nothing():
    ex = _example()
    prompts = _prompts(61, 1, 200, 32)
    runs = []
    for budget in (None, 512):
        server = ex.Server(ex.Decoder(layers=2, dense=2), prompts, 12, budget=budget)
        runs.append(server.generate())
        assert server.healthy()
    # the same rotation, the same rows, the same attention
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


def test_generated_steps_of_a_captured_graph_are_the_eager_ones():
    ex = _example()
    prompts = _prompts(61, 1, 200, 32)
    logits = []
    for captured in (True, False):
        server = ex.Server(ex.Decoder(layers=2, dense=2), prompts, 12, bits=4, budget=48, recent=4)
        if captured:
            logits.append(server.generate()[1])
        else:
            logits.append(torch.stack([server.step().clone() for _ in range(12)], 1))
        assert server.healthy() and server.rows.tolist() == [48, 13, 48, 44]
    assert torch.equal(*logits)


def test_servers_that_cannot_be():
    ex = _example()
    with pytest.raises(ValueError, match="bits"):
        ex.Server(ex.Decoder(), _prompts(5), 2, bits=8)
    with pytest.raises(ValueError, match="refined"):
        ex.Server(ex.Decoder(), _prompts(5), 2, budget=4)
