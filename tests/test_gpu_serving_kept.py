"""What the page-pool serving example keeps within a budget, step by step (needs a B200).

Before a step the test knows each row's token and what weight it has so far; the step's own
weights are worked out in 64 bits from the rows in the pool and the step's queries and keys, which
are the server's own (the same operations on the same inputs).  The server's sums are off from these
by the attention's errors, 2^-10 of a weight at the most (test_gpu_paged_more.py bounds them by a
hundredth of that here), so that a token is dropped in place of one that weighs less only
where the two lie that close.
"""

import pytest
import torch

import fp4_helpers as fp4
from refinekv_b200 import apply_rotary
from test_gpu_serving_budget import _held, _prompts
from test_gpu_serving_example import _example

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("budget,recent", [(40, 8), (40, 0), (12, 12), (33, 1)])
def test_the_newest_and_the_heaviest_stay(bits, budget, recent):
    ex = _example()
    model = ex.Decoder(layers=1, dense=1)
    prompts = _prompts(61, 1, 200, 32)
    server = ex.Server(model, prompts, 12, bits=bits, budget=budget, recent=recent)
    for step in range(10):
        counts = server.rows.tolist()
        x = model.embed[server.tokens]
        q, k, _ = model.project(0, x)
        q, k = apply_rotary(q, k, server.lengths, server.cos_sin)
        k = fp4.values(*fp4.quantise(k.float())) if bits == 4 else k.double()
        before = [_held(server, i, n)[0] for i, n in enumerate(counts)]
        tokens, weights = server.held[0].clone(), server.weights[0].double()
        server.step()
        for i, keys in enumerate(before):
            keys = torch.cat([keys, k[i:i + 1]])
            heads = q[i].double().view(model.hk, -1, model.dim)
            p = torch.einsum("hgd,thd->hgt", heads, keys).mul(model.dim ** -0.5).softmax(-1).sum(1)
            now = len(prompts[i]) + step
            for h in range(model.hk):
                had = tokens[i, h, :counts[i]].tolist() + [now]
                worth = dict(zip(had, (weights[i, h, :counts[i] + 1] + p[h]).tolist()))
                new = min(len(had), budget)
                left = server.held[0][i, h, :new].tolist()
                assert len(set(left)) == new and set(left) <= set(had)
                newest = {t for t in had if t > now - recent}
                assert newest <= set(left)
                dropped = set(had) - set(left)
                if dropped and set(left) - newest:
                    most = max(worth[t] for t in dropped)
                    least = min(worth[t] for t in set(left) - newest)
                    assert most <= least * (1 + 2 ** -9), (step, i, h)
                # their weights went along with them
                got = dict(zip(left, server.weights[0][i, h, :new].tolist()))
                assert all(abs(got[t] - worth[t]) <= 2 ** -10 * worth[t] for t in left)
    assert server.healthy()


@pytest.mark.parametrize("budget,recent", [(8, 16), (0, 0), (-3, 0), (8, -1), (8, 9)])
def test_a_budget_that_cannot_be_is_refused_at_once(budget, recent):
    ex = _example()
    with pytest.raises(ValueError, match="budget"):
        ex.Server(ex.Decoder(layers=2, dense=2), _prompts(40), 2, budget=budget, recent=recent)
