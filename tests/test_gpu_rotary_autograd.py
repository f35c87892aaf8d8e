"""The rotation next to torch's automatic differentiation (needs a B200).

Rotated values have the bounds of test_gpu_rotary.py.
"""

import pytest
import torch
from torch.autograd import forward_ad

from refinekv_b200 import apply_rotary, paged_append, rotary_table
from test_gpu_rotary import assert_rotated, rotate64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(dtype=torch.float32):
    gen = torch.Generator(device=DEV).manual_seed(1)
    make = lambda heads: torch.randn(9, heads, 64, generator=gen, device=DEV, dtype=dtype)  # noqa: E731
    at = torch.randint(0, 40, (9,), generator=gen, device=DEV)
    return make(4), make(2), make(4), make(2), at, rotary_table(48, 40)


@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tangents_are_rotated_with_their_rows(interleaved, inverse, dtype):
    q, k, dq, dk, at, table = _inputs(dtype)
    sign = -1.0 if inverse else 1.0
    kw = dict(interleaved=interleaved, inverse=inverse)
    with forward_ad.dual_level():
        out_q, out_k = apply_rotary(forward_ad.make_dual(q, dq), forward_ad.make_dual(k, dk), at,
                                    table, **kw)
        got_q, got_k = forward_ad.unpack_dual(out_q), forward_ad.unpack_dual(out_k)
        for got, rows, tangent in ((got_q, q, dq), (got_k, k, dk)):
            assert_rotated(got.primal, *rotate64(rows, at, table, interleaved, sign))
            assert_rotated(got.tangent, *rotate64(tangent, at, table, interleaved, sign))
        # one of the two alone, and no key
        only_q, plain_k = apply_rotary(forward_ad.make_dual(q, dq), k, at, table, **kw)
        assert torch.equal(forward_ad.unpack_dual(only_q).tangent, got_q.tangent)
        still = forward_ad.unpack_dual(plain_k).tangent
        assert still is None or not bool(still.any())
        plain_q, only_k = apply_rotary(q, forward_ad.make_dual(k, dk), at, table, **kw)
        assert torch.equal(forward_ad.unpack_dual(only_k).tangent, got_k.tangent)
        alone, none = apply_rotary(forward_ad.make_dual(q, dq), None, at, table, **kw)
        assert none is None
        assert torch.equal(forward_ad.unpack_dual(alone).tangent, got_q.tangent)


def test_tangent_against_differences():
    q, _, dq, _, at, table = _inputs()
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(
            apply_rotary(forward_ad.make_dual(q, dq), None, at, table)[0]).tangent
    # linear: a step of any size; both sides within 2^-21 of values below 16
    ahead, behind = (apply_rotary(q + h * dq, None, at, table)[0] for h in (1, -1))
    assert float(((ahead - behind).double() / 2 - tangent.double()).abs().max()) <= 16 * 2 ** -20


def test_tangents_are_not_rotated_in_place():
    q, _, dq, _, at, table = _inputs()
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="in place"):
            apply_rotary(forward_ad.make_dual(q, dq), None, at, table, in_place=True)


def test_a_table_that_wants_a_gradient_is_refused():
    q, k, _, _, at, table = _inputs()
    learnt = table.clone().requires_grad_()
    with pytest.raises(ValueError, match="cos_sin"):
        apply_rotary(q, k, at, learnt)
    with pytest.raises(ValueError, match="cos_sin"):
        apply_rotary(q.clone().requires_grad_(), k, at, learnt)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="cos_sin"):
            apply_rotary(q, k, at, forward_ad.make_dual(table, table))
    want = apply_rotary(q, k, at, table)
    for got in (apply_rotary(q, k, at, learnt.detach()), _no_grad(q, k, at, learnt)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@torch.no_grad()
def _no_grad(q, k, at, table):
    return apply_rotary(q, k, at, table)


def test_rows_rotated_in_place_cannot_be_what_autograd_saved():
    q, k, _, _, at, table = _inputs()
    for rows in (0, 1):
        mine = [q.clone(), k.clone()]
        weight = torch.ones_like(mine[rows], requires_grad=True)
        loss = (weight * mine[rows]).sum()  # saves the rows for the weight's gradient
        apply_rotary(mine[0], mine[1], at, table, in_place=True)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_pools_written_by_an_append_cannot_be_what_autograd_saved():
    pools = [torch.ones(2, 2, 16, 64, device=DEV, dtype=torch.bfloat16) for _ in "kv"]
    k = torch.zeros(1, 2, 64, device=DEV, dtype=torch.bfloat16)
    table = torch.zeros(1, 2, device=DEV, dtype=torch.int32)
    at = torch.zeros(1, device=DEV, dtype=torch.int32)
    for pool in pools:
        weight = torch.ones_like(pool, requires_grad=True)
        loss = (weight * pool).sum()
        paged_append(k, k, *pools, table, at)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_inference_tensors_are_written_all_the_same():
    q, k, _, _, at, table = _inputs()
    want = apply_rotary(q, k, at, table)
    with torch.inference_mode():
        mine = [q.clone(), k.clone()]
        apply_rotary(*mine, at, table, in_place=True)
        assert torch.equal(mine[0], want[0]) and torch.equal(mine[1], want[1])
        pools = [torch.zeros(2, 2, 16, 64, device=DEV, dtype=torch.bfloat16) for _ in "kv"]
        row = torch.ones(1, 2, 64, device=DEV, dtype=torch.bfloat16)
        paged_append(row, row, *pools, torch.zeros(1, 2, device=DEV, dtype=torch.int32),
                     torch.zeros(1, device=DEV, dtype=torch.int32))
        assert float(pools[0].sum()) == 128.0 == float(pools[1].sum())
    apply_rotary(*mine, at, table, inverse=True, in_place=True)  # and outside of the mode
