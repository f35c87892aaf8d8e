"""The rotation next to torch's automatic differentiation (needs a B200).

Rotated values have the bounds of test_gpu_rotary.py.
"""

import pytest
import torch
from torch.autograd import forward_ad

from refinekv_b200 import apply_rotary, rotary_table
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
