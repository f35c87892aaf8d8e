"""Rotary positions against the formula in 64 bits (needs a B200).

Bounds, from the kernel's roundings: with u = 2^-24 each rotated channel
a c - b s takes two rounded products and one rounded sum, so it is within
2 u (|a c| + |b s|) of the exact value to first order; 2^-22 covers it.  A
bf16 result adds half a unit in its last place: 2^(e - 8) for a result in
[2^e, 2^(e + 1)), whose bf16 neighbours are 2^(e - 7) apart.
"""

import pytest
import torch

from refinekv_b200 import apply_rotary, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rotate64(x, positions, table, interleaved=False, sign=1.0):
    """The rotation in fp64, and the sum of the magnitudes that enter each channel."""
    r = table.shape[1]
    row = table.double()[positions.long()].unsqueeze(-2)
    c, s = row[..., : r // 2], sign * row[..., r // 2:]
    x = x.double()
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), x.abs()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = (a * c).abs() + (b * s).abs()
    size[..., second] = (b * c).abs() + (a * s).abs()
    return y, size


def assert_rotated(got, want, size):
    tol = size * 2 ** -22
    if got.dtype == torch.bfloat16:
        half_ulp = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 1 - 8)
        tol = tol * 1.01 + half_ulp + 1e-38
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


@pytest.mark.parametrize("lead,hq,hk,dim,rotary", [
    ((1,), 32, 8, 128, 128),
    ((37,), 28, 4, 128, 64),
    ((5,), 3, 0, 80, 40),      # 20 pairs: no whole 16-byte pieces
    ((300,), 1, 2, 96, 96),
    ((2, 17), 6, 3, 64, 32),
    ((3, 1), 1, 1, 2, 2),
    ((4,), 2, 1, 256, 250),
    ((2,), 70, 1, 1024, 1024),
    ((9,), 5, 1, 24, 16),      # eight copied channels: no multiple of 16
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_matches_the_formula(lead, hq, hk, dim, rotary, dtype, interleaved):
    gen = torch.Generator(device=DEV).manual_seed(dim + rotary)
    table = rotary_table(rotary, 1000, scaling={"type": "yarn", "factor": 4.0,
                                                "original_max_position_embeddings": 256})
    q = _normal(gen, *lead, hq, dim, dtype=dtype)
    k = _normal(gen, *lead, hk, dim, dtype=dtype) if hk else None
    at = torch.randint(0, 1000, lead, generator=gen, device=DEV,
                       dtype=torch.int64 if interleaved else torch.int32)
    at.view(-1)[0] = 999
    got_q, got_k = apply_rotary(q, k, at, table, interleaved=interleaved)
    assert got_q.dtype == dtype and got_q.shape == q.shape
    assert_rotated(got_q, *rotate64(q, at, table, interleaved))
    if hk:
        assert_rotated(got_k, *rotate64(k, at, table, interleaved))
    else:
        assert got_k is None
    assert torch.equal(got_q[..., rotary:], q[..., rotary:])
    back, _ = apply_rotary(q, None, at, table, interleaved=interleaved, inverse=True)
    assert_rotated(back, *rotate64(q, at, table, interleaved, -1.0))
    mine, mine_k = apply_rotary(q.clone(), None if k is None else k.clone(), at, table,
                                interleaved=interleaved, in_place=True)
    assert torch.equal(mine, got_q) and (k is None or torch.equal(mine_k, got_k))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,rotary", [(torch.bfloat16, 96), (torch.bfloat16, 20),
                                          (torch.float32, 96), (torch.float32, 20)])
def test_rotation_has_the_bits_of_the_fp32_formula(dtype, rotary, interleaved):
    """Each product and sum is rounded by itself: the elementwise formula, bit for bit."""
    gen = torch.Generator(device=DEV).manual_seed(rotary)
    table = rotary_table(rotary, 5000, scaling={"type": "yarn", "factor": 4.0,
                                                "original_max_position_embeddings": 1024})
    q = _normal(gen, 200, 6, 128, dtype=dtype)
    at = torch.randint(0, 5000, (200,), generator=gen, device=DEV)
    row = table[at][:, None]
    c, s = row[..., : rotary // 2], row[..., rotary // 2:]
    x = q.float()
    first = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    second = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    for sign in (1.0, -1.0):
        want = x.clone()
        a, b = x[..., first], x[..., second]
        want[..., first] = a * c - b * (s * sign)
        want[..., second] = b * c + a * (s * sign)
        got, _ = apply_rotary(q, None, at, table, interleaved=interleaved, inverse=sign < 0)
        assert torch.equal(got, want.to(dtype))


def test_strides_of_models_and_servers():
    gen = torch.Generator(device=DEV).manual_seed(1)
    table = rotary_table(64, 500)
    at = torch.randint(0, 500, (2, 33), generator=gen, device=DEV)
    # (batch, heads, tokens, dim), as models keep it; the result keeps that layout
    q, k = _normal(gen, 2, 5, 33, 64), _normal(gen, 2, 3, 33, 64)
    got_q, got_k = apply_rotary(q.transpose(1, 2), k.transpose(1, 2), at, table)
    assert got_q.transpose(1, 2).is_contiguous()
    assert_rotated(got_q, *rotate64(q.transpose(1, 2), at, table))
    assert_rotated(got_k, *rotate64(k.transpose(1, 2), at, table))
    # one projection cut into queries and keys, rotated in place
    both = _normal(gen, 66, 8 * 64)
    want = rotate64(both.view(66, 8, 64)[:, :6], at.view(-1), table)
    tail = both[:, 6 * 64:].clone()
    apply_rotary(both.view(66, 8, 64)[:, :4], both.view(66, 8, 64)[:, 4:6], at.view(-1), table,
                 in_place=True)
    assert_rotated(both.view(66, 8, 64)[:, :6], *want)
    assert torch.equal(both[:, 6 * 64:], tail)
    # rows that start at odd elements, rows with a stride in the head dim, shared heads, shared
    # positions, a table wider than its rows
    odd = _normal(gen, 7, 3, 65)[..., 1:]
    assert_rotated(apply_rotary(odd, None, at.view(-1)[:7], table)[0],
                   *rotate64(odd, at.view(-1)[:7], table))
    skewed = _normal(gen, 7, 64, 3).transpose(1, 2)
    assert_rotated(apply_rotary(skewed, None, at.view(-1)[:7], table)[0],
                   *rotate64(skewed, at.view(-1)[:7], table))
    shared = _normal(gen, 7, 1, 64).expand(7, 4, 64)
    assert_rotated(apply_rotary(shared, None, at.view(-1)[:7], table)[0],
                   *rotate64(shared, at.view(-1)[:7], table))
    same = at[:1, :5].expand(2, 5)
    batch = _normal(gen, 2, 5, 2, 64)
    assert_rotated(apply_rotary(batch, None, same, table)[0], *rotate64(batch, same, table))
    wide = torch.full((500, 70), float("nan"), device=DEV)
    wide[:, 1:65] = table
    assert torch.equal(apply_rotary(batch, None, same, wide[:, 1:65])[0],
                       apply_rotary(batch, None, same, table)[0])


def test_positions_outside_the_table_give_nan_in_their_own_rows():
    gen = torch.Generator(device=DEV).manual_seed(2)
    table = rotary_table(32, 10)
    q = _normal(gen, 4, 2, 64, dtype=torch.float32)
    at = torch.tensor([3, 10, -1, 1 << 40], device=DEV)
    got, _ = apply_rotary(q, None, at, table)
    assert_rotated(got[:1], *rotate64(q[:1], at[:1], table))
    assert bool(got[1:, :, :32].isnan().all()) and torch.equal(got[1:, :, 32:], q[1:, :, 32:])


def test_empty_inputs_and_infinities():
    table = rotary_table(8, 4)
    q, k = torch.empty(0, 3, 8, device=DEV), torch.empty(0, 1, 8, device=DEV)
    at = torch.empty(0, device=DEV, dtype=torch.int32)
    got = apply_rotary(q, k, at, table)
    assert got[0].shape == q.shape and got[1].shape == k.shape
    q = torch.ones(2, 1, 8, device=DEV)
    q[0, 0, 1], q[1, 0, 2] = float("inf"), float("nan")
    at = torch.tensor([1, 1], device=DEV)
    got = apply_rotary(q, None, at, table)[0]
    want = rotate64(q, at, table)[0].float()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_is_the_inverse_rotation(interleaved, dtype):
    gen = torch.Generator(device=DEV).manual_seed(3)
    table = rotary_table(48, 300, scaling={"type": "yarn", "factor": 2.0,
                                           "original_max_position_embeddings": 128})
    at = torch.randint(0, 300, (29,), generator=gen, device=DEV)
    q = _normal(gen, 29, 6, 64, dtype=dtype).requires_grad_()
    k1 = _normal(gen, 29, 1, 64, dtype=dtype).requires_grad_()
    gq, gk = _normal(gen, 29, 6, 64, dtype=dtype), _normal(gen, 29, 3, 64, dtype=dtype)
    out = apply_rotary(q, k1.expand(29, 3, 64), at, table, interleaved=interleaved)
    torch.autograd.backward(out, (gq, gk))
    assert_rotated(q.grad, *rotate64(gq, at, table, interleaved, -1.0))
    # a key shared by three heads collects their gradients: three rounded rows, two more sums
    want, size = rotate64(gk, at, table, interleaved, -1.0)
    eps = 2 ** -8 if dtype == torch.bfloat16 else 2 ** -23
    off = (k1.grad.double() - want.sum(1, keepdim=True)).abs()
    assert bool((off <= 3 * (2 ** -22 + eps) * size.sum(1, keepdim=True)).all())
    # unused outputs and a second derivative
    only = _normal(gen, 29, 6, 64, dtype=torch.float32).requires_grad_()
    y, none = apply_rotary(only, None, at, table, interleaved=interleaved)
    assert none is None
    (first,) = torch.autograd.grad(y.square().sum(), only, create_graph=True)
    (second,) = torch.autograd.grad(first.sum(), only)
    # sum of squares of a rotation scaled by a: gradient 2 a^2 x, whose sum has gradient 2 a^2
    amplitude = float((table[0, 0]).double()) ** 2
    scale = torch.ones(64, device=DEV, dtype=torch.float64)
    scale[:48] = amplitude
    assert float((first.detach().double() - 2 * scale * only.detach().double()).abs().max()) <= 1e-4
    assert float((second.double() - 2 * scale).abs().max()) <= 1e-4


def test_gradient_against_differences():
    gen = torch.Generator(device=DEV).manual_seed(4)
    table = rotary_table(32, 100)
    at = torch.randint(0, 100, (11,), generator=gen, device=DEV)
    x = _normal(gen, 11, 3, 32, dtype=torch.float32).requires_grad_()
    g, v = (_normal(gen, 11, 3, 32, dtype=torch.float32) for _ in range(2))
    apply_rotary(x, None, at, table)[0].backward(g)
    with torch.no_grad():  # the map is linear: a step of any size gives the derivative
        ahead, behind = (apply_rotary(x + h * v, None, at, table)[0].double() for h in (1, -1))
    slope = float((g.double() * (ahead - behind) / 2).sum())
    # every entry of either side is within 2^-21 of values whose size is below 12
    assert abs(slope - float((x.grad.double() * v.double()).sum())) <= 1056 * 12 * 5 * 2 ** -21


def test_other_streams_and_graphs():
    gen = torch.Generator(device=DEV).manual_seed(5)
    table = rotary_table(128, 4096)
    q, k = _normal(gen, 64, 32, 128), _normal(gen, 64, 8, 128)
    at = torch.arange(64, device=DEV)
    want = apply_rotary(q, k, at, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = at + 0
        got = apply_rotary(q, k, late, table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_rotary(q, k, at, table)
    at += 100
    graph.replay()
    fresh = apply_rotary(q, k, at, table)
    assert torch.equal(out[0], fresh[0]) and torch.equal(out[1], fresh[1])


def test_refusals():
    table = rotary_table(64, 10)
    q = torch.zeros(3, 2, 64, device=DEV)
    at = torch.zeros(3, device=DEV, dtype=torch.int32)
    for bad, error in [
        (lambda: apply_rotary(q.half(), None, at, table), TypeError),
        (lambda: apply_rotary(q, q.bfloat16(), at, table), TypeError),
        (lambda: apply_rotary(q, None, at.float(), table), TypeError),
        (lambda: apply_rotary(q, None, at, table.double()), TypeError),
        (lambda: apply_rotary(q, None, at[:2], table), ValueError),
        (lambda: apply_rotary(q, None, at.cpu(), table), ValueError),
        (lambda: apply_rotary(q, q[:2], at, table), ValueError),
        (lambda: apply_rotary(q[..., :32], None, at, table), ValueError),  # 64 rotary channels
        (lambda: apply_rotary(q, None, at, table.cpu()), ValueError),
        (lambda: apply_rotary(q, None, at, table[:0]), ValueError),
        (lambda: apply_rotary(q[:, :1].expand(3, 2, 64), None, at, table, in_place=True), ValueError),
        (lambda: apply_rotary(q.transpose(1, 2)[:, :2, :2], None, at, table[:, :2],
                              in_place=True), ValueError),
        (lambda: apply_rotary(q.clone().requires_grad_(), None, at, table, in_place=True),
         ValueError),
    ]:
        with pytest.raises(error):
            bad()
