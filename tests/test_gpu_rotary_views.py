"""Rotation of overlapping views (needs a B200).  Bounds of test_gpu_rotary.py."""

import pytest
import torch

from refinekv_b200 import apply_rotary, rotary_table
from test_gpu_rotary import _normal, assert_rotated, rotate64

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("shape,strides", [
    ((3, 2, 64), (200, 1, 1)),    # heads that are one element apart
    ((5, 4, 64), (1, 80, 1)),     # tokens that are one element apart
    ((4, 3, 64), (0, 0, 1)),
    ((6, 3, 64), (64, 32, 1)),    # heads that overlap by half
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_overlapping_views_are_rotated_into_rows_of_their_own(shape, strides, dtype):
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = _normal(gen, 2000, dtype=dtype).as_strided(shape, strides)
    table = rotary_table(32, 50)
    at = torch.randint(0, 50, shape[:1], generator=gen, device=DEV)
    got, got_key = apply_rotary(x, x, at, table)
    assert got.shape == x.shape
    assert_rotated(got, *rotate64(x, at, table))
    assert torch.equal(got_key, got)
