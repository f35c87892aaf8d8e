"""Integer arrays that are not aligned to their elements are refused before a device is touched
(no GPU): a kernel's load from one would fault."""

import pytest

from refinekv_b200 import _native
from test_rotary_cpu import _append, _attend, _rotary, lib  # noqa: F401  (lib: the fixture)


@pytest.mark.parametrize("change", [dict(positions=18), dict(positions=20, positions_i64=1)])
def test_rotary(lib, change):  # noqa: F811
    assert _rotary(lib, **change) == _native.RKV_ERR_ALIGNMENT
    assert lib.rkv_last_error()


@pytest.mark.parametrize("change", [
    dict(positions=18), dict(positions=20, positions_i64=1), dict(page_table=17),
    dict(sequence_ids=22), dict(status=21),
])
def test_append(lib, change):  # noqa: F811
    assert _append(lib, **change) == _native.RKV_ERR_ALIGNMENT
    assert lib.rkv_last_error()


@pytest.mark.parametrize("change", [dict(page_table=18), dict(lengths=17), dict(lse=30)])
def test_attention(lib, change):  # noqa: F811
    assert _attend(lib, **change) == _native.RKV_ERR_ALIGNMENT
    assert lib.rkv_last_error()
