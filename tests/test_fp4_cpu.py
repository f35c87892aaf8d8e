"""Pools of 4 bits: what the C entries and the package refuse before they touch a device (no GPU)."""

import pytest
import torch

import fp4_helpers as fp4
from refinekv_b200 import _native, fp4_pool, paged_append, paged_read


@pytest.fixture(scope="module")
def lib():
    from conftest import native_build_module

    native_build_module().build()
    return _native.load()


def _append_args(**kw):
    names = ("key value query query_out key_pool value_pool page_table sequence_ids positions "
             "cos_sin status ks0 ks1 vs0 vs1 qs0 qs1 os0 os1 kp0 kp1 kp2 vp0 vp1 vp2 table_stride "
             "sequences table_blocks pages block tokens query_heads kv_heads dim rotary rows "
             "row_stride dtype i64 interleaved key_scale value_scale").split()
    base = dict.fromkeys(names, 0)
    slab = 16 * 36
    base.update(key=16, value=16, key_pool=16, value_pool=16, page_table=16, positions=16, ks0=128,
                ks1=64, vs0=128, vs1=64, kp0=2 * slab, kp1=slab, vp0=2 * slab, vp1=slab,
                table_stride=4, sequences=2, table_blocks=4, pages=8, block=16, tokens=2, kv_heads=2,
                dim=64)
    return _native.APPEND_FP4_ARGS.pack(*{**base, **kw}.values())


@pytest.mark.parametrize("change,code,message", [
    (dict(tokens=-1), 1, b"out of range"),
    (dict(kv_heads=0), 1, b"out of range"),
    (dict(dim=80), 2, b"head_dim"),
    (dict(block=8), 2, b"block_size"),
    (dict(dtype=2), 1, b"dtype"),
    (dict(key=0), 1, b"non-null"),
    (dict(query_heads=4), 1, b"query"),
    (dict(query_heads=-1), 1, b"query heads"),
    (dict(cos_sin=16, rotary=63, rows=4, row_stride=64), 1, b"rotary_dim"),
    (dict(cos_sin=16, rotary=128, rows=4, row_stride=128), 1, b"rotary_dim"),
    (dict(cos_sin=16, rotary=64, rows=0, row_stride=64), 1, b"cos_sin"),
    (dict(cos_sin=18, rotary=64, rows=4, row_stride=64), 3, b"aligned"),
    (dict(key=17), 3, b"rows"),
    (dict(positions=18), 3, b"positions"),
    (dict(key_scale=18), 3, b"scales"),
    (dict(key_pool=24), 3, b"16 bytes"),
    (dict(kp1=16 * 36 + 8), 3, b"16 bytes"),
    (dict(vp0=40), 3, b"16 bytes"),
])
def test_append_refuses(lib, change, code, message):
    assert lib.rkv_paged_append_fp4(_append_args(**change), None) == code
    assert message in lib.rkv_last_error()


def test_nothing_to_append_is_nothing_done(lib):
    assert lib.rkv_paged_append_fp4(_append_args(tokens=0), None) == 0
    assert lib.rkv_paged_append_fp4(None, None) == 1


def _read_args(**kw):
    names = ("key_pool value_pool key_out value_out page_table sequence_ids positions status "
             "key_scale value_scale kp0 kp1 kp2 vp0 vp1 vp2 ko0 ko1 vo0 vo1 table_stride sequences "
             "table_blocks pages block tokens kv_heads dim pool_dtype dtype i64").split()
    base = dict.fromkeys(names, 0)
    slab = 16 * 36
    base.update(key_pool=16, value_pool=16, key_out=16, value_out=16, page_table=16, positions=16,
                kp0=2 * slab, kp1=slab, vp0=2 * slab, vp1=slab, ko0=128, ko1=64, vo0=128, vo1=64,
                table_stride=4, sequences=2, table_blocks=4, pages=8, block=16, tokens=2, kv_heads=2,
                dim=64, pool_dtype=2)
    return _native.READ_ARGS.pack(*{**base, **kw}.values())


@pytest.mark.parametrize("change,code,message", [
    (dict(tokens=1 << 31), 1, b"out of range"),
    (dict(dim=272), 2, b"head_dim"),
    (dict(block=128), 2, b"block_size"),
    (dict(pool_dtype=1), 1, b"bf16 or fp4"),
    (dict(dtype=2), 1, b"bf16 or fp4"),
    (dict(pool_dtype=0, kp2=64, vp2=64, key_scale=16), 1, b"scales"),
    (dict(value_out=0), 1, b"non-null"),
    (dict(status=18), 3, b"status"),
    (dict(key_pool=8), 3, b"16 bytes"),
    (dict(pool_dtype=0, kp2=60), 3, b"16 bytes"),
    (dict(ko0=4), 3, b"16 bytes"),
])
def test_read_refuses(lib, change, code, message):
    assert lib.rkv_paged_read(_read_args(**change), None) == code
    assert message in lib.rkv_last_error()


def test_the_package_refuses_cpu_tensors_and_odd_pools():
    pool = fp4_pool(2, 1, 16, 32, device="cpu")
    assert pool.shape == (2, 1, 16, 18) and not bool(pool.any())
    table = torch.zeros(1, 2, dtype=torch.int32)
    row, at = torch.zeros(1, 1, 32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_append(row, row, pool, pool, table, at)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_read(pool, pool, table, at)
    with pytest.raises(ValueError, match="HND"):
        paged_read(pool, pool, table, at, layout="NHD")
    for bad in ((-1, 1, 16, 32), (1, 0, 16, 32), (1, 1, 24, 32), (1, 1, 16, 48)):
        with pytest.raises(ValueError):
            fp4_pool(*bad, device="cpu")


def test_the_definition_used_by_the_tests_is_torchs_e4m3():
    bits = torch.arange(0x7f, dtype=torch.uint8)
    assert torch.equal(bits.view(torch.float8_e4m3fn).double(), fp4.SCALES)
    # ties of a bf16 block: amax 6 t with t between two scales, quotients between two codes
    x = torch.tensor([6.0 * 1.0625] + [1.25 * 1.0, 1.75, 0.25, 0.75, 2.5, 3.5, 5.0] + [0.0] * 8)
    codes, scales = fp4.quantise(x)
    assert scales.tolist() == [0x38]  # 1.0625 lies between 1 and 1.125: the even one
    assert fp4.values(codes, scales)[:8].tolist() == [6.0, 1.0, 2.0, 0.0, 1.0, 2.0, 4.0, 4.0]
