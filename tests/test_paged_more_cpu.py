"""What the C entries of the attention with more to it and of the eviction refuse before they touch
a device (no GPU)."""

import math

import pytest

from refinekv_b200 import _native


@pytest.fixture(scope="module")
def lib():
    from conftest import native_build_module

    native_build_module().build()
    return _native.load()


def _more_args(**kw):
    names = ("query output lse key_pool value_pool page_table lengths workspace workspace_size qs0 qs1 "
             "kp0 kp1 kp2 vp0 vp1 vp2 table_stride sequences table_blocks pages block kv_heads group "
             "dim dtype window scale slopes key_scale value_scale weights scores scores_size ws0 ws1 "
             "width pool_dtype prefix softcap").split()
    base = dict.fromkeys(names, 0)
    slab = 16 * 36
    base.update(query=16, output=16, key_pool=16, value_pool=16, page_table=16, lengths=16,
                workspace=256, workspace_size=1 << 30, qs0=256, qs1=64, kp0=2 * slab, kp1=slab,
                vp0=2 * slab, vp1=slab, table_stride=4, sequences=2, table_blocks=4, pages=8, block=16,
                kv_heads=2, group=2, dim=64, pool_dtype=2, scale=0.125, softcap=0.0)
    return _native.PAGED_MORE_ARGS.pack(*{**base, **kw}.values())


@pytest.mark.parametrize("change,code,message", [
    (dict(pool_dtype=1), 1, b"bf16 or fp4"),
    (dict(pool_dtype=0, kp2=64, vp2=64, key_scale=16), 1, b"scales"),
    (dict(softcap=-1.0), 1, b"softcap"),
    (dict(softcap=math.nan), 1, b"softcap"),
    (dict(softcap=1e-60), 1, b"softcap"),
    (dict(softcap=1e-39), 1, b"softcap"),  # not a normal number
    (dict(softcap=1e60), 1, b"softcap"),
    (dict(prefix=-1), 1, b"prefix"),
    (dict(slopes=18), 3, b"slopes"),
    (dict(weights=18), 3, b"weights"),
    (dict(dim=80), 2, b"head_dim"),
    (dict(group=17), 2, b"group"),
    (dict(block=128), 2, b"block_size"),
    (dict(sequences=4097), 2, b"sequences"),
    (dict(key_pool=24), 3, b"16-byte"),
    (dict(vp1=16 * 36 + 8), 3, b"16-byte"),
    (dict(table_blocks=1 << 40), 1, b"page table"),
    (dict(workspace=0), 4, b"workspace"),
])
def test_attention_refuses(lib, change, code, message):
    assert lib.rkv_paged_attention_more(_more_args(**change), None) == code
    assert message in lib.rkv_last_error()


def test_no_sequences_are_nothing(lib):
    assert lib.rkv_paged_attention_more(_more_args(sequences=0), None) == 0
    assert lib.rkv_paged_attention_more(None, None) == 1


def _evict_args(**kw):
    names = ("key_pool value_pool page_table lengths lengths_out weights positions workspace "
             "workspace_size kp0 kp1 kp2 vp0 vp1 vp2 ws0 ws1 ps0 ps1 width position_width table_stride "
             "sequences table_blocks pages block kv_heads dim pool_dtype budget recent").split()
    base = dict.fromkeys(names, 0)
    slab = 16 * 36
    base.update(key_pool=16, value_pool=16, page_table=16, lengths=16, lengths_out=32, weights=16,
                workspace=256, workspace_size=1 << 20, kp0=2 * slab, kp1=slab, vp0=2 * slab, vp1=slab,
                ws0=128, ws1=64, width=64, table_stride=4, sequences=2, table_blocks=4, pages=8,
                block=16, kv_heads=2, dim=64, pool_dtype=2, budget=32, recent=4)
    return _native.EVICT_ARGS.pack(*{**base, **kw}.values())


@pytest.mark.parametrize("change,code,message", [
    (dict(dim=16), 2, b"head_dim"),
    (dict(block=48), 2, b"block_size"),
    (dict(kv_heads=0), 2, b"KV heads"),
    (dict(pool_dtype=1), 1, b"bf16 or fp4"),
    (dict(pages=-1), 1, b"pool sizes"),
    (dict(budget=0), 1, b"budget"),
    (dict(recent=33), 1, b"budget"),
    (dict(width=63), 1, b"weights"),
    (dict(positions=16, position_width=63), 1, b"positions"),
    (dict(lengths_out=0), 1, b"non-null"),
    (dict(lengths_out=16), 1, b"lengths_out"),
    (dict(key_pool=8), 3, b"16 bytes"),
    (dict(pool_dtype=0, kp2=36), 3, b"16 bytes"),
    (dict(weights=18), 3, b"aligned"),
    (dict(workspace=128), 4, b"workspace"),
    (dict(workspace_size=512), 4, b"workspace"),
])
def test_eviction_refuses(lib, change, code, message):
    assert lib.rkv_paged_evict(_evict_args(**change), None) == code
    assert message in lib.rkv_last_error()


def test_eviction_workspace(lib):
    size = lib.rkv_paged_evict_workspace_size
    assert lib.rkv_paged_evict(_evict_args(sequences=0), None) == 0
    assert lib.rkv_paged_evict(None, None) == 1
    assert size(2, 2, 64, 32) == 256 + 256 + 4 * 32 * 8
    assert size(2, 2, 64, 64) == size(2, 2, 64, 1 << 40) == 512
    assert size(2, 2, 64, 63) == 512 + 4 * 8
    for bad in ((-1, 2, 64, 32), (2, 0, 64, 32), (2, 2, -64, 32), (2, 2, 64, 0), (4097, 2, 64, 32)):
        assert size(*bad) == 0
