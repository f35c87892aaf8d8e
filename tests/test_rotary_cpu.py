"""Rotary tables, and the refusals of the paged operators before a device is touched (no GPU)."""

import math

import pytest
import torch

from refinekv_b200 import _native, apply_rotary, paged_append, paged_attention, rotary_table


@pytest.fixture(scope="module")
def lib():
    from conftest import native_build_module

    native_build_module().build()
    return _native.load()


def test_table_rows_are_cosines_then_sines():
    table = rotary_table(6, 70000, base=500.0, device="cpu")
    assert table.shape == (70000, 6) and table.dtype == torch.float32
    for p in (0, 1, 69999):
        for i in range(3):
            angle = p * 500.0 ** (-2 * i / 6)
            # an fp64 angle near 7e4 is off by 1.5e-11 at most, then one rounding to fp32
            assert abs(float(table[p, i]) - math.cos(angle)) <= 2 ** -24
            assert abs(float(table[p, 3 + i]) - math.sin(angle)) <= 2 ** -24


def _library_frequencies(kind, dim, base, scaling):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    config = LlamaConfig(hidden_size=dim, num_attention_heads=1, head_dim=dim,
                         max_position_embeddings=131072)
    config.rope_parameters = {"rope_theta": base, **scaling}
    return ROPE_INIT_FUNCTIONS[kind](config, "cpu")


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
], ids=lambda s: s["rope_type"])
def test_scaled_frequencies_match_the_model_library(scaling):
    from refinekv_b200.rotary import _frequencies

    got, amplitude = _frequencies(128, 500000.0, scaling)
    want, want_amplitude = _library_frequencies(scaling["rope_type"], 128, 500000.0, scaling)
    # the library works in fp32: a power and a few products, 2^-23 each
    torch.testing.assert_close(got, want.double(), rtol=2 ** -19, atol=0)
    assert abs(amplitude - want_amplitude) <= 1e-6
    table = rotary_table(128, 4, base=500000.0, scaling=scaling, device="cpu")
    want_row = torch.cat([(3 * got).cos(), (3 * got).sin()]) * amplitude
    torch.testing.assert_close(table[3].double(), want_row, rtol=2 ** -23, atol=0)


def test_ntk_slows_the_slowest_pair_by_the_factor():
    from refinekv_b200.rotary import _frequencies

    plain, _ = _frequencies(64, 10000.0, None)
    scaled, amplitude = _frequencies(64, 10000.0, {"type": "ntk", "factor": 4.0})
    assert amplitude == 1.0 and float(scaled[0]) == 1.0
    assert abs(float(plain[-1] / scaled[-1]) - 4.0) <= 1e-9


@pytest.mark.parametrize("kwargs,match", [
    (dict(rotary_dim=5), "even"), (dict(positions=0), "positions"), (dict(base=1.0), "base"),
    (dict(scaling={"type": "linear"}), "factor"), (dict(scaling={"type": "spiral", "factor": 2}), "type"),
    (dict(scaling={"type": "linear", "factor": 0.5}), "factor"),
    (dict(scaling={"type": "yarn", "factor": 2.0}), "original_max"),
])
def test_bad_tables_are_refused(kwargs, match):
    with pytest.raises(ValueError, match=match):
        rotary_table(**{"rotary_dim": 8, "positions": 4, "device": "cpu", **kwargs})


def test_cpu_tensors_are_refused():
    x = torch.zeros(3, 2, 64)
    at, table = torch.zeros(3, dtype=torch.int32), torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        apply_rotary(x, None, at, table)
    with pytest.raises(ValueError, match="query must have shape"):
        apply_rotary(x[0], None, at, table)
    pool = torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_append(x, x, pool, pool, torch.zeros(3, 2, dtype=torch.int32), at)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention(x, pool, pool, torch.zeros(3, 2, dtype=torch.int32), at)
    with pytest.raises(ValueError, match="layout"):
        paged_append(x, x, pool, pool, torch.zeros(3, 2, dtype=torch.int32), at, layout="HDN")


ROTARY_FIELDS = ("query", "key", "query_out", "key_out", "positions", "cos_sin", *["qs"] * 3,
                 *["ks"] * 3, *["qos"] * 3, *["kos"] * 3, *["ps"] * 2, "positions_i64",
                 "table_rows", "table_stride", "batch", "tokens", "query_heads", "key_heads",
                 "head_dim", "rotary_dim", "dtype", "interleaved", "inverse")
APPEND_FIELDS = ("key", "value", "query", "query_out", "key_pool", "value_pool", "page_table",
                 "sequence_ids", "positions", "cos_sin", "status", *["ks"] * 2, *["vs"] * 2,
                 *["qs"] * 2, *["qos"] * 2, *["kps"] * 3, *["vps"] * 3, "page_table_stride",
                 "sequences", "table_blocks", "pool_pages", "block_size", "tokens", "query_heads",
                 "kv_heads", "head_dim", "rotary_dim", "table_rows", "table_stride", "dtype",
                 "positions_i64", "interleaved")


PAGED_FIELDS = ("query", "output", "lse", "key_pool", "value_pool", "page_table", "lengths",
                "workspace", "workspace_size", *["qs"] * 2, *["kps"] * 3, *["vps"] * 3,
                "page_table_stride", "sequences", "table_blocks", "pool_pages", "block_size",
                "kv_heads", "group", "head_dim", "query_dtype", "window", "scale")


def test_packed_arguments_have_the_headers_fields():
    """The packed structs count every 8-byte field of the header's declarations, in its order."""
    import pathlib
    import re

    header = (pathlib.Path(__file__).parents[1] / "include" / "refinekv_b200.h").read_text()
    for name, packer, fields in (("rotary", _native.ROTARY_ARGS, ROTARY_FIELDS),
                                 ("append", _native.APPEND_ARGS, APPEND_FIELDS),
                                 ("paged", _native.PAGED_ARGS, PAGED_FIELDS)):
        body = re.search(r"typedef struct rkv_%s_args \{(.*?)\}" % name, header, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = []
        for field in filter(None, (f.strip() for f in body.split(";"))):
            word, count = re.search(r"(\w+)(?:\[(\d)\])?$", field).groups()
            names += [word] * int(count or 1)
        assert packer.size == 8 * len(names) == 8 * len(fields)
        for have, want in zip(fields, names):
            assert have == want or want.endswith("_strides"), (have, want)


def _rotary(lib, **change):
    values = dict(query=16, query_out=16, positions=16, cos_sin=16, qs=128, qos=128, table_rows=4,
                  table_stride=64, batch=1, tokens=2, query_heads=2, head_dim=64, rotary_dim=64)
    values.update(change)
    return lib.rkv_rotary(_native.ROTARY_ARGS.pack(*[values.get(f, 0) for f in ROTARY_FIELDS]),
                          None)


@pytest.mark.parametrize("change,code", [
    (dict(query=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(positions=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(cos_sin=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(table_rows=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(table_stride=32), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(rotary_dim=66), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(rotary_dim=31), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(head_dim=63), _native.RKV_ERR_UNSUPPORTED),
    (dict(head_dim=1026), _native.RKV_ERR_UNSUPPORTED),
    (dict(tokens=1 << 31), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(batch=1 << 20, tokens=1 << 20), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(tokens=-1), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(dtype=7), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(query=17), _native.RKV_ERR_ALIGNMENT),
    (dict(cos_sin=18), _native.RKV_ERR_ALIGNMENT),
    (dict(tokens=0), _native.RKV_OK),
])
def test_rotary_entry_point_refuses_before_touching_a_device(lib, change, code):
    assert _rotary(lib, **change) == code
    assert bool(lib.rkv_last_error()) == (code != _native.RKV_OK)
    assert lib.rkv_rotary(None, None) == _native.RKV_ERR_INVALID_ARGUMENT


def _append(lib, **change):
    values = dict(key=16, value=16, key_pool=16, value_pool=16, page_table=16, positions=16,
                  ks=128, vs=128, kps=4096, vps=4096, page_table_stride=2, sequences=2,
                  table_blocks=2, pool_pages=4, block_size=32, tokens=2, kv_heads=2, head_dim=64)
    values.update(change)
    return lib.rkv_paged_append(
        _native.APPEND_ARGS.pack(*[values.get(f, 0) for f in APPEND_FIELDS]), None)


@pytest.mark.parametrize("change,code", [
    (dict(key=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(page_table=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(query_heads=2), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(cos_sin=16, rotary_dim=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(block_size=48), _native.RKV_ERR_UNSUPPORTED),
    (dict(head_dim=80), _native.RKV_ERR_UNSUPPORTED),
    (dict(kv_heads=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(pool_pages=-1), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(value_pool=17), _native.RKV_ERR_ALIGNMENT),
    (dict(tokens=0), _native.RKV_OK),
])
def test_append_entry_point_refuses_before_touching_a_device(lib, change, code):
    assert _append(lib, **change) == code
    assert lib.rkv_paged_append(None, None) == _native.RKV_ERR_INVALID_ARGUMENT


def _attend(lib, **change):
    values = dict(query=16, output=16, key_pool=16, value_pool=16, page_table=16, lengths=16,
                  workspace=256, workspace_size=1 << 30, qs=128, kps=4096, vps=4096,
                  page_table_stride=2, sequences=2, table_blocks=2, pool_pages=4, block_size=32,
                  kv_heads=2, group=4, head_dim=64, scale=0.125)
    values.update(change)
    return lib.rkv_paged_attention(
        _native.PAGED_ARGS.pack(*[values.get(f, 0) for f in PAGED_FIELDS]), None)


@pytest.mark.parametrize("change,code", [
    (dict(query=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(lengths=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(key_pool=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(pool_pages=0), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(window=-1), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(table_blocks=1 << 31), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(query_dtype=2), _native.RKV_ERR_INVALID_ARGUMENT),
    (dict(group=17), _native.RKV_ERR_UNSUPPORTED),
    (dict(group=0), _native.RKV_ERR_UNSUPPORTED),
    (dict(head_dim=288), _native.RKV_ERR_UNSUPPORTED),
    (dict(block_size=8), _native.RKV_ERR_UNSUPPORTED),
    (dict(sequences=4097), _native.RKV_ERR_UNSUPPORTED),
    (dict(workspace=0), _native.RKV_ERR_WORKSPACE),
    (dict(workspace_size=16), _native.RKV_ERR_WORKSPACE),
    (dict(query=24), _native.RKV_ERR_ALIGNMENT),
    (dict(kps=100), _native.RKV_ERR_ALIGNMENT),
    (dict(sequences=0), _native.RKV_OK),
])
def test_attention_entry_point_refuses_before_touching_a_device(lib, change, code):
    assert _attend(lib, **change) == code
    assert lib.rkv_paged_attention(None, None) == _native.RKV_ERR_INVALID_ARGUMENT
