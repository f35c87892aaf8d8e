"""Rotary tables from whole rope-scaling dictionaries, as model configurations keep them (no GPU)."""

import pytest
import torch

from refinekv_b200 import rotary_table
from refinekv_b200.rotary import _frequencies
from test_rotary_cpu import _library_frequencies

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize("keys", [
    {"mscale": 0.707, "mscale_all_dim": 0.707},
    {"mscale": 1.0, "mscale_all_dim": 0.707},
    {"mscale": 1.0, "mscale_all_dim": 1.0, "beta_fast": 32, "beta_slow": 1},
    {"mscale": 0.707},            # one of the two alone has no effect
    {"mscale_all_dim": 0.707},
    {"mscale": 0.707, "mscale_all_dim": 0.0},
    {"mscale": 0.707, "mscale_all_dim": 0.5, "attention_factor": 1.25},
    {"attention_factor": 1.0},
    {"beta_fast": 16, "beta_slow": 2},
    {"truncate": False},
])
def test_yarn_amplitude_follows_the_configuration(keys):
    scaling = {**YARN, **keys}
    got, amplitude = _frequencies(64, 10000.0, scaling)
    want, want_amplitude = _library_frequencies("yarn", 64, 10000.0, scaling)
    # the library works in fp32: a power and a few products, 2^-23 each
    torch.testing.assert_close(got, want.double(), rtol=2 ** -19, atol=0)
    assert abs(amplitude - want_amplitude) <= 1e-6
    row = rotary_table(64, 4, scaling=scaling, device="cpu")[0]  # cosines of 0, then sines
    torch.testing.assert_close(row[:32], torch.full((32,), want_amplitude), rtol=1e-6, atol=0)


LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


@pytest.mark.parametrize("scaling", [{"rope_type": "default"}, {"rope_type": "linear", "factor": 4.0},
                                     LLAMA3, YARN], ids=lambda s: s["rope_type"])
def test_the_base_may_be_in_the_dictionary(scaling):
    want = rotary_table(64, 50, base=500000.0, scaling=scaling, device="cpu")
    whole = {**scaling, "rope_theta": 500000.0}
    assert torch.equal(rotary_table(64, 50, scaling=whole, device="cpu"), want)
    assert torch.equal(rotary_table(64, 50, base=500000, scaling=whole, device="cpu"), want)
    assert torch.equal(rotary_table(64, 50, base=500000.0, device="cpu", scaling={
        **scaling, "rope_theta": None}), want)
    with pytest.raises(ValueError, match="rope_theta"):
        rotary_table(64, 50, base=10000.0, scaling=whole, device="cpu")
    with pytest.raises(ValueError, match="base"):
        rotary_table(64, 50, scaling={**scaling, "rope_theta": 1.0}, device="cpu")
    # without either: 10000
    assert torch.equal(rotary_table(64, 50, scaling=scaling, device="cpu"),
                       rotary_table(64, 50, base=10000.0, scaling=scaling, device="cpu"))


@pytest.mark.parametrize("scaling,match", [
    ({**YARN, "beta_fats": 16}, "beta_fats"),                      # misspelt
    ({**YARN, "low_freq_factor": 1.0}, "low_freq_factor"),         # another type's
    ({**LLAMA3, "mscale": 1.0}, "mscale"),
    ({"rope_type": "linear", "factor": 2.0, "short_factor": [1.0]}, "short_factor"),
    ({"factor": 8.0}, "factor"),                                   # a factor without a type
    ({"full_attention": {"rope_type": "default"}}, "full_attention"),
    ({k: v for k, v in LLAMA3.items() if k != "low_freq_factor"}, "low_freq_factor"),
    ({k: v for k, v in LLAMA3.items() if k != "high_freq_factor"}, "high_freq_factor"),
    ({**LLAMA3, "high_freq_factor": None}, "high_freq_factor"),
    ({**LLAMA3, "high_freq_factor": 1.0}, "high_freq_factor"),     # no band between the two
    ({**YARN, "factor": None}, "factor"),
    ({**YARN, "original_max_position_embeddings": 0}, "original_max_position_embeddings"),
])
def test_keys_that_are_missing_or_not_understood_are_refused(scaling, match):
    with pytest.raises(ValueError, match=match):
        rotary_table(64, 4, scaling=scaling, device="cpu")


def test_absent_keys_may_be_none_and_harmless_ones_are_accepted():
    plain = rotary_table(64, 50, scaling=YARN, device="cpu")
    more = dict(YARN, mscale=None, beta_fast=None, attention_factor=None, type="yarn",
                partial_rotary_factor=0.5, max_position_embeddings=163840)
    assert torch.equal(rotary_table(64, 50, scaling=more, device="cpu"), plain)
    linear = {"type": "linear", "factor": 2.0}
    assert torch.equal(
        rotary_table(64, 50, device="cpu",
                     scaling={**linear, "original_max_position_embeddings": 4096}),
        rotary_table(64, 50, device="cpu", scaling=linear))
