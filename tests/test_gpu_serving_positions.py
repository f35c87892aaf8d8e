"""The serving example with a prompt longer than a few thousand tokens (needs a B200)."""

import pytest
import torch

from test_gpu_serving_example import _example

pytestmark = pytest.mark.gpu


def test_the_rotation_table_covers_the_longest_request():
    ex = _example()
    model = ex.Decoder(layers=2, dense=1)
    gen = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 512, (n,), generator=gen) for n in (4095, 5000, 3)]
    server = ex.Server(model, prompts, 4, ex.rkv.RefineKVConfig(eps=0.0))
    tokens, logits = server.generate()
    assert bool(logits.isfinite().all()) and server.healthy()
    assert server.cos_sin.shape[0] >= 5004


def test_a_table_too_short_for_a_request_is_refused():
    ex = _example()
    model = ex.Decoder(layers=1, dense=1)
    with pytest.raises(ValueError, match="positions"):
        ex.Server(model, [torch.zeros(30, dtype=torch.int64)], 4, positions=32)
