"""The page-pool serving example against the same decoder without cache, pages or kernels.

The reference runs the whole sequence through plain fp32 attention at once,
teacher-forced on the generated tokens.  The example keeps activations, keys
and values in bf16 (2^-8 each, through two layers), so its logits must agree to
2 % of their scale, as the adapter's decoders must, and its greedy tokens wherever the
reference's best logit leads by more than that.
"""

import importlib.util
import pathlib

import pytest
import torch

pytestmark = pytest.mark.gpu
EXAMPLE = (pathlib.Path(__file__).resolve().parents[1] / "refinekv-release_b200" / "examples"
           / "serve_page_pool.py")


def _example():
    spec = importlib.util.spec_from_file_location("serve_page_pool", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain_logits(model, tokens):
    length = len(tokens)
    half = model.dim // 2
    w = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = (torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * w)[:, None]
    c, s = angle.cos().float(), angle.sin().float()

    def turn(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    x = model.embed[tokens].float()
    seen = torch.ones(length, length, device="cuda", dtype=torch.bool).tril()
    for layer in range(model.layers):
        y = torch.nn.functional.rms_norm(x, x.shape[-1:])
        rows = (y @ model.qkv[layer].float()).unflatten(-1, (-1, model.dim))
        q, k, v = rows.split([model.hq, model.hk, model.hk], dim=-2)
        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(model.hq // model.hk, 1) for t in (k, v))
        scores = torch.einsum("qhd,khd->hqk", q, k) * model.dim ** -0.5
        p = scores.masked_fill(~seen, float("-inf")).softmax(-1)
        x = x + torch.einsum("hqk,khd->qhd", p, v).flatten(1) @ model.out[layer].float()
    return model.logits(x)


@pytest.mark.parametrize("dense", [2, 1, 0])
def test_served_tokens_match_the_plain_decoder(dense):
    ex = _example()
    model = ex.Decoder(layers=2, dense=dense)
    gen = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 512, (n,), generator=gen) for n in (61, 1, 200, 32)]
    # eps 0 refines every block: the refined layers are exact too
    server = ex.Server(model, prompts, 12, ex.rkv.RefineKVConfig(eps=0.0))
    tokens, logits = server.generate()
    assert server.healthy()
    assert tokens.shape == (4, 12) and server.lengths.tolist() == [len(p) + 12 for p in prompts]
    for i, prompt in enumerate(prompts):
        row = torch.cat([prompt.cuda(), tokens[i]])
        want = _plain_logits(model, row)
        scale = float(want.abs().max())
        got = logits[i]
        assert float((got - want[len(prompt):]).abs().max()) <= 0.02 * scale
        best = want[len(prompt) - 1:-1]
        chosen = best.gather(1, tokens[i][:, None])[:, 0]
        assert bool((best.amax(-1) - chosen <= 0.04 * scale).all())
