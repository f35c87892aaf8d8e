"""Serve prompts of different lengths from one page pool, dense and refined layers together.

    python refinekv-release_b200/examples/serve_page_pool.py [--prompts 700,95,1301] [--new 32]

A small random-weight decoder (attention layers only) runs the serving path a
host engine would: every layer keeps its keys and values in a pool of 32-token
pages, one page table is shared by the layers, and a request's pages come from
a free list.  Prefill rotates the prompt (``apply_rotary``), attends causally
and writes the rotated keys and the values to the pool (``paged_append``).  A
decode step is captured once as a CUDA graph and replayed while the sequences
grow:

* a dense layer appends the new token, rotated on the way, and attends over each
  sequence's own length of the pool (``paged_append``, ``paged_attention``);
* a refined layer reads the same pool through ``attach_page_pool``: the prompt's
  block summaries, built from the prompt's keys and values, decide which pages
  are read (``sparse_attention``); the generated tokens are its suffix.
"""

from __future__ import annotations

import argparse
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))
import refinekv_b200 as rkv  # noqa: E402

BLOCK = 32


class Decoder:
    """Random weights; ``dense`` layers first, refined layers after them."""

    def __init__(self, layers=2, dense=1, q_heads=8, kv_heads=2, dim=64, vocab=512, seed=0,
                 device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.hq, self.hk, self.dim, self.layers, self.dense = q_heads, kv_heads, dim, layers, dense
        width = q_heads * dim

        def weight(*shape):
            w = torch.randn(shape, generator=gen, device=device) * shape[0] ** -0.5
            return w.to(torch.bfloat16)

        self.embed = weight(vocab, width) * vocab ** 0.5
        self.qkv = [weight(width, (q_heads + 2 * kv_heads) * dim) for _ in range(layers)]
        self.out = [weight(width, width) for _ in range(layers)]
        self.head = weight(width, vocab)

    def project(self, layer, x):
        """(tokens, heads, dim) queries, keys and values: slices of one projection."""
        x = torch.nn.functional.rms_norm(x, x.shape[-1:])
        rows = (x @ self.qkv[layer]).unflatten(-1, (-1, self.dim))
        return rows.split([self.hq, self.hk, self.hk], dim=-2)

    def logits(self, x):
        return torch.nn.functional.rms_norm(x, x.shape[-1:]).float() @ self.head.float()


class Server:
    """``positions``: rows of the rotation table, by default as many as the longest request has."""

    def __init__(self, model: Decoder, prompts, new_tokens: int, config=None, positions=None):
        self.m, self.new, self.config = model, new_tokens, config or rkv.RefineKVConfig()
        dev = model.embed.device
        self.n = len(prompts)
        longest = max(map(len, prompts)) + new_tokens
        if positions is not None and positions < longest:
            raise ValueError(f"positions: the longest request has {longest} tokens")
        self.cos_sin = rkv.rotary_table(model.dim, positions or longest, device=dev)
        # Every request takes the pages of its prompt and its new tokens from the free list.
        need = [-(-(len(p) + new_tokens) // BLOCK) for p in prompts]
        free = torch.randperm(sum(need) + 1, device=dev).to(torch.int32)
        self.table = torch.zeros(self.n, max(need), device=dev, dtype=torch.int32)
        for i, count in enumerate(need):
            self.table[i, :count], free = free[:count], free[count:]
        shape = (sum(need) + 1, model.hk, BLOCK, model.dim)
        self.pools = [tuple(torch.zeros(shape, device=dev, dtype=torch.bfloat16) for _ in "kv")
                      for _ in range(model.layers)]
        self.workspaces = [{} for _ in range(model.layers)]
        last = [self._prefill(i, prompt.to(dev)) for i, prompt in enumerate(prompts)]
        self._summarise()
        # What a captured step reads and moves on: the last token, the length of each sequence
        # without it, and the generated tokens before it.
        self.tokens = torch.stack(last)
        self.lengths = torch.tensor([len(p) for p in prompts], device=dev, dtype=torch.int32)
        self.suffix = torch.zeros((), device=dev, dtype=torch.int32)

    def _prefill(self, slot, prompt):
        m, length = self.m, len(prompt)
        at = torch.arange(length, device=prompt.device, dtype=torch.int32)
        x = m.embed[prompt]
        self.prompt_kv = getattr(self, "prompt_kv", [[] for _ in range(m.layers)])
        for layer in range(m.layers):
            q, k, v = m.project(layer, x)
            q, k = rkv.apply_rotary(q, k, at, self.cos_sin)
            rkv.paged_append(k, v, *self.pools[layer], self.table, at,
                             sequence_ids=torch.full_like(at, slot),
                             workspace=self.workspaces[layer])
            if layer >= m.dense:
                self.prompt_kv[layer].append((k.transpose(0, 1), v.transpose(0, 1)))
            y = torch.nn.functional.scaled_dot_product_attention(
                *(r.transpose(0, 1)[None] for r in (q, k, v)), is_causal=True, enable_gqa=True)
            x = x + y[0].transpose(0, 1).flatten(1) @ m.out[layer]
        return m.logits(x[-1:]).argmax(-1)[0]

    def _summarise(self):
        """The refined layers' summaries, bound to the pool, and their suffix buffers."""
        m = self.m
        self.summaries, self.suffix_kv = {}, {}
        for layer in range(m.dense, m.layers):
            keys, values = zip(*self.prompt_kv[layer])
            summary = rkv.build_summary_batch(list(keys), list(values), self.config)
            self.summaries[layer] = rkv.attach_page_pool(
                summary, *self.pools[layer], self.table[:, :summary.num_blocks])
            shape = (self.n * m.hk, self.new, m.dim)
            self.suffix_kv[layer] = tuple(
                torch.zeros(shape, device=m.embed.device, dtype=torch.bfloat16) for _ in "kv")
        del self.prompt_kv

    def step(self):
        """One token for every sequence; writes the next tokens and returns the logits."""
        m = self.m
        x = m.embed[self.tokens]
        grown, seen = self.lengths + 1, self.suffix + 1
        for layer in range(m.layers):
            q, k, v = m.project(layer, x)
            ws = self.workspaces[layer]
            if layer < m.dense:
                q = rkv.paged_append(k, v, *self.pools[layer], self.table, self.lengths, query=q,
                                     cos_sin=self.cos_sin, workspace=ws)
                y = rkv.paged_attention(q, *self.pools[layer], self.table, grown, workspace=ws)
            else:
                q, k = rkv.apply_rotary(q, k, self.lengths, self.cos_sin)
                for buffer, rows in zip(self.suffix_kv[layer], (k, v)):
                    buffer.index_copy_(1, self.suffix.view(1).long(), rows.flatten(0, 1)[:, None])
                query = q.reshape(self.n * m.hk, m.hq // m.hk, 1, m.dim)
                y = rkv.sparse_attention(query, self.summaries[layer], *self.suffix_kv[layer],
                                         self.config, workspace=ws, suffix_length=seen).output
            x = x + y.reshape(self.n, -1) @ m.out[layer]
        logits = m.logits(x)
        self.tokens.copy_(logits.argmax(-1))
        self.lengths.copy_(grown)
        self.suffix.copy_(seen)
        return logits

    def generate(self):
        """(sequences, new tokens) greedy tokens and the logits after each of them."""
        tokens, logits = [self.tokens.clone()], [self.step().clone()]  # the warm-up is a real step
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = self.step()
        for _ in range(self.new - 1):
            tokens.append(self.tokens.clone())
            graph.replay()
            logits.append(out.clone())
        return torch.stack(tokens, 1), torch.stack(logits, 1)

    def healthy(self):
        return all(rkv.attention.device_status(ws) == 0 for ws in self.workspaces)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", default="700,95,1301", help="prompt lengths")
    ap.add_argument("--new", type=int, default=32, help="tokens to generate for each")
    args = ap.parse_args()
    model = Decoder()
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, model.embed.shape[0], (int(n),), generator=gen)
               for n in args.prompts.split(",")]
    server = Server(model, prompts, args.new)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    tokens, _ = server.generate()
    end.record()
    end.synchronize()
    for prompt, row in zip(prompts, tokens.tolist()):
        print(f"prompt of {len(prompt)} tokens -> {row[:12]} ...")
    print(f"{args.new} steps of {len(prompts)} sequences: {start.elapsed_time(end):.1f} ms "
          f"(capture included), healthy: {server.healthy()}")


if __name__ == "__main__":
    main()
