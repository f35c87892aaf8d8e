"""What is measured of the paged serving operators: rotary positions, appending to a page pool, paged attention.

``own`` False computes the operators in plain torch operations (32 bits, rounded once at the end), True calls
``refinekv_b200``.  Sequences keep their keys and values in a pool of pages; ``page_table[s, b]`` is the physical page of
logical block ``b`` of sequence ``s``; ``lengths`` are the sequences' tokens.  Rotation tables hold, per position, the
cosines and then the sines of the rotary channel pairs.
"""

import math
import pathlib
import sys

import torch

own = False

#: (query heads, KV heads, head dim) of the shapes drawn: Llama-3.1-8B, Qwen2.5-7B, and generic ones.
SHAPES = ((32, 8, 128), (28, 4, 128), (64, 8, 64), (16, 2, 256), (12, 4, 96), (8, 8, 128), (16, 1, 128))

#: Elements of the largest listed cache (t: sequences x tokens x KV heads x dim); a drawn one has no more.
MOST_CACHE = 16 * 32768 * 8 * 128


def listed():
    return [
        # One decoded token's queries and keys in one layer: the smallest call, all latency.
        dict(name="rotary-token", op="rotary", batch=0, tokens=1, hq=32, hk=8, dim=128, rotary=128, dtype="bf16",
             interleaved=False, inverse=False, start=5000, rows=8192, scaling="none"),
        # A chunk of a long prompt in one layer, positions stretched for a 128K context.
        dict(name="rotary-prompt", op="rotary", batch=0, tokens=8192, hq=32, hk=8, dim=128, rotary=128, dtype="bf16",
             interleaved=False, inverse=False, start=100003, rows=131072, scaling="yarn"),
        # The backward pass (inverse rotation) of a batch kept as (batch, heads, tokens, dim), fp32, part of the head.
        dict(name="rotary-partial-fp32", op="rotary", batch=3, tokens=1021, hq=28, hk=4, dim=96, rotary=64, dtype="fp32",
             interleaved=True, inverse=True, start=0, rows=4096, scaling="linear"),
        # One decode step of a few sequences: rotate the queries and keys, append one row each.
        dict(name="append-step", op="append", sequences=8, longest=2048, chunk=1, hq=32, hk=8, dim=128, rotary=128, dtype="bf16",
             interleaved=False, block=32, layout="HND", query=True, scaling="none"),
        # The prompts of a dozen requests entering the pool, ragged, with their queries.
        dict(name="append-prompts", op="append", sequences=12, longest=4096, chunk=0, hq=32, hk=8, dim=128, rotary=128, dtype="bf16",
             interleaved=False, block=32, layout="HND", query=True, scaling="yarn"),
        # Chunked prefill far into three sequences, fp32 projections, small pages, no queries.
        dict(name="append-chunk-nhd", op="append", sequences=3, longest=31003, chunk=1003, hq=28, hk=4, dim=128, rotary=64, dtype="fp32",
             interleaved=True, block=16, layout="NHD", query=False, scaling="none"),
        # The first tokens of one conversation: the smallest attention, all latency.
        dict(name="attend-one-short", op="attend", sequences=1, longest=333, even=True, hq=32, hk=8, dim=128, dtype="bf16",
             block=32, layout="HND", window=0, lse=False),
        # One 128K-token conversation: the dense layers of a long-context decode.
        dict(name="attend-one-128k", op="attend", sequences=1, longest=131072, even=True, hq=32, hk=8, dim=128, dtype="bf16",
             block=32, layout="HND", window=0, lse=True),
        # A server's mixed batch: short and long sequences, empty slots, small pages, seven queries a head.
        dict(name="attend-ragged", op="attend", sequences=48, longest=6000, even=False, hq=28, hk=4, dim=128, dtype="bf16",
             block=16, layout="NHD", window=0, lse=False),
        # A full batch of long sequences: the largest, bound by the memory's rate.
        dict(name="attend-batch-32k", op="attend", sequences=16, longest=32768, even=True, hq=32, hk=8, dim=128, dtype="bf16",
             block=64, layout="HND", window=0, lse=False),
        # Sliding-window layers, small heads, fp32 queries whose parts are joined with another's by their log-sum-exp.
        dict(name="attend-window-fp32", op="attend", sequences=24, longest=16384, even=False, hq=64, hk=8, dim=64, dtype="fp32",
             block=32, layout="HND", window=4096, lse=True),
        # One layer's whole decode step of a batch: append the new token's keys and values, then attend.
        dict(name="step-batch", op="step", sequences=32, longest=4096, even=False, hq=32, hk=8, dim=128, rotary=128, dtype="bf16",
             interleaved=False, block=32, layout="HND", window=0, lse=False, scaling="none"),
    ]


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(("rotary", "append", "attend", "attend", "step"))
    hq, hk, dim = rng.choice(SHAPES)
    c = dict(op=op, hq=hq, hk=hk, dim=dim, dtype=rng.choice(("bf16", "bf16", "fp32")))
    rotation = dict(rotary=rng.choice((dim, dim, dim // 2)), interleaved=rng.random() < 0.4,
                    scaling=rng.choice(("none", "linear", "yarn")))
    if op == "rotary":
        batch = rng.choice((0, 0, 2, 5))
        tokens = _log(rng, 1, 16384 // max(1, batch))
        return dict(c, **rotation, batch=batch, tokens=tokens, inverse=rng.random() < 0.3, start=rng.randrange(100000), rows=131072)
    pool = dict(block=rng.choice((16, 32, 64)), layout=rng.choice(("HND", "NHD")))
    if op == "append":
        sequences = _log(rng, 1, 64)
        chunk = rng.choice((0, 1, 1, _log(rng, 2, 2048)))
        longest = max(chunk, _log(rng, 1, 32768 // sequences))
        return dict(c, **rotation, **pool, sequences=sequences, longest=longest, chunk=min(chunk, 32768 // sequences), query=rng.random() < 0.7)
    sequences = _log(rng, 1, 64)
    longest = _log(rng, 2, min(131072, MOST_CACHE // (sequences * hk * dim)))
    c = dict(c, **pool, sequences=sequences, longest=longest, even=rng.random() < 0.4,
             window=rng.choice((0, 0, 0, _log(rng, 1, 8192))), lse=rng.random() < 0.5)
    return c if op == "attend" else dict(c, **rotation)


def _lengths(case):
    """Tokens of each sequence: all the longest, or spread below it with every ninth slot empty."""
    n, longest = case["sequences"], case["longest"]
    if case.get("even") or n == 1:
        return [longest] * n
    floor = 1 if case["op"] in ("append", "step") else 0
    spread = [max(1, math.ceil(longest * ((i * 0.6180339887) % 1.0))) for i in range(n)]
    spread[0] = longest
    return [floor if i % 9 == 7 else length for i, length in enumerate(spread)]


def _frequencies(rotary, scaling, base=500000.0):
    w = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    if scaling == "linear":
        return w / 4, 1.0
    if scaling == "yarn":  # slow channels stretched four times, fast ones kept, a ramp between
        turns = 32768 * w / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return w * keep + w / 4 * (1 - keep), 0.1 * math.log(4) + 1
    return w, 1.0


def _table(rotary, rows, scaling):
    w, scale = _frequencies(rotary, scaling)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * w.cuda()
    return torch.cat([angle.cos(), angle.sin()], 1).mul_(scale).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = {"bf16": torch.bfloat16, "fp32": torch.float32}[case["dtype"]]

    def normal(*shape, dtype=dtype):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    hq, hk, dim = case["hq"], case["hk"], case["dim"]
    s = dict(case=case, interleaved=case.get("interleaved", False))
    if case["op"] == "rotary":
        batch, tokens = case["batch"], case["tokens"]
        s["cos_sin"] = _table(case["rotary"], case["rows"], case["scaling"])
        at = torch.arange(tokens, device="cuda", dtype=torch.int64) + case["start"] % max(1, case["rows"] - tokens)
        if batch:  # a model's (batch, heads, tokens, dim)
            s["query"], s["key"] = (normal(batch, h, tokens, dim).transpose(1, 2) for h in (hq, hk))
            at = at.expand(batch, tokens).contiguous()
        else:  # a server's (tokens, heads, dim), cut out of one projection
            both = normal(tokens, (hq + 2 * hk) * dim)
            s["query"] = both[:, : hq * dim].view(tokens, hq, dim)
            s["key"] = both[:, hq * dim : (hq + hk) * dim].view(tokens, hk, dim)
        s["positions"] = at
        return s
    lengths, block, n = _lengths(case), case["block"], case["sequences"]
    blocks = max(1, -(-max(lengths) // block))
    pages = n * blocks + 3
    shape = (pages, hk, block, dim) if case["layout"] == "HND" else (pages, block, hk, dim)
    s["key_pool"], s["value_pool"] = normal(*shape, dtype=torch.bfloat16), normal(*shape, dtype=torch.bfloat16)
    order = torch.randperm(pages, generator=gen, device="cuda")[: n * blocks]
    s["page_table"] = order.view(n, blocks).to(torch.int32)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["workspace"] = {}
    if case["op"] == "attend":
        s["query"] = normal(n, hq, dim)
        return s
    s["cos_sin"] = _table(case["rotary"], blocks * block, case["scaling"])
    # the new tokens of each sequence: its last `chunk` ones (all where chunk is 0; one each in a step)
    new = [min(length, case.get("chunk", 1) or length) for length in lengths]
    s["positions"] = torch.cat([torch.arange(a - m, a) for a, m in zip(lengths, new)]).to("cuda", torch.int32)
    s["sequence_ids"] = None
    if new != [1] * n:
        s["sequence_ids"] = torch.repeat_interleave(torch.arange(n), torch.tensor(new)).to("cuda", torch.int32)
    tokens = sum(new)
    both = normal(tokens, (hq + 2 * hk) * dim)
    s["query"] = both[:, : hq * dim].view(tokens, hq, dim) if case.get("query", True) else None
    s["key"] = both[:, hq * dim : (hq + hk) * dim].view(tokens, hk, dim)
    s["value"] = both[:, (hq + hk) * dim :].view(tokens, hk, dim)
    return s


# ---- the plain forms -------------------------------------------------------------------------


def _rotated(x, positions, cos_sin, interleaved, inverse=False):
    r = cos_sin.shape[1]
    row = cos_sin[positions].unsqueeze(-2)
    cos, sin = row[..., : r // 2], row[..., r // 2 :]
    if inverse:
        sin = -sin
    x32 = x.float()
    a, b = (x32[..., 0:r:2], x32[..., 1:r:2]) if interleaved else (x32[..., : r // 2], x32[..., r // 2 : r])
    y, z = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([turned, x32[..., r:]], -1).to(x.dtype)


def _append(s):
    positions, block = s["positions"].long(), s["case"]["block"]
    ids = torch.arange(len(positions), device="cuda") if s["sequence_ids"] is None else s["sequence_ids"].long()
    page, row = s["page_table"][ids, positions // block].long(), positions % block
    rows = (page, slice(None), row) if s["case"]["layout"] == "HND" else (page, row)
    s["key_pool"][rows] = _rotated(s["key"], positions, s["cos_sin"], s["interleaved"]).to(torch.bfloat16)
    s["value_pool"][rows] = s["value"].to(torch.bfloat16)
    return None if s["query"] is None else _rotated(s["query"], positions, s["cos_sin"], s["interleaved"])


def _visible(pool, s):
    """(sequences, KV heads, tokens, dim) in 32 bits."""
    rows = pool[s["page_table"].long()]  # (sequences, blocks, ...)
    rows = rows.permute(0, 2, 1, 3, 4) if s["case"]["layout"] == "HND" else rows.permute(0, 3, 1, 2, 4)
    return rows.float().flatten(2, 3)


def _attend(query, s):
    case = s["case"]
    n, hk, dim = case["sequences"], case["hk"], case["dim"]
    # a query is rounded to the cache's type before use
    q = query.to(torch.bfloat16).float().view(n, hk, -1, dim)
    scores = q @ _visible(s["key_pool"], s).transpose(2, 3) * dim**-0.5
    at, length = torch.arange(scores.shape[-1], device="cuda"), s["lengths"].view(n, 1, 1, 1)
    seen = at < length
    if case["window"]:
        seen = seen & (at >= length - case["window"])
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    out = p @ _visible(s["value_pool"], s) / total.masked_fill(total == 0, 1.0)
    lse = (top + total.log()).view(n, -1)
    out = out.view(n, -1, dim).to(query.dtype)
    return [out, lse] if case["lse"] else [out]


def _plain(s):
    case = s["case"]
    if case["op"] == "rotary":
        return [_rotated(s[x], s["positions"], s["cos_sin"], s["interleaved"], case["inverse"]) for x in ("query", "key")]
    if case["op"] == "attend":
        return _attend(s["query"], s)
    query = _append(s)
    if case["op"] == "step":
        return _attend(query, s) + [s["key_pool"], s["value_pool"]]
    return [s["key_pool"], s["value_pool"]] + ([] if query is None else [query])


# ---- the framework's calls -------------------------------------------------------------------


def _package():
    root = str(pathlib.Path(__file__).resolve().parent.parent / "refinekv-release_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import refinekv_b200

    return refinekv_b200


def _own(s):
    rkv, case = _package(), s["case"]
    if case["op"] == "rotary":
        return list(rkv.apply_rotary(s["query"], s["key"], s["positions"], s["cos_sin"], interleaved=s["interleaved"],
                                     inverse=case["inverse"]))
    query = s["query"]
    if case["op"] != "attend":
        query = rkv.paged_append(s["key"], s["value"], s["key_pool"], s["value_pool"], s["page_table"], s["positions"],
                                 layout=case["layout"], sequence_ids=s["sequence_ids"], query=query, cos_sin=s["cos_sin"],
                                 interleaved=s["interleaved"], workspace=s["workspace"])
        if case["op"] == "append":
            return [s["key_pool"], s["value_pool"]] + ([] if query is None else [query])
    out = rkv.paged_attention(query, s["key_pool"], s["value_pool"], s["page_table"], s["lengths"], layout=case["layout"],
                              window=case["window"] or None, return_lse=case["lse"], workspace=s["workspace"])
    out = list(out) if case["lse"] else [out]
    return out + [s["key_pool"], s["value_pool"]] if case["op"] == "step" else out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    hq, hk, dim = case["hq"], case["hk"], case["dim"]
    wide = 2 if case["dtype"] == "bf16" else 4
    read = flops = 0
    if case["op"] == "rotary":
        tokens = case["tokens"] * max(1, case["batch"])
        # queries and keys in and out, a position and a table row each
        distinct = case["tokens"]
        return dict(bytes=2 * tokens * (hq + hk) * dim * wide + tokens * 8 + distinct * case["rotary"] * 4,
                    flops=3 * tokens * (hq + hk) * case["rotary"])
    lengths = _lengths(case)
    if case["op"] != "attend":
        new = sum(min(n, case.get("chunk", 1) or n) for n in lengths)
        heads = hk + (hq if case.get("query", True) else 0)
        rows = new if case.get("chunk", 1) else max(lengths)  # whole prompts share the table's rows
        read += new * (hk * dim * 2 * (wide + 2) + (heads - hk) * dim * 2 * wide + 4) + rows * case["rotary"] * 4
        flops += 3 * new * heads * case["rotary"]
    if case["op"] != "append":
        seen = sum(min(n, case["window"] or n) for n in lengths)
        read += seen * hk * dim * 4 + len(lengths) * hq * (2 * dim * wide + (4 if case["lse"] else 0))
        flops += 4 * seen * hq * dim
    return dict(bytes=read, flops=flops)


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _turn64(x, positions, cos_sin, interleaved, sign=1.0):
    """Pairs as complex numbers, times the table's."""
    half = cos_sin.shape[1] // 2
    table = cos_sin.double()[positions.long()]
    spin = torch.complex(table[..., :half], sign * table[..., half:]).unsqueeze(-2)
    y = x.double().clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    z = torch.complex(y[..., first], y[..., second]) * spin
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        sign = -1.0 if case["inverse"] else 1.0
        return [_turn64(s[x], s["positions"], s["cos_sin"], s["interleaved"], sign) for x in ("query", "key")]
    hnd = case["layout"] == "HND"
    # (pages, block, KV heads, dim) views of the pools
    pools = [s[x].double().transpose(1, 2) if hnd else s[x].double() for x in ("key_pool", "value_pool")]
    query = s["query"]
    if case["op"] != "attend":
        at = s["positions"].long()
        owner = s["sequence_ids"].long() if s["sequence_ids"] is not None else torch.arange(len(at), device="cuda")
        flat = s["page_table"].long()[owner, at // case["block"]] * case["block"] + at % case["block"]
        new = [_turn64(s["key"], at, s["cos_sin"], s["interleaved"]), s["value"].double()]
        for pool, rows in zip(pools, new):
            pool[flat // case["block"], flat % case["block"]] = rows
        if query is not None:
            query = _turn64(query, at, s["cos_sin"], s["interleaved"])
        if case["op"] == "append":
            whole = [p.transpose(1, 2) if hnd else p for p in pools]
            return whole + ([] if query is None else [query])
        query = query.to(s["query"].dtype)  # the appended rows and the rotated queries are kept in their types
    n, hk, hq, dim = case["sequences"], case["hk"], case["hq"], case["dim"]
    out = torch.zeros(n, hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
    q = query.to(torch.bfloat16).double().view(n, hk, hq // hk, dim)
    for i, length in enumerate(_lengths(case)):
        low = max(0, length - case["window"]) if case["window"] else 0
        if length == low:
            continue
        table = s["page_table"][i].long()[low // case["block"] : -(-length // case["block"])]
        skip = low - low // case["block"] * case["block"]
        k, v = (p[table].flatten(0, 1)[skip : skip + length - low].to(torch.bfloat16).double() for p in pools)
        logits = torch.einsum("hgd,thd->hgt", q[i], k) / math.sqrt(dim)
        lse[i] = torch.logsumexp(logits, -1).flatten()
        out[i] = torch.einsum("hgt,thd->hgd", torch.softmax(logits, -1), v).flatten(0, 1)
    answer = [out, lse] if case["lse"] else [out]
    if case["op"] == "step":
        answer += [p.transpose(1, 2) if hnd else p for p in pools]
    return answer
