"""What is measured of the page pool's further operators: a pool held in 4 bits, attention with a cap, a bias or a prefix, and eviction.

``own`` False computes the operators in plain torch operations (32 bits, rounded once at the end), True calls
``refinekv_b200``.  Sequences keep their keys and values in a pool of pages; ``page_table[s, b]`` is the physical page of
logical block ``b`` of sequence ``s``; ``lengths`` are the sequences' tokens.

A pool of 4 bits is uint8, (pages, KV heads, block, dim / 2 + dim / 16).  The slab of a page's KV head holds the codes of
its rows, one row after another (dim / 2 bytes each, channel 2i in the low half of byte i), and after them the scales of
its rows (dim / 16 bytes each).  A code is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; 16 channels share a scale, an
e4m3 number.  What a code stands for is code * scale, times the KV head's own fp32 factor where there is one.
"""

import functools
import math
import pathlib
import sys

import torch

own = False

#: (query heads, KV heads, head dim) of the shapes drawn: Llama-3.1-8B, Qwen2.5-7B, and generic ones.
SHAPES = ((32, 8, 128), (28, 4, 128), (64, 8, 64), (16, 2, 256), (12, 4, 96), (8, 8, 128), (16, 1, 128))

#: Elements of the largest listed cache (t: sequences x tokens x KV heads x dim); a drawn one has no more.
MOST_CACHE = 16 * 32768 * 8 * 128

_ATTEND = dict(op="attend", even=False, hq=32, hk=8, dim=128, dtype="bf16", block=32, layout="HND", bits=16, window=0, prefix=0,
               softcap=0.0, slopes=False, factors=False, weights=False, lse=False)
_APPEND = dict(op="append", hq=32, hk=8, dim=128, rotary=128, dtype="bf16", interleaved=False, block=32, query=True, factors=False,
               scaling="none")
_EVICT = dict(op="evict", even=False, hk=8, dim=128, block=32, layout="HND", bits=16, aged=False)


def listed():
    return [
        # One decode step of a few sequences: rotate the queries and keys, hold one row each in 4 bits.
        dict(_APPEND, name="fp4-append-step", sequences=8, longest=2048, chunk=1),
        # The prompts of a dozen requests entering the pool of 4 bits, ragged, with their queries.
        dict(_APPEND, name="fp4-append-prompts", sequences=12, longest=4096, chunk=0, scaling="yarn"),
        # The first tokens of one conversation: the smallest attention over 4 bits, all latency.
        dict(_ATTEND, name="fp4-attend-short", sequences=1, longest=333, even=True, bits=4),
        # One 128K-token conversation held in 4 bits.
        dict(_ATTEND, name="fp4-attend-128k", sequences=1, longest=131072, even=True, bits=4, lse=True),
        # A full batch of long sequences in 4 bits: the largest, bound by the memory's rate.
        dict(_ATTEND, name="fp4-attend-batch-32k", sequences=16, longest=32768, even=True, bits=4, block=64),
        # A server's mixed batch in 4 bits: short and long sequences, empty slots, small pages, fp32 queries, a factor per head.
        dict(_ATTEND, name="fp4-attend-ragged-fp32", sequences=48, longest=6000, hq=28, hk=4, block=16, bits=4, dtype="fp32",
             factors=True, lse=True),
        # The same batch from a bf16 pool, its scores capped.
        dict(_ATTEND, name="cap-ragged", sequences=48, longest=6000, hq=28, hk=4, block=16, layout="NHD", softcap=50.0),
        # Sliding-window layers that keep their first tokens, a bias by distance, small heads, fp32 queries.
        dict(_ATTEND, name="bias-window-prefix-fp32", sequences=24, longest=16384, hq=64, dim=64, dtype="fp32", window=4096, prefix=100,
             slopes=True, lse=True),
        # A decode step that adds up what weight each token gets, in a batch of middling sequences.
        dict(_ATTEND, name="weigh-batch", sequences=16, longest=8192, weights=True),
        # The same over one long conversation in 4 bits.
        dict(_ATTEND, name="weigh-fp4-128k", sequences=1, longest=131072, even=True, bits=4, weights=True),
        # A step of a batch whose every cache is full: one token of each KV head goes.
        dict(_EVICT, name="evict-step", sequences=32, longest=4097, even=True, budget=4096, recent=256, aged=True),
        # Long prompts brought down to a budget after prefill.
        dict(_EVICT, name="evict-prompts", sequences=8, longest=32768, budget=4096, recent=512),
    ]


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "evict"))
    hq, hk, dim = rng.choice(SHAPES)
    block = rng.choice((16, 32, 64))
    if op == "append":
        sequences = _log(rng, 1, 64)
        chunk = rng.choice((0, 1, 1, _log(rng, 2, 2048)))
        longest = max(chunk, _log(rng, 1, 24576 // sequences))
        return dict(_APPEND, hq=hq, hk=hk, dim=dim, block=block, sequences=sequences, longest=longest, chunk=min(chunk, 24576 // sequences),
                    query=rng.random() < 0.7, rotary=rng.choice((dim, dim, dim // 2)), interleaved=rng.random() < 0.4,
                    dtype=rng.choice(("bf16", "bf16", "fp32")), factors=rng.random() < 0.5, scaling=rng.choice(("none", "linear", "yarn")))
    bits = rng.choice((4, 16))
    c = dict(hk=hk, dim=dim, block=block, bits=bits, layout="HND" if bits == 4 else rng.choice(("HND", "NHD")), even=rng.random() < 0.4)
    if op == "evict":
        sequences = _log(rng, 1, 64)
        longest = _log(rng, 64, min(131072, MOST_CACHE // 4 // (sequences * hk * dim)))
        budget = _log(rng, 1, longest)
        return dict(_EVICT, **{**c, "sequences": sequences, "longest": longest, "budget": budget, "recent": rng.randrange(budget + 1),
                               "aged": rng.random() < 0.5})
    sequences = _log(rng, 1, 64)
    longest = _log(rng, 2, min(131072, MOST_CACHE // (sequences * hk * dim)))
    form = rng.choice(("plain", "cap", "bias", "prefix", "weights")) if bits == 4 else rng.choice(("cap", "bias", "prefix", "weights"))
    window = _log(rng, 1, 8192) if form == "prefix" or rng.random() < 0.2 else 0
    return dict(_ATTEND, **{**c, "sequences": sequences, "longest": longest, "hq": hq, "dtype": rng.choice(("bf16", "bf16", "fp32")),
                            "window": window, "prefix": _log(rng, 1, 512) if form == "prefix" else 0,
                            "softcap": rng.choice((20.0, 30.0, 50.0)) if form == "cap" or rng.random() < 0.2 else 0.0,
                            "slopes": form == "bias", "weights": form == "weights", "factors": bits == 4 and rng.random() < 0.4,
                            "lse": rng.random() < 0.5})


def _lengths(case):
    """Tokens of each sequence: all the longest, or spread below it with every ninth slot empty (one token, for an append)."""
    n, longest = case["sequences"], case["longest"]
    if case.get("even") or n == 1:
        return [longest] * n
    floor = 1 if case["op"] == "append" else 0
    spread = [max(1, math.ceil(longest * ((i * 0.6180339887) % 1.0))) for i in range(n)]
    spread[0] = longest
    return [floor if i % 9 == 7 else length for i, length in enumerate(spread)]


# ---- 4 bits in plain operations ----------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _levels():
    sizes = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(sizes + [-x for x in sizes], device="cuda")


def _to_codes(x):
    """(rows, dim) fp32 -> uint8 codes (rows, dim / 2) and scales (rows, dim / 16)."""
    blocks = x.unflatten(-1, (-1, 16))
    most = blocks.abs().amax(-1)
    # a true quotient: by a plain number, the GPU would multiply by its reciprocal, and ties would fall elsewhere
    scale = (most / torch.full_like(most, 6.0)).clamp(max=448.0).to(torch.float8_e4m3fn)
    by = scale.float()
    y = blocks / by.masked_fill(by == 0, math.inf)[..., None]
    size = y.abs()
    # the nearest level, ties to the even code
    code = ((size > 0.25).byte() + (size >= 0.75).byte() + (size > 1.25).byte() + (size >= 1.75).byte() + (size > 2.5).byte()
            + (size >= 3.5).byte() + (size > 5.0).byte())
    code = (code + 8 * torch.signbit(y).byte()).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], scale.view(torch.uint8)


def _from_codes(codes, scales):
    """fp32 values (..., dim) of codes (..., dim / 2) and scales (..., dim / 16)."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    values = _levels()[code.int()].unflatten(-1, (-1, 16))
    return (values * scales.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)


def _split(pool, dim):
    """Views (pages, KV heads, block, dim / 2) and (pages, KV heads, block, dim / 16) of a pool of 4 bits."""
    pages, heads, block, _ = pool.shape
    flat = pool.view(pages, heads, -1)
    return flat[..., : block * dim // 2].unflatten(-1, (block, -1)), flat[..., block * dim // 2 :].unflatten(-1, (block, -1))


# ---- inputs --------------------------------------------------------------------------------------


def _table(rotary, rows, scaling, base=500000.0):
    w = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    size = 1.0
    if scaling == "linear":
        w = w / 4
    elif scaling == "yarn":  # slow channels stretched four times, fast ones kept, a ramp between
        keep = ((32768 * w / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
        w, size = w * keep + w / 4 * (1 - keep), 0.1 * math.log(4) + 1
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * w.cuda()
    return torch.cat([angle.cos(), angle.sin()], 1).mul_(size).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hk, dim, block, n = case["hk"], case["dim"], case["block"], case["sequences"]
    lengths = _lengths(case)
    blocks = max(1, -(-max(lengths) // block))
    pages = n * blocks + 3
    s = dict(case=case, workspace={}, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    # a few channels of the keys are several times the others, as rotated keys' are
    loud = 1 + 4 * (torch.rand(hk, dim, generator=gen, device="cuda") < 0.06)

    def factor():
        return 0.25 + torch.rand(hk, generator=gen, device="cuda") if case.get("factors") else None

    s["key_scale"], s["value_scale"] = factor(), factor()

    def pool(keys):
        if case.get("bits", 4) == 16:
            hnd = case["layout"] == "HND"
            x = torch.randn((pages, hk, block, dim) if hnd else (pages, block, hk, dim), generator=gen, device="cuda", dtype=torch.bfloat16)
            return x.mul_(loud[:, None] if hnd else loud) if keys else x
        held = torch.zeros(pages, hk, block, dim * 9 // 16, device="cuda", dtype=torch.uint8)
        codes, scales = _split(held, dim)
        step = max(1, (1 << 25) // (hk * block * dim))
        for low in range(0, pages if case["op"] != "append" else 0, step):
            x = torch.randn(min(step, pages - low), hk, block, dim, generator=gen, device="cuda")
            codes[low : low + step], scales[low : low + step] = _to_codes(x * loud[:, None] if keys else x)
        return held

    s["key_pool"], s["value_pool"] = pool(True), pool(False)
    order = torch.randperm(pages, generator=gen, device="cuda")[: n * blocks]
    s["page_table"] = order.view(n, blocks).to(torch.int32)
    if case["op"] == "evict":
        # what the steps so far have added up, a few tokens far above the rest
        s["weights"] = torch.randn(n, hk, blocks * block, generator=gen, device="cuda").mul_(1.5).exp_().mul_(0.01)
        s["positions"] = None
        if case["aged"]:  # the rows below the budget hold the survivors of earlier evictions, in no order
            k = min(case["budget"], blocks * block)
            at = torch.arange(blocks * block, device="cuda").expand(n, hk, -1).clone()
            at[..., :k] = torch.rand(n, hk, k, generator=gen, device="cuda").argsort(-1)
            s["positions"] = at.to(torch.int32)
        reach = torch.tensor([min(length, case["budget"]) for length in lengths])
        s["kept_at"] = torch.cat([torch.arange(m) for m in reach.tolist()]).to("cuda", torch.int32)
        s["kept_of"] = torch.repeat_interleave(torch.arange(n), reach).to("cuda", torch.int32)
        return s
    hq = case["hq"]
    dtype = {"bf16": torch.bfloat16, "fp32": torch.float32}[case["dtype"]]
    if case["op"] == "attend":
        s["query"] = torch.randn(n, hq, dim, generator=gen, device="cuda", dtype=dtype)
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq) if case["slopes"] else None
        s["weights"] = None
        if case["weights"]:
            s["weights"] = torch.rand(n, hk, blocks * block, generator=gen, device="cuda") * 0.01
        return s
    s["cos_sin"] = _table(case["rotary"], blocks * block, case["scaling"])
    # the new tokens of each sequence: its last `chunk` ones, all where chunk is 0
    new = [min(length, case["chunk"] or length) for length in lengths]
    s["positions"] = torch.cat([torch.arange(a - m, a) for a, m in zip(lengths, new)]).to("cuda", torch.int32)
    s["sequence_ids"] = None
    if new != [1] * n:
        s["sequence_ids"] = torch.repeat_interleave(torch.arange(n), torch.tensor(new)).to("cuda", torch.int32)
    tokens = sum(new)
    both = torch.randn(tokens, (hq + 2 * hk) * dim, generator=gen, device="cuda", dtype=dtype)
    s["query"] = both[:, : hq * dim].view(tokens, hq, dim) if case["query"] else None
    s["key"] = both[:, hq * dim : (hq + hk) * dim].view(tokens, hk, dim).mul_(loud)
    s["value"] = both[:, (hq + hk) * dim :].view(tokens, hk, dim)
    return s


# ---- the plain forms -----------------------------------------------------------------------------


def _rotated(x, positions, cos_sin, interleaved):
    r = cos_sin.shape[1]
    row = cos_sin[positions].unsqueeze(-2)
    cos, sin = row[..., : r // 2], row[..., r // 2 :]
    x = x.float()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2 : r])
    y, z = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _rows_at(s, positions, ids):
    positions, block = positions.long(), s["case"]["block"]
    ids = torch.arange(len(positions), device="cuda") if ids is None else ids.long()
    return s["page_table"][ids, positions // block].long(), slice(None), positions % block


def _read(s, at, factor, pool):
    codes, scales = _split(s[pool], s["case"]["dim"])
    values = _from_codes(codes[at], scales[at])
    return values if factor is None else values * factor[:, None]


def _append(s):
    at = _rows_at(s, s["positions"], s["sequence_ids"])
    keys = _rotated(s["key"], s["positions"].long(), s["cos_sin"], s["case"]["interleaved"])
    for pool, rows, factor in (("key_pool", keys, s["key_scale"]), ("value_pool", s["value"].float(), s["value_scale"])):
        if factor is not None:
            rows = rows / factor[:, None]
        codes, scales = _split(s[pool], s["case"]["dim"])
        codes[at], scales[at] = _to_codes(rows)
    out = [_read(s, at, s["key_scale"], "key_pool").bfloat16(), _read(s, at, s["value_scale"], "value_pool").bfloat16()]
    if s["query"] is not None:
        out.append(_rotated(s["query"], s["positions"].long(), s["cos_sin"], s["case"]["interleaved"]).to(s["query"].dtype))
    return out


def _visible(pool, factor, s):
    """(sequences, KV heads, tokens, dim) in 32 bits."""
    table = s["page_table"].long()
    if s["case"]["bits"] == 4:
        codes, scales = _split(pool, s["case"]["dim"])
        rows = _from_codes(codes[table], scales[table]).permute(0, 2, 1, 3, 4)
        if factor is not None:
            rows = rows * factor.view(1, -1, 1, 1, 1)
    else:
        rows = pool[table].permute(0, 2, 1, 3, 4) if s["case"]["layout"] == "HND" else pool[table].permute(0, 3, 1, 2, 4)
    return rows.float().flatten(2, 3)


def _attend(s):
    case = s["case"]
    n, hk, hq, dim = case["sequences"], case["hk"], case["hq"], case["dim"]
    # a query is rounded to bf16 before use
    q = s["query"].to(torch.bfloat16).float().view(n, hk, -1, dim)
    scores = q @ _visible(s["key_pool"], s["key_scale"], s).transpose(2, 3) * dim**-0.5
    at, length = torch.arange(scores.shape[-1], device="cuda"), s["lengths"].view(n, 1, 1, 1)
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    if case["slopes"]:
        scores = scores + s["slopes"].view(1, hk, hq // hk, 1) * (at - (length - 1))
    seen = at < length
    if case["window"]:
        seen = seen & ((at >= length - case["window"]) | (at < case["prefix"]))
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    safe = total.masked_fill(total == 0, 1.0)
    out = p @ _visible(s["value_pool"], s["value_scale"], s) / safe
    answer = [out.view(n, hq, dim).to(s["query"].dtype)]
    if case["lse"]:
        answer.append((top + total.log()).view(n, hq))
    if case["weights"]:
        s["weights"] += (p / safe).sum(2)
        answer.append(s["weights"])
    return answer


def _evict(s):
    case = s["case"]
    n, hk, block, k = case["sequences"], case["hk"], case["block"], case["budget"]
    weights = s["weights"].clone()
    positions = None if s["positions"] is None else s["positions"].clone()
    at, length = torch.arange(weights.shape[-1], device="cuda"), s["lengths"].view(n, 1, 1)
    there = at < length
    age = at.expand_as(weights) if positions is None else positions
    newest = age.masked_fill(~there, -1).amax(-1, keepdim=True)
    worth = weights.masked_fill(age > newest - case["recent"], math.inf).masked_fill(~there, -math.inf)
    order = worth.sort(dim=-1, descending=True, stable=True).indices[..., :k]
    keep = torch.zeros_like(there.expand_as(weights)).scatter(-1, order, True) & there
    full = (length > k).expand_as(weights)
    holes, movers = (~keep & (at < k) & full).nonzero(as_tuple=True), (keep & (at >= k) & full).nonzero(as_tuple=True)
    to, src = ((s["page_table"][x[0], x[2] // block].long(), x[1], x[2] % block) for x in (holes, movers))
    for pool in ("key_pool", "value_pool"):
        if case["bits"] == 4:
            for part in _split(s[pool], case["dim"]):
                part[to] = part[src]
        elif case["layout"] == "HND":
            s[pool][to] = s[pool][src]
        else:
            s[pool][to[0], to[2], to[1]] = s[pool][src[0], src[2], src[1]]
    for values in (weights, positions):
        if values is not None:
            values[holes] = values[movers]
    weights.masked_fill_(full & there & (at >= k), 0.0)
    return _evicted(s, s["lengths"].clamp(max=k), weights, positions)


def _evicted(s, lengths, weights, positions, read=None):
    """What an eviction leaves: the rows of a bf16 pool, or those that a pool of 4 bits stands for."""
    if s["case"]["bits"] == 16:
        rows = [s["key_pool"], s["value_pool"]]
    elif read is None:
        at = _rows_at(s, s["kept_at"], s["kept_of"])
        rows = [_read(s, at, None, pool).bfloat16() for pool in ("key_pool", "value_pool")]
    else:
        rows = list(read(s["key_pool"], s["value_pool"], s["page_table"], s["kept_at"], sequence_ids=s["kept_of"]))
    return [lengths, weights] + ([] if positions is None else [positions]) + rows


# ---- the framework's calls -----------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _package():
    root = str(pathlib.Path(__file__).resolve().parent.parent / "refinekv-release_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import refinekv_b200

    return refinekv_b200


def _own(s):
    rkv, case = _package(), s["case"]
    pools = s["key_pool"], s["value_pool"], s["page_table"]
    if case["op"] == "append":
        factors = dict(key_scale=s["key_scale"], value_scale=s["value_scale"])
        query = rkv.paged_append(s["key"], s["value"], *pools, s["positions"], sequence_ids=s["sequence_ids"], query=s["query"],
                                 cos_sin=s["cos_sin"], interleaved=case["interleaved"], workspace=s["workspace"], **factors)
        rows = list(rkv.paged_read(*pools, s["positions"], sequence_ids=s["sequence_ids"], **factors))
        return rows + ([] if query is None else [query])
    if case["op"] == "evict":
        weights = s["weights"].clone()
        positions = None if s["positions"] is None else s["positions"].clone()
        lengths = rkv.paged_evict(*pools, s["lengths"], weights, case["budget"], recent=case["recent"], positions=positions,
                                  layout=case["layout"], workspace=s["workspace"])
        return _evicted(s, lengths, weights, positions, rkv.paged_read)
    out = rkv.paged_attention(s["query"], *pools, s["lengths"], layout=case["layout"], window=case["window"] or None,
                              prefix=case["prefix"], softcap=case["softcap"] or None, slopes=s["slopes"], key_scale=s["key_scale"],
                              value_scale=s["value_scale"], weights=s["weights"], return_lse=case["lse"], workspace=s["workspace"])
    return (list(out) if case["lse"] else [out]) + ([s["weights"]] if case["weights"] else [])


def run(state):
    return _own(state) if own else {"append": _append, "attend": _attend, "evict": _evict}[state["case"]["op"]](state)


def _seen(case, length):
    window = case["window"]
    return length if not window or length <= window else window + min(case["prefix"], length - window)


def work(case):
    hk, dim = case["hk"], case["dim"]
    lengths = _lengths(case)
    row = dim * 9 // 16 if case.get("bits", 4) == 4 else dim * 2  # bytes of a key or a value
    if case["op"] == "evict":
        k, r = case["budget"], case["recent"]
        read = flops = 0
        for n in lengths:
            if n > k:  # every weight once, and the rows that change place: expected for weights in no order
                moved = k - k * (k - r) / max(1, n - r) if r <= n - k else k * (n - k) / n
                read += hk * (4 * n + max(1, moved) * (4 * row + 8))
                flops += hk * n
        return dict(bytes=max(read, len(lengths) * 8), flops=flops)
    hq, wide = case["hq"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "append":
        new = [min(n, case["chunk"] or n) for n in lengths]
        heads = hk + (hq if case["query"] else 0)
        table = sum(new) if case["chunk"] else max(lengths)  # whole prompts share the table's rows
        # keys, values and queries in, codes and queries out, and the rows read back
        return dict(bytes=sum(new) * (hk * 2 * (dim * wide + 2 * row + 2 * dim) + (heads - hk) * dim * 2 * wide + 4) + table * case["rotary"] * 4,
                    flops=sum(new) * (3 * heads * case["rotary"] + 8 * hk * dim))
    seen = sum(_seen(case, n) for n in lengths)
    # a sequence's weights are read and written once, and the scores are needed again when their sum is known
    return dict(bytes=seen * hk * (2 * row + (8 if case["weights"] else 0)) + len(lengths) * hq * (2 * dim * wide + (4 if case["lse"] else 0)),
                flops=4 * seen * hq * dim)


# ---- the definitions in 64 bits -------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _powers():
    return torch.tensor([2.0**k for k in range(-64, 64)], dtype=torch.float64, device="cuda")


def _two64(k):
    """2^k, exactly."""
    return _powers()[k.long() + 64]


def _held64(pool, page, head, row, dim):
    """fp64 values of rows of a pool of 4 bits, from the bits' meaning."""
    pages, heads, block, _ = pool.shape
    flat = pool.view(pages, heads, -1)
    byte = flat[page[..., None], head[..., None], row[..., None] * (dim // 2) + torch.arange(dim // 2, device="cuda")].long()
    nibble = torch.stack([byte % 16, byte // 16], -1).flatten(-2)
    rest = nibble % 8
    power, half = rest // 2, (rest % 2).double()
    size = torch.where(power == 0, 0.5 * half, _two64(power - 1) * (1 + 0.5 * half))
    value = torch.where(nibble >= 8, -size, size)
    bits = flat[page[..., None], head[..., None], block * (dim // 2) + row[..., None] * (dim // 16)
                + torch.arange(dim // 16, device="cuda")].long()
    power, part = bits // 8 % 16, (bits % 8).double() / 8
    scale = torch.where(power == 0, part * 2.0**-6, (1 + part) * _two64(power - 7))
    return value * scale.repeat_interleave(16, -1)


def _nearest64(x):
    """What (rows, dim) numbers become in 4 bits, in 64 bits."""
    block = x.reshape(*x.shape[:-1], -1, 16)
    most = block.abs().max(-1, keepdim=True).values
    want = (most / torch.full_like(most, 6.0)).clamp(max=448.0)
    unit = _two64((torch.frexp(want).exponent - 1).clamp(min=-6) - 3)
    scale = torch.round(want / unit) * unit
    y = (block / scale.masked_fill(scale == 0, math.inf)).clamp(-6, 6)
    unit = _two64((torch.frexp(y).exponent - 1).clamp(min=0) - 1)
    return (torch.round(y / unit) * unit * scale).reshape(x.shape)


def _turn64(x, positions, cos_sin, interleaved):
    """Pairs as complex numbers, times the table's."""
    half = cos_sin.shape[1] // 2
    table = cos_sin.double()[positions.long()]
    spin = torch.complex(table[..., :half], table[..., half:]).unsqueeze(-2)
    y = x.double().clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    z = torch.complex(y[..., first], y[..., second]) * spin
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _rows64(s, pool, i, at):
    """(KV heads, rows, dim) of sequence i's rows `at` (KV heads, rows)."""
    case = s["case"]
    page = s["page_table"][i].long()[at // case["block"]]
    head, row = torch.arange(case["hk"], device="cuda")[:, None].expand_as(at), at % case["block"]
    if case["bits"] == 4:
        return _held64(s[pool], page, head, row, case["dim"])
    return s[pool][(page, head, row) if case["layout"] == "HND" else (page, row, head)].double()


def _exact_evict(s):
    case = s["case"]
    k, lengths = case["budget"], _lengths(case)
    weights, positions = s["weights"].double().clone(), None if s["positions"] is None else s["positions"].clone()
    pools = [s[x].clone() for x in ("key_pool", "value_pool")]
    kept_rows = [[], []]
    for i, n in enumerate(lengths):
        source = torch.arange(min(n, k), device="cuda").repeat(case["hk"], 1)
        for h in range(case["hk"]) if n > k else ():
            age = torch.arange(n, device="cuda") if positions is None else positions[i, h, :n].long()
            worth = weights[i, h, :n].clone()
            worth[age > age.max() - case["recent"]] = math.inf
            # ties go to the lowest row: of equal ones the reversed ascending order ends with it
            kept = (n - 1 - worth.flip(0).sort(stable=True).indices.flip(0))[:k].sort().values
            gone = torch.ones(k, dtype=torch.bool, device="cuda")
            gone[kept[kept < k]] = False
            source[h, gone] = kept[kept >= k]
            weights[i, h, :k] = weights[i, h, source[h]]
            if positions is not None:
                positions[i, h, :k] = positions[i, h, source[h]]
        weights[i, :, k:n] = 0
        for j, pool in enumerate(("key_pool", "value_pool")):
            rows = _rows64(s, pool, i, source)
            if case["bits"] == 4:
                kept_rows[j].append(rows.transpose(0, 1))
                continue
            at = torch.arange(min(n, k), device="cuda")
            page, row = s["page_table"][i].long()[at // case["block"]], at % case["block"]
            head = torch.arange(case["hk"], device="cuda")[:, None]
            pools[j][(page, head, row) if case["layout"] == "HND" else (page, row, head)] = rows.to(torch.bfloat16)
    new = torch.tensor([min(n, k) for n in lengths], dtype=torch.int32, device="cuda")
    rows = [torch.cat(x) for x in kept_rows] if case["bits"] == 4 else [p.double() for p in pools]
    return [new, weights] + ([] if positions is None else [positions]) + rows


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(s)
    if case["op"] == "append":
        keys = _turn64(s["key"], s["positions"], s["cos_sin"], case["interleaved"])
        answer = []
        for rows, factor in ((keys, s["key_scale"]), (s["value"].double(), s["value_scale"])):
            by = 1.0 if factor is None else factor.double()[:, None]
            answer.append(_nearest64(rows / by) * by)
        return answer + ([] if s["query"] is None else [_turn64(s["query"], s["positions"], s["cos_sin"], case["interleaved"])])
    n, hk, hq, dim = case["sequences"], case["hk"], case["hq"], case["dim"]
    out = torch.zeros(n, hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
    weights = None if s["weights"] is None else s["weights"].double()
    q = s["query"].to(torch.bfloat16).double().view(n, hk, hq // hk, dim)
    by = [torch.ones(hk, device="cuda").double() if s[x] is None else s[x].double() for x in ("key_scale", "value_scale")]
    for i, length in enumerate(_lengths(case)):
        at = torch.arange(length, device="cuda")
        if case["window"]:
            at = at[(at >= length - case["window"]) | (at < case["prefix"])]
        if len(at) == 0:
            continue
        keys, values = (_rows64(s, x, i, at.repeat(hk, 1)) * f[:, None, None] for x, f in zip(("key_pool", "value_pool"), by))
        logits = torch.einsum("hgd,htd->hgt", q[i], keys) / math.sqrt(dim)
        if case["softcap"]:
            logits = torch.tanh(logits / case["softcap"]) * case["softcap"]
        if case["slopes"]:
            logits = logits - s["slopes"].double().view(hk, -1, 1) * (length - 1 - at)
        p = torch.softmax(logits, -1)
        lse[i] = torch.logsumexp(logits, -1).flatten()
        out[i] = torch.einsum("hgt,htd->hgd", p, values).flatten(0, 1)
        if weights is not None:
            weights[i][:, at] += p.sum(1)
    return [out] + ([lse] if case["lse"] else []) + ([weights] if case["weights"] else [])
