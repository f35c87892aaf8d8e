"""Serving from a page pool: appending new tokens, and dense attention of one new token.

No counterpart in the reference, which keeps one contiguous cache per layer
and decodes one sequence.  A server keeps the keys and values of many
sequences of different lengths in a pool of fixed-size pages; a page table
gives each sequence's pages.  ``attach_page_pool`` lets the refined layers
decode from such a pool; here is what fills it (``paged_append``), what reads
rows back (``paged_read``) and what the dense layers decode with
(``paged_attention``).

Pools are bf16, ``(pages, kv_heads, block, dim)`` (``layout="HND"``) or
``(pages, block, kv_heads, dim)`` (``"NHD"``), or hold a row in 4 bits a
channel (``fp4_pool``); page tables are int32
``(sequences, blocks)``.  Everything that changes from step to step
(positions, lengths, page tables) is read on the device, so a captured CUDA
graph serves growing sequences.  Results carry no gradient.

Pass the ``workspace`` dict of a layer or a server to every call: without one,
each call allocates its outputs and zero-fills its scratch anew.  A captured
graph keeps using the buffers it was captured with, so it wants a dict of its
own: a call of another shape replaces them in the dict.
"""

from __future__ import annotations

import functools
import math

import torch

from . import _native
from .attention import MAX_GROUP, _buffer, _scratch
from .rotary import _DTYPES, _POSITIONS, check_table, mark_written
from .summary import SUPPORTED_HEAD_DIMS, require_cuda_tensor

_BLOCKS = (16, 32, 64)


@functools.lru_cache(maxsize=None)
def _scratch_bytes(index: int, group: int, dim: int, dtype: int) -> int:
    """``paged_attention``'s workspace size on a device: it follows from the head shape and the
    pools' type alone."""
    with torch.cuda.device(index):
        return _native.load().rkv_paged_more_workspace_size(group, dim, dtype)


def _pools(key_pool, value_pool, layout):
    """(pages, kv_heads, block, dim) and both pools' (page, head, row) strides, checked."""
    if layout not in ("HND", "NHD"):
        raise ValueError("layout must be 'HND' or 'NHD'")
    shape = key_pool.shape
    if len(shape) != 4 or value_pool.shape != shape:
        raise ValueError("key and value pools must have the same 4-D shape")
    if not key_pool.is_cuda:
        require_cuda_tensor(key_pool, "key_pool")
    if key_pool.dtype is not torch.bfloat16 or value_pool.dtype is not torch.bfloat16:
        raise TypeError("page pools must be bf16")
    if value_pool.device != key_pool.device:
        raise ValueError("key and value pools must be on the same device")
    ks, vs = key_pool.stride(), value_pool.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("pool rows must be contiguous in head_dim")
    if layout == "HND":
        pages, heads, block, dim = shape
        ks, vs = ks[:3], vs[:3]
    else:
        pages, block, heads, dim = shape
        ks, vs = (ks[0], ks[2], ks[1]), (vs[0], vs[2], vs[1])
    if block not in _BLOCKS:
        raise ValueError("pool blocks must hold 16, 32 or 64 tokens")
    if dim not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {SUPPORTED_HEAD_DIMS}")
    return pages, heads, block, dim, ks, vs


def fp4_pool(pages: int, kv_heads: int, block: int, head_dim: int, *, device="cuda") -> torch.Tensor:
    """A zeroed page pool of 4 bits a channel: (pages, kv_heads, block, head_dim * 9 / 16) bytes.

    16 channels share an e4m3 scale (the greatest of them / 6), and a channel is
    one of 0, 0.5, 1, 1.5, 2, 3, 4 or 6 times it, with a sign: 72 bytes for a row of
    128 instead of 256.  The slab of a page's KV head, ``pool[page, head]``, holds
    the codes of its rows, row after row (head_dim / 2 bytes each, channel 2i in
    the low half of byte i), then their scales (head_dim / 16 bytes each).
    ``paged_append``, ``paged_read`` and ``paged_attention`` take such pools where
    they take bf16 ones, with an optional fp32 factor for each KV head
    (``key_scale``, ``value_scale``: a row is divided by it before it is held, and
    multiplied by it after): scales lie between 2^-9 and 448, so channels above
    2688 times the factor are cut off and ones far below 0.01 times it lose digits.
    """
    if block not in _BLOCKS:
        raise ValueError("pool blocks must hold 16, 32 or 64 tokens")
    if head_dim not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {SUPPORTED_HEAD_DIMS}")
    if pages < 0 or kv_heads < 1:
        raise ValueError("a pool has pages of at least one KV head")
    return torch.zeros(pages, kv_heads, block, head_dim * 9 // 16, device=device, dtype=torch.uint8)


def _fp4_pools(key_pool, value_pool, layout):
    """``_pools`` of two pools of 4 bits: strides in bytes, the third of them unused."""
    if layout != "HND":
        raise ValueError("a pool of 4 bits has layout 'HND'")
    shape = key_pool.shape
    if len(shape) != 4 or value_pool.shape != shape:
        raise ValueError("key and value pools must have the same 4-D shape")
    if not key_pool.is_cuda:
        require_cuda_tensor(key_pool, "key_pool")
    if value_pool.dtype is not torch.uint8:
        raise TypeError("key and value pools must both be bf16 or both of 4 bits (uint8)")
    if value_pool.device != key_pool.device:
        raise ValueError("key and value pools must be on the same device")
    pages, heads, block, row = shape
    dim = row * 16 // 9
    if dim not in SUPPORTED_HEAD_DIMS or dim * 9 != row * 16:
        raise ValueError(f"a pool of 4 bits has rows of 9 / 16 of a head_dim in {SUPPORTED_HEAD_DIMS}")
    if block not in _BLOCKS:
        raise ValueError("pool blocks must hold 16, 32 or 64 tokens")
    ks, vs = key_pool.stride(), value_pool.stride()
    if ks[2:] != (row, 1) or vs[2:] != (row, 1):
        raise ValueError("the slab of a page's KV head must be contiguous")
    return pages, heads, block, dim, (*ks[:2], 0), (*vs[:2], 0)


def _factors(key_scale, value_scale, heads, device):
    """The addresses of the KV heads' factors of a pool of 4 bits (0: none)."""
    if key_scale is None and value_scale is None:
        return 0, 0
    at = [0, 0]
    for i, factor in enumerate((key_scale, value_scale)):
        if factor is None:
            continue
        if factor.shape != (heads,) or factor.device != device or factor.stride(0) != 1:
            raise ValueError("key_scale and value_scale must be contiguous (kv_heads,) on the "
                             "pools' device")
        if factor.dtype is not torch.float32:
            raise TypeError("key_scale and value_scale must be fp32")
        at[i] = factor.data_ptr()
    return at


def _table(page_table, device):
    """(sequences, blocks, stride) of an int32 page table (1-D: one sequence)."""
    shape, stride = page_table.shape, page_table.stride()
    if len(shape) == 1:
        shape, stride = (1, shape[0]), (shape[0], stride[0])
    if len(shape) != 2 or stride[1] != 1 or page_table.device != device:
        raise ValueError("page_table must be (sequences, blocks) with contiguous rows on the "
                         "pools' device")
    if page_table.dtype != torch.int32:
        raise TypeError("page_table must be int32")
    return shape[0], shape[1], stride[0]


def paged_append(key: torch.Tensor, value: torch.Tensor, key_pool: torch.Tensor,
                 value_pool: torch.Tensor, page_table: torch.Tensor, positions: torch.Tensor, *,
                 layout: str = "HND", sequence_ids: torch.Tensor | None = None,
                 query: torch.Tensor | None = None, cos_sin: torch.Tensor | None = None,
                 interleaved: bool = False, key_scale: torch.Tensor | None = None,
                 value_scale: torch.Tensor | None = None,
                 workspace: dict | None = None) -> torch.Tensor | None:
    """Write new tokens' keys and values into the pool's pages, rotated on the way.

    ``key``/``value``: (tokens, kv_heads, head_dim) bf16 or fp32, any strides
    with contiguous rows (slices of a fused projection, say).  Token t is
    token ``positions[t]`` (int32 or int64) of sequence ``sequence_ids[t]``
    (int32; without it token t belongs to sequence t: one new token each) and
    goes to page ``page_table[sequence, position // block]``, row
    ``position % block``, rounded once to bf16.  With ``cos_sin`` (see
    ``apply_rotary``) keys are rotated by their positions first, and so is
    ``query`` ((tokens, q_heads, head_dim), the keys' dtype) when given.  Into
    pools of 4 bits (``fp4_pool``) rows go from fp32 in one rounding too, divided in
    fp32 by ``key_scale`` and ``value_scale`` ((kv_heads,) fp32) where these are given;
    16 channels that hold an infinity or a NaN, or whose quotients do, become NaN.

    Returns the rotated queries (backed by ``workspace``, reused by the next
    call of the same shape), or None without ``query``.  The pools are
    written in place.  Any mix of prompts, chunks and single tokens goes in
    one call; no two tokens of a call may name the same sequence and position.

    A negative position is padding (an idle slot of a captured step): nothing
    is written and its query row is zero.  A position past the page table's
    row or the rotation table, a sequence id outside the page table or a page
    outside the pool writes nothing and sets bit 1 of the status word
    (``attention.device_status(workspace)``).
    """
    fp4 = key_pool.dtype is torch.uint8
    pages, heads, block, dim, ks, vs = (_fp4_pools if fp4 else _pools)(key_pool, value_pool, layout)
    device = key_pool.device
    factors = ()
    if fp4:
        factors = _factors(key_scale, value_scale, heads, device)
    elif key_scale is not None or value_scale is not None:
        raise ValueError("key_scale and value_scale belong to pools of 4 bits")
    sequences, blocks, table_stride = _table(page_table, device)
    shape, dtype = key.shape, key.dtype
    if len(shape) != 3 or value.shape != shape or shape[1] != heads or shape[2] != dim:
        raise ValueError("key and value must be (tokens, kv_heads, head_dim) matching the pools")
    if key.device != device or value.device != device:
        raise ValueError("key and value must be on the pools' device")
    if dtype not in _DTYPES or value.dtype != dtype:
        raise TypeError("key and value must both be BF16 or both FP32")
    tokens = shape[0]
    if positions.shape != (tokens,) or positions.device != device:
        raise ValueError("positions must be (tokens,) on the pools' device")
    if positions.dtype not in _POSITIONS:
        raise TypeError("positions must be int32 or int64")
    if sequence_ids is None:
        if tokens > sequences:
            raise ValueError("more tokens than sequences: pass sequence_ids")
        ids = 0
    else:
        if sequence_ids.shape != (tokens,) or sequence_ids.device != device:
            raise ValueError("sequence_ids must be (tokens,) on the pools' device")
        if sequence_ids.dtype != torch.int32:
            raise TypeError("sequence_ids must be int32")
        if not sequence_ids.is_contiguous():
            sequence_ids = sequence_ids.contiguous()
        ids = sequence_ids.data_ptr()
    table = rotary = rows = row_stride = 0
    if cos_sin is not None:
        check_table(cos_sin, dim, device)
        table, rotary = cos_sin.data_ptr(), cos_sin.shape[1]
        rows, row_stride = cos_sin.shape[0], cos_sin.stride(0)
    key_strides, value_strides = key.stride(), value.stride()
    if key_strides[2] != 1:
        key = key.contiguous()
        key_strides = key.stride()
    if value_strides[2] != 1:
        value = value.contiguous()
        value_strides = value.stride()
    if not positions.is_contiguous():
        positions = positions.contiguous()
    out = None
    query_ptr = out_ptr = query_heads = 0
    query_strides = out_strides = (0, 0)
    if query is not None:
        like = query.shape
        if len(like) != 3 or like[0] != tokens or like[2] != dim or query.device != device:
            raise ValueError("query must be (tokens, q_heads, head_dim) on the pools' device")
        if query.dtype != dtype:
            raise TypeError("query must have the keys' dtype")
        query_strides = query.stride()
        if query_strides[2] != 1:
            query = query.contiguous()
            query_strides = query.stride()
        query_strides = query_strides[:2]
        out = _buffer(workspace, "append_query", like, device, dtype)
        query_ptr, out_ptr, query_heads = query.data_ptr(), out.data_ptr(), like[1]
        out_strides = (query_heads * dim, dim)
    status = 0
    if workspace is not None:
        status = _scratch(workspace, "rkv_append_status", 256, device).data_ptr()
    lib = _native.load()
    _native.launch(
        lib.rkv_paged_append_fp4 if fp4 else lib.rkv_paged_append,
        (_native.APPEND_FP4_ARGS if fp4 else _native.APPEND_ARGS).pack(
            key.data_ptr(), value.data_ptr(), query_ptr, out_ptr, key_pool.data_ptr(),
            value_pool.data_ptr(), page_table.data_ptr(), ids, positions.data_ptr(), table, status,
            key_strides[0], key_strides[1], value_strides[0], value_strides[1], *query_strides,
            *out_strides, *ks, *vs,
            table_stride, sequences, blocks, pages, block, tokens, query_heads, heads, dim, rotary,
            rows, row_stride, _DTYPES[dtype], positions.dtype is torch.int64, interleaved, *factors),
        device)
    mark_written(key_pool, value_pool)
    return out


def paged_read(key_pool: torch.Tensor, value_pool: torch.Tensor, page_table: torch.Tensor,
               positions: torch.Tensor, *, layout: str = "HND",
               sequence_ids: torch.Tensor | None = None, key_scale: torch.Tensor | None = None,
               value_scale: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
               workspace: dict | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that a pool's pages hold, as dense rows: ``paged_append`` read back.

    Token t is token ``positions[t]`` (int32 or int64) of sequence
    ``sequence_ids[t]`` (int32; without it token t is one of sequence t).
    Returns new (tokens, kv_heads, head_dim) keys and values in ``dtype`` (bf16 or
    fp32): what a chunk of a prompt needs of the tokens before it, or a summary
    of a pool of 4 bits (its rows in bf16 are exact where there is no ``key_scale``
    or ``value_scale``).  A negative position gives a zero row.  A position past
    the page table's row, a sequence id outside the page table or a page outside
    the pool gives a NaN row and sets bit 1 of the status word
    (``attention.device_status(workspace)``).
    """
    fp4 = key_pool.dtype is torch.uint8
    pages, heads, block, dim, ks, vs = (_fp4_pools if fp4 else _pools)(key_pool, value_pool, layout)
    device = key_pool.device
    if fp4:
        factors = _factors(key_scale, value_scale, heads, device)
    elif key_scale is not None or value_scale is not None:
        raise ValueError("key_scale and value_scale belong to pools of 4 bits")
    else:
        factors = (0, 0)
    sequences, blocks, table_stride = _table(page_table, device)
    if positions.ndim != 1 or positions.device != device:
        raise ValueError("positions must be (tokens,) on the pools' device")
    if positions.dtype not in _POSITIONS:
        raise TypeError("positions must be int32 or int64")
    if dtype not in _DTYPES:
        raise TypeError("rows are read as BF16 or FP32")
    tokens = positions.shape[0]
    ids = 0
    if sequence_ids is None:
        if tokens > sequences:
            raise ValueError("more tokens than sequences: pass sequence_ids")
    else:
        if sequence_ids.shape != (tokens,) or sequence_ids.device != device:
            raise ValueError("sequence_ids must be (tokens,) on the pools' device")
        if sequence_ids.dtype != torch.int32:
            raise TypeError("sequence_ids must be int32")
        if not sequence_ids.is_contiguous():
            sequence_ids = sequence_ids.contiguous()
        ids = sequence_ids.data_ptr()
    if not positions.is_contiguous():
        positions = positions.contiguous()
    keys = torch.empty(tokens, heads, dim, device=device, dtype=dtype)
    values = torch.empty_like(keys)
    status = 0
    if workspace is not None:
        status = _scratch(workspace, "rkv_append_status", 256, device).data_ptr()
    _native.launch(
        _native.load().rkv_paged_read,
        _native.READ_ARGS.pack(
            key_pool.data_ptr(), value_pool.data_ptr(), keys.data_ptr(), values.data_ptr(),
            page_table.data_ptr(), ids, positions.data_ptr(), status, *factors, *ks, *vs,
            heads * dim, dim, heads * dim, dim, table_stride, sequences, blocks, pages, block, tokens,
            heads, dim, _native.DTYPE_FP4 if fp4 else _native.DTYPE_BF16, _DTYPES[dtype],
            positions.dtype is torch.int64),
        device)
    return keys, values


def paged_attention(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, *, layout: str = "HND",
                    scale: float | None = None, window: int | None = None, prefix: int = 0,
                    softcap: float | None = None, slopes: torch.Tensor | None = None,
                    key_scale: torch.Tensor | None = None, value_scale: torch.Tensor | None = None,
                    weights: torch.Tensor | None = None, return_lse: bool = False,
                    workspace: dict | None = None):
    """Exact attention of one new token per sequence over its own length of the pool.

    ``query``: (sequences, q_heads, head_dim) bf16 or fp32, any strides; query
    head r reads KV head r // (q_heads // kv_heads), at most 16 to a KV head; at most 4096 sequences.
    ``lengths``: (sequences,) int32, the tokens of each sequence now in the
    pool (the new one included, once ``paged_append`` has written it); a
    sequence of length 0 (an idle slot) gives a zero row.  ``scale`` defaults
    to head_dim ** -0.5; ``window`` limits each query to the last ``window``
    tokens, next to which the first ``prefix`` stay visible.  Rows of a page past
    a sequence's length, pages past it and tokens between its prefix and its window
    are never used, whatever they hold.  An fp32 query is
    rounded to bf16 first, like every query of this package; its
    probabilities, sums and output stay fp32.

    The logit of token j of a sequence of L is ``c * tanh(scale * q.k / c)`` with
    ``softcap`` c (without it ``scale * q.k``), plus ``slopes[head] * (j - (L -
    1))`` with ``slopes``, (q_heads,) fp32: a bias that grows with the distance.

    Pools may hold 4 bits a channel (``fp4_pool``), with the ``key_scale`` and
    ``value_scale`` that ``paged_append`` was given: the attention is exact over
    what the pool stands for, but for weights held to 2^-11 of themselves (fp32
    queries: 2^-22) and channels of a query below 2^-29 of its greatest one, which lose
    digits.  Rows whose logits spread by many nats (steep ``slopes``) take longer there.

    ``weights``: (sequences, kv_heads, tokens) fp32, contiguous in its last
    dimension and at least as wide as the page table's row in tokens: to each
    visible token's entry the softmax weight that it got is added, summed over the
    query heads of its KV head (what ``paged_evict`` goes by).  A query whose sum is
    not finite adds nothing.  Takes a second launch and scratch for the logits, 4
    bytes a query head and token of the page table's width, however short the
    sequences are (256 of 128K tokens' width and 32 heads: 4.3 GB); it stays in the
    ``workspace``.

    Returns the (sequences, q_heads, head_dim) output in the query's dtype or,
    with ``return_lse``, (output, lse) with the fp32 natural-log sum of the
    exponentials (-inf for an empty row): outputs over parts of a sequence join
    as sum_i exp(lse_i - lse) output_i.  Backed by ``workspace``, reused by the
    next call of the same shape.  A length past the page table's row or a
    visible page outside the pool sets bit 1 of
    ``attention.device_status(workspace)`` and makes that sequence's output (and
    lse) NaN; a negative length sets it and counts as 0.
    One launch (two with ``weights``); its results repeat bit for bit.
    """
    fp4 = key_pool.dtype is torch.uint8
    pages, heads, block, dim, ks, vs = (_fp4_pools if fp4 else _pools)(key_pool, value_pool, layout)
    device = key_pool.device
    sequences, blocks, table_stride = _table(page_table, device)
    shape, dtype = query.shape, query.dtype
    if len(shape) != 3 or shape[0] != sequences or shape[2] != dim:
        raise ValueError("query must be (sequences, q_heads, head_dim) matching the page table "
                         "and the pools")
    if query.device != device:
        raise ValueError("query must be on the pools' device")
    if dtype not in _DTYPES:
        raise TypeError("the CUDA backend requires BF16 or FP32 queries")
    group = shape[1] // heads
    if group * heads != shape[1] or not 1 <= group <= MAX_GROUP:
        raise ValueError("q_heads must be 1 to 16 times the pools' KV heads")
    if lengths.shape != (sequences,) or lengths.device != device:
        raise ValueError("lengths must be (sequences,) on the pools' device")
    if lengths.dtype != torch.int32:
        raise TypeError("lengths must be int32")
    if window is not None and window < 1:
        raise ValueError("window must be at least 1")
    if prefix < 0:
        raise ValueError("prefix must not be negative")
    if not fp4 and (key_scale is not None or value_scale is not None):
        raise ValueError("key_scale and value_scale belong to pools of 4 bits")
    scale = dim ** -0.5 if scale is None else float(scale)
    qs = query.stride()
    width = 2 if dtype == torch.bfloat16 else 4
    if qs[2] != 1 or (query.data_ptr() | qs[0] * width | qs[1] * width) & 15:
        query = query.clone(memory_format=torch.contiguous_format)
        qs = query.stride()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    plain = not (fp4 or softcap is not None or slopes is not None or weights is not None
                 or (prefix and window is not None))
    more = ()
    if not plain:
        slopes, more = _more(sequences, heads, group, blocks * block, device, prefix, softcap,
                             slopes, key_scale, value_scale, weights, fp4, workspace)
    out = _buffer(workspace, "paged_output", shape, device, dtype)
    lse = None
    if return_lse or weights is not None:
        lse = _buffer(workspace, "paged_lse", shape[:2], device, torch.float32)
    kind = _native.DTYPE_FP4 if fp4 else _native.DTYPE_BF16
    scratch = _scratch(workspace, "rkv_paged_scratch",
                       _scratch_bytes(device.index, group, dim, kind), device)
    lib = _native.load()
    _native.launch(
        lib.rkv_paged_attention if plain else lib.rkv_paged_attention_more,
        (_native.PAGED_ARGS if plain else _native.PAGED_MORE_ARGS).pack(
            query.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
            key_pool.data_ptr(), value_pool.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
            scratch.data_ptr(), scratch.numel(), qs[0], qs[1], *ks, *vs, table_stride, sequences,
            blocks, pages, block, heads, group, dim, _DTYPES[dtype], window or 0, scale, *more),
        device)
    if weights is not None:
        mark_written(weights)
    return (out, lse) if return_lse else out


def _token_rows(name, rows, dtype, sequences, heads, capacity, device):
    """Checks (sequences, kv_heads, tokens) rows that are written in place."""
    shape = rows.shape
    if (len(shape) != 3 or shape[0] != sequences or shape[1] != heads or shape[2] < capacity
            or rows.device != device):
        raise ValueError(f"{name} must be (sequences, kv_heads, tokens) on the pools' device, with at "
                         "least the page table's tokens")
    if rows.dtype is not dtype:
        raise TypeError(f"{name} must be {'fp32' if dtype is torch.float32 else 'int32'}")
    if rows.is_contiguous():
        return
    *outer, last = rows.stride()
    extent, apart = shape[2], last == 1 or shape[2] <= 1
    for stride, count in sorted(zip(outer, shape)):
        apart = apart and (count <= 1 or stride >= extent)
        extent += stride * (count - 1) if count > 1 else 0
    if not apart:
        raise ValueError(f"{name} must have contiguous rows that do not overlap")


def _more(sequences, heads, group, capacity, device, prefix, softcap, slopes, key_scale,
          value_scale, weights, fp4, workspace):
    """The checked arguments of ``rkv_paged_attention_more`` behind ``rkv_paged_attention``'s, and
    the slopes as they must be kept until the launch."""
    if softcap is None:
        softcap = 0.0
    elif not (0 < softcap < math.inf):
        raise ValueError("softcap must be positive and finite")
    slopes_ptr = 0
    if slopes is not None:
        if slopes.shape != (heads * group,) or slopes.device != device:
            raise ValueError("slopes must be (q_heads,) on the pools' device")
        if slopes.dtype is not torch.float32:
            raise TypeError("slopes must be fp32")
        slopes = slopes.contiguous()
        slopes_ptr = slopes.data_ptr()
    factors = _factors(key_scale, value_scale, heads, device)
    weights_ptr = scores_ptr = scores_size = tokens = 0
    strides = (0, 0)
    if weights is not None:
        _token_rows("weights", weights, torch.float32, sequences, heads, capacity, device)
        strides = weights.stride()[:2]
        count = sequences * heads * group * capacity
        scores = workspace.get("paged_scores") if workspace is not None else None
        if scores is None or scores.device != device or scores.numel() < count:
            scores = torch.empty(max(count, 4), device=device, dtype=torch.float32)
            if workspace is not None:
                workspace["paged_scores"] = scores
        weights_ptr, scores_ptr, scores_size = weights.data_ptr(), scores.data_ptr(), 4 * scores.numel()
        tokens = weights.shape[2]
        slopes = (slopes, scores)  # both live until the launch
    return slopes, (slopes_ptr, *factors, weights_ptr, scores_ptr, scores_size, *strides, tokens,
                    _native.DTYPE_FP4 if fp4 else _native.DTYPE_BF16, prefix, softcap)


@functools.lru_cache(maxsize=None)
def _evict_bytes(sequences: int, heads: int, capacity: int, budget: int) -> int:
    return _native.load().rkv_paged_evict_workspace_size(sequences, heads, capacity, budget)


def paged_evict(key_pool: torch.Tensor, value_pool: torch.Tensor, page_table: torch.Tensor,
                lengths: torch.Tensor, weights: torch.Tensor, budget: int, *, recent: int = 0,
                positions: torch.Tensor | None = None, layout: str = "HND",
                workspace: dict | None = None) -> torch.Tensor:
    """Bring sequences down to ``budget`` tokens a KV head: those that got the most weight stay.

    ``lengths``: (sequences,) int32, the rows each sequence has in the pool (bf16 or
    4 bits, ``fp4_pool``).  ``weights``: (sequences, kv_heads, tokens) fp32, what
    ``paged_attention`` adds up.  Of a KV head's rows in a sequence of more than
    ``budget`` are kept the ``recent`` newest and of the others the ones of
    greatest weight (of equal ones the first; NaN counts least).  Kept rows at or
    behind row ``budget`` move into the places of dropped ones before it, keys,
    values, weights and all, so that the sequence is its first ``budget`` rows
    again; weights behind it become zero, ready for the next tokens.

    Rows are then in no order of position, and each KV head has its own tokens:
    ``paged_attention`` does not see that, but a ``window``, ``slopes`` or block
    summaries no longer fit such a sequence.  ``positions``: (sequences, kv_heads,
    tokens) int32 says which token each row holds, moves along and decides which
    rows are newest (those above the greatest less ``recent``); without it they are
    the last rows, which holds for a first eviction.  A token appended later goes to
    row ``lengths`` (``paged_append``'s position) but is rotated by its own position
    (``apply_rotary``).

    A sequence's pages must be its own: rows that move into a page which another
    sequence's table names too would change that sequence, so copy shared pages first.

    Returns the new lengths, ``min(lengths, budget)`` (backed by ``workspace``, reused
    by the next call that is not given them as ``lengths``).  The ``workspace`` also
    keeps the list of moves, 8 bytes a KV head and row that could move, min(budget, the
    page table's tokens - budget) of them (256 sequences of 128K tokens' width, 8 KV heads,
    a budget of 64K: 1.1 GB).  Pools, weights and positions are written in place;
    nothing carries a gradient.  A length past the page table leaves its sequence
    as it is, a negative one counts as 0, and a row from a page outside the pool is
    NaN where it goes; each sets bit 1 of ``attention.device_status(workspace)``.
    """
    fp4 = key_pool.dtype is torch.uint8
    pages, heads, block, dim, ks, vs = (_fp4_pools if fp4 else _pools)(key_pool, value_pool, layout)
    device = key_pool.device
    sequences, blocks, table_stride = _table(page_table, device)
    if lengths.shape != (sequences,) or lengths.device != device:
        raise ValueError("lengths must be (sequences,) on the pools' device")
    if lengths.dtype != torch.int32:
        raise TypeError("lengths must be int32")
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    capacity = blocks * block
    if budget < 1:
        raise ValueError("budget must be at least 1")
    if not 0 <= recent <= budget:
        raise ValueError("recent must be between 0 and budget")
    _token_rows("weights", weights, torch.float32, sequences, heads, capacity, device)
    positions_ptr = positions_width = 0
    position_strides = (0, 0)
    if positions is not None:
        _token_rows("positions", positions, torch.int32, sequences, heads, capacity, device)
        positions_ptr, positions_width = positions.data_ptr(), positions.shape[2]
        position_strides = positions.stride()[:2]
    out = _buffer(workspace, "evict_lengths", (sequences,), device, torch.int32)
    if sequences and out.data_ptr() == lengths.data_ptr():  # the last call's answer
        out = _buffer(workspace, "evict_lengths_other", (sequences,), device, torch.int32)
    scratch = _scratch(workspace, "rkv_evict_scratch",
                       _evict_bytes(sequences, heads, capacity, budget), device)
    _native.launch(
        _native.load().rkv_paged_evict,
        _native.EVICT_ARGS.pack(
            key_pool.data_ptr(), value_pool.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
            out.data_ptr(), weights.data_ptr(), positions_ptr, scratch.data_ptr(), scratch.numel(),
            *ks, *vs, *weights.stride()[:2], *position_strides, weights.shape[2], positions_width,
            table_stride, sequences, blocks, pages, block, heads, dim,
            _native.DTYPE_FP4 if fp4 else _native.DTYPE_BF16, budget, recent),
        device)
    mark_written(key_pool, value_pool, weights, positions)
    return out
