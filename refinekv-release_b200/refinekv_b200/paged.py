"""Serving from a page pool: appending new tokens, and dense attention of one new token.

No counterpart in the reference, which keeps one contiguous cache per layer
and decodes one sequence.  A server keeps the keys and values of many
sequences of different lengths in a pool of fixed-size pages; a page table
gives each sequence's pages.  ``attach_page_pool`` lets the refined layers
decode from such a pool; here is what fills it (``paged_append``) and what
the dense layers decode with (``paged_attention``).

Pools are bf16, ``(pages, kv_heads, block, dim)`` (``layout="HND"``) or
``(pages, block, kv_heads, dim)`` (``"NHD"``); page tables are int32
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

import torch

from . import _native
from .attention import MAX_GROUP, _buffer, _scratch
from .rotary import _DTYPES, _POSITIONS, check_table, mark_written
from .summary import SUPPORTED_HEAD_DIMS, require_cuda_tensor

_BLOCKS = (16, 32, 64)


@functools.lru_cache(maxsize=None)
def _scratch_bytes(index: int, group: int, dim: int) -> int:
    """``paged_attention``'s workspace size on a device: it follows from the head shape alone."""
    with torch.cuda.device(index):
        return _native.load().rkv_paged_workspace_size(group, dim)


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
                 interleaved: bool = False, workspace: dict | None = None) -> torch.Tensor | None:
    """Write new tokens' keys and values into the pool's pages, rotated on the way.

    ``key``/``value``: (tokens, kv_heads, head_dim) bf16 or fp32, any strides
    with contiguous rows (slices of a fused projection, say).  Token t is
    token ``positions[t]`` (int32 or int64) of sequence ``sequence_ids[t]``
    (int32; without it token t belongs to sequence t: one new token each) and
    goes to page ``page_table[sequence, position // block]``, row
    ``position % block``, rounded once to bf16.  With ``cos_sin`` (see
    ``apply_rotary``) keys are rotated by their positions first, and so is
    ``query`` ((tokens, q_heads, head_dim), the keys' dtype) when given.

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
    pages, heads, block, dim, ks, vs = _pools(key_pool, value_pool, layout)
    device = key_pool.device
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
    _native.launch(
        _native.load().rkv_paged_append,
        _native.APPEND_ARGS.pack(
            key.data_ptr(), value.data_ptr(), query_ptr, out_ptr, key_pool.data_ptr(),
            value_pool.data_ptr(), page_table.data_ptr(), ids, positions.data_ptr(), table, status,
            key_strides[0], key_strides[1], value_strides[0], value_strides[1], *query_strides,
            *out_strides, *ks, *vs,
            table_stride, sequences, blocks, pages, block, tokens, query_heads, heads, dim, rotary,
            rows, row_stride, _DTYPES[dtype], positions.dtype is torch.int64, interleaved),
        device)
    mark_written(key_pool, value_pool)
    return out


def paged_attention(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, *, layout: str = "HND",
                    scale: float | None = None, window: int | None = None,
                    return_lse: bool = False, workspace: dict | None = None):
    """Exact attention of one new token per sequence over its own length of the pool.

    ``query``: (sequences, q_heads, head_dim) bf16 or fp32, any strides; query
    head r reads KV head r // (q_heads // kv_heads), at most 16 to a KV head; at most 4096 sequences.
    ``lengths``: (sequences,) int32, the tokens of each sequence now in the
    pool (the new one included, once ``paged_append`` has written it); a
    sequence of length 0 (an idle slot) gives a zero row.  ``scale`` defaults
    to head_dim ** -0.5; ``window`` limits each query to the last ``window``
    tokens.  Rows of a page past a sequence's length, pages past it and pages
    before its window are never used, whatever they hold.  An fp32 query is
    rounded to bf16 first, like every query of this package; its
    probabilities, sums and output stay fp32.

    Returns the (sequences, q_heads, head_dim) output in the query's dtype or,
    with ``return_lse``, (output, lse) with the fp32 natural-log sum of the
    exponentials (-inf for an empty row): outputs over parts of a sequence join
    as sum_i exp(lse_i - lse) output_i.  Backed by ``workspace``, reused by the
    next call of the same shape.  A length past the page table's row or a
    visible page outside the pool sets bit 1 of
    ``attention.device_status(workspace)`` and makes that sequence's output (and
    lse) NaN; a negative length sets it and counts as 0.
    One launch; its results repeat bit for bit.
    """
    pages, heads, block, dim, ks, vs = _pools(key_pool, value_pool, layout)
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
    scale = dim ** -0.5 if scale is None else float(scale)
    qs = query.stride()
    width = 2 if dtype == torch.bfloat16 else 4
    if qs[2] != 1 or (query.data_ptr() | qs[0] * width | qs[1] * width) & 15:
        query = query.clone(memory_format=torch.contiguous_format)
        qs = query.stride()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    out = _buffer(workspace, "paged_output", shape, device, dtype)
    lse = _buffer(workspace, "paged_lse", shape[:2], device, torch.float32) if return_lse else None
    scratch = _scratch(workspace, "rkv_paged_scratch", _scratch_bytes(device.index, group, dim),
                       device)
    _native.launch(
        _native.load().rkv_paged_attention,
        _native.PAGED_ARGS.pack(
            query.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
            key_pool.data_ptr(), value_pool.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
            scratch.data_ptr(), scratch.numel(), qs[0], qs[1], *ks, *vs, table_stride, sequences,
            blocks, pages, block, heads, group, dim, _DTYPES[dtype], window or 0, scale),
        device)
    return (out, lse) if return_lse else out
