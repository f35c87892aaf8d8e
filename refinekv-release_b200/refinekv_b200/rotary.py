"""Rotary positions of queries and keys.

No counterpart in the reference, which attaches behind a model that has
rotated its own queries and keys; a server that fills a page pool
(``paged_append``) and decodes from it needs the rotation itself.  The angles
come from a table (``rotary_table``, or any fp32 table of the same layout), so
every frequency scaling for long contexts is the table's, not the kernel's.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _native
from .summary import require_cuda_tensor

_POSITIONS = (torch.int32, torch.int64)
_DTYPES = {torch.bfloat16: _native.DTYPE_BF16, torch.float32: _native.DTYPE_F32}


#: The keys of a scaling dictionary that each type reads; the first ones it cannot do without.
_SCALINGS = {
    "default": ((), ()),
    "none": ((), ()),
    "linear": (("factor",), ()),
    "ntk": (("factor",), ()),
    "yarn": (("factor", "original_max_position_embeddings"),
             ("attention_factor", "beta_fast", "beta_slow", "mscale", "mscale_all_dim",
              "truncate")),
    "llama3": (("factor", "original_max_position_embeddings", "low_freq_factor",
                "high_freq_factor"), ()),
}
#: Keys that say nothing about the angles of a table of a given width.
_NEUTRAL = ("partial_rotary_factor", "max_position_embeddings", "original_max_position_embeddings")


def _frequencies(rotary_dim: int, base: float, scaling: dict | None):
    """fp64 angular frequencies of the pairs and the amplitude of the table."""
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    plain = base ** -exponent
    scaling = {key: value for key, value in (scaling or {}).items() if value is not None}
    kind = scaling.pop("rope_type", scaling.pop("type", "default"))
    if kind not in _SCALINGS:
        raise ValueError("scaling type must be 'linear', 'ntk', 'yarn' or 'llama3'")
    needed, optional = _SCALINGS[kind]
    for key in needed:
        if key not in scaling:
            raise ValueError(f"scaling {kind!r} needs {key!r}")
    for key in scaling:
        if key not in (*needed, *optional, *_NEUTRAL):
            raise ValueError(f"scaling {kind!r} does not know {key!r}")
    if not needed:
        return plain, 1.0
    factor = float(scaling["factor"])
    if not math.isfinite(factor) or factor < 1:
        raise ValueError("scaling factor must be at least 1")
    if kind == "linear":
        return plain / factor, 1.0
    if kind == "ntk":  # the base stretched so that the slowest pair slows by `factor`
        if rotary_dim == 2:
            return plain, 1.0
        return (base * factor ** (rotary_dim / (rotary_dim - 2))) ** -exponent, 1.0
    original = float(scaling["original_max_position_embeddings"])
    if not math.isfinite(original) or original <= 0:
        raise ValueError("original_max_position_embeddings must be positive")
    if kind == "llama3":
        # Pairs that turn more than high_freq_factor times within the original
        # context are kept, fewer than low_freq_factor times slowed by
        # `factor`, and blended linearly in between.
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not 0 <= low < high:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        turns = original * plain / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return plain * keep + plain / factor * (1 - keep), 1.0

    # YaRN: the same idea, blended linearly over the channel index between the
    # (rounded) channels that turn beta_fast and beta_slow times.
    def channel(turns):
        return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    first, last = channel(scaling.get("beta_fast") or 32), channel(scaling.get("beta_slow") or 1)
    if scaling.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rotary_dim - 1)
    if first == last:
        last += 0.001
    index = torch.arange(rotary_dim // 2, dtype=torch.float64)
    slow = ((index - first) / (last - first)).clamp(0, 1)
    amplitude = scaling.get("attention_factor")
    if amplitude is None:
        def grown(by):
            return 0.1 * by * math.log(factor) + 1

        mscale, all_dim = scaling.get("mscale"), scaling.get("mscale_all_dim")
        amplitude = grown(mscale) / grown(all_dim) if mscale and all_dim else grown(1.0)
    return plain / factor * slow + plain * (1 - slow), float(amplitude)


def rotary_table(rotary_dim: int, positions: int, *, base: float | None = None,
                 scaling: dict | None = None, device="cuda") -> torch.Tensor:
    """The fp32 (positions, rotary_dim) table ``apply_rotary`` and ``paged_append`` read.

    Row p holds the cosines of p * frequency of the rotary_dim / 2 pairs, then
    their sines, computed in fp64 and rounded once (an fp32 product of a
    position near 10^5 with a frequency is off by up to 4e-3 rad).
    ``scaling`` is a model configuration's rope scaling: ``{"rope_type":
    "linear" | "ntk" | "yarn" | "llama3", "factor": ...}`` with that type's
    further keys (one that the type does not know is refused), and ``rope_theta``, the base, unless ``base`` is given (10000
    without either).  Built once and kept by the caller.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if positions < 1:
        raise ValueError("positions must be positive")
    scaling = dict(scaling or {})
    theta = scaling.pop("rope_theta", None)
    if theta is not None and base is not None and float(theta) != float(base):
        raise ValueError("base and the scaling's 'rope_theta' differ: give one of them")
    base = float(base if base is not None else theta if theta is not None else 10000.0)
    if not math.isfinite(base) or base <= 1:
        raise ValueError("base (rope_theta) must be finite and above 1")
    frequency, amplitude = _frequencies(rotary_dim, base, scaling)
    frequency = frequency.to(device)
    table = torch.empty(positions, rotary_dim, device=device, dtype=torch.float32)
    step = max(1, (1 << 24) // rotary_dim)  # bounds the fp64 temporaries
    for low in range(0, positions, step):
        high = min(positions, low + step)
        angle = torch.arange(low, high, device=device, dtype=torch.float64)[:, None] * frequency
        table[low:high, : rotary_dim // 2] = angle.cos() * amplitude
        table[low:high, rotary_dim // 2:] = angle.sin() * amplitude
    return table


def check_table(cos_sin: torch.Tensor, dim: int, device: torch.device) -> None:
    """The argument checks of a cos/sin table shared with ``paged_append``."""
    shape = cos_sin.shape
    if len(shape) != 2 or cos_sin.stride(1) != 1 or shape[0] < 1:
        raise ValueError("cos_sin must be a (positions, rotary_dim) table with contiguous rows")
    if cos_sin.dtype is not torch.float32:
        raise TypeError("cos_sin must be fp32")
    if cos_sin.device != device:
        raise ValueError("cos_sin must be on the rows' device")
    rotary = shape[1]
    if rotary < 2 or rotary % 2 or rotary > dim:
        raise ValueError("rotary_dim (cos_sin's width) must be even and at most head_dim")


_NO_STRIDES = (0, 0, 0)


def _strides(tensor: torch.Tensor) -> tuple:
    """(batch, token, head) element strides of a 3-D or 4-D tensor of rows."""
    stride = tensor.stride()
    return stride[:3] if len(stride) == 4 else (0, stride[0], stride[1])


def _like(rows):
    """An output for `rows`: their layout where they have one, each row contiguous in any case
    (overlapping views may be given another innermost dimension)."""
    out = torch.empty_like(rows)
    return out if out.stride(-1) == 1 else torch.empty(rows.shape, device=rows.device,
                                                       dtype=rows.dtype)


def _launch(query, key, positions, cos_sin, interleaved, inverse, in_place):
    if query.stride(-1) != 1:
        if in_place:
            raise ValueError("query must be contiguous in head_dim to be rotated in place")
        query = query.contiguous()
    strides = out_strides = _strides(query)
    query_out = query
    if not in_place:
        query_out = _like(query)
        out_strides = _strides(query_out)
    key_out, key_ptr, key_out_ptr, key_heads = None, 0, 0, 0
    key_strides = key_out_strides = _NO_STRIDES
    if key is not None:
        if key.stride(-1) != 1:
            if in_place:
                raise ValueError("key must be contiguous in head_dim to be rotated in place")
            key = key.contiguous()
        key_strides = key_out_strides = _strides(key)
        key_out, key_ptr = key, key.data_ptr()
        key_out_ptr, key_heads = key_ptr, key.shape[-2]
        if not in_place:
            key_out = _like(key)
            key_out_ptr, key_out_strides = key_out.data_ptr(), _strides(key_out)
    batch, (tokens, heads, dim) = 1, query.shape[-3:]
    at = positions.stride()
    if len(at) == 2:
        batch = query.shape[0]
    else:
        at = (0, at[0])
    rows, rotary = cos_sin.shape
    _native.launch(
        _native.load().rkv_rotary,
        _native.ROTARY_ARGS.pack(
            query.data_ptr(), key_ptr, query_out.data_ptr(), key_out_ptr, positions.data_ptr(),
            cos_sin.data_ptr(), *strides, *key_strides, *out_strides, *key_out_strides, *at,
            positions.dtype is torch.int64, rows, cos_sin.stride(0), batch, tokens, heads,
            key_heads, dim, rotary, _DTYPES[query.dtype], interleaved, inverse),
        query.device)
    return query_out, key_out


def _is_dual(tensor) -> bool:
    """Whether the tensor carries a tangent of forward-mode differentiation (outside of a dual
    level, which is asked first because it is cheap, none does)."""
    return (forward_ad._current_level >= 0 and tensor is not None
            and forward_ad.unpack_dual(tensor).tangent is not None)


def mark_written(*tensors) -> None:
    """Raise the version counters of tensors that a kernel wrote in place, so that autograd
    refuses to use one that it saved before (inference tensors have no counter)."""
    torch.autograd.graph.increment_version([t for t in tensors
                                            if t is not None and not t.is_inference()])


class _Rotary(torch.autograd.Function):
    """The rotation is linear in its rows: its backward pass is the inverse rotation, and tangents
    are rotated like the rows."""

    @staticmethod
    def forward(ctx, query, key, positions, cos_sin, interleaved, inverse):
        ctx.save_for_backward(positions, cos_sin)
        ctx.save_for_forward(positions, cos_sin)
        ctx.flags = interleaved, inverse, key is not None
        out = _launch(query, key, positions, cos_sin, interleaved, inverse, False)
        return out if key is not None else out[0]

    @staticmethod
    def backward(ctx, query_grad, key_grad=None):
        positions, cos_sin = ctx.saved_tensors
        interleaved, inverse, both = ctx.flags
        query_grad, key_grad = apply_rotary(query_grad, key_grad if both else None, positions,
                                            cos_sin, interleaved=interleaved,
                                            inverse=not inverse)
        return query_grad, key_grad, None, None, None, None

    @staticmethod
    def jvp(ctx, query_tangent, key_tangent, *_):
        positions, cos_sin = ctx.saved_tensors
        interleaved, inverse, both = ctx.flags
        out = apply_rotary(query_tangent, key_tangent if both else None, positions, cos_sin,
                           interleaved=interleaved, inverse=inverse)
        return out if both else out[0]


def apply_rotary(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor,
                 cos_sin: torch.Tensor, *, interleaved: bool = False, inverse: bool = False,
                 in_place: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotate queries and keys by their positions in one launch.

    ``query``: (tokens, heads, head_dim) or (batch, tokens, heads, head_dim)
    bf16 or fp32, any strides with contiguous rows (a model's (batch, heads,
    tokens, dim) tensor goes in as ``x.transpose(1, 2)``); ``key`` the same
    with its own head count, or None.  ``positions``: int32 or int64, the
    leading shape (tokens,) or (batch, tokens).  ``cos_sin``: an fp32
    (positions, rotary_dim) table (``rotary_table``); its width rotary_dim may
    be less than head_dim: the channels after it are copied.  Pair i of the
    rotary channels is (i, i + rotary_dim / 2), or (2i, 2i + 1) with
    ``interleaved``.  ``inverse`` negates the sines: the transposed map, which is the
    backward pass, and which undoes a rotation where the table's amplitude is 1 (with
    amplitude a the two give a^2 times the rows).  A position outside the table
    gives NaN in the rotary channels.

    Returns (query, key) in new tensors, or the arguments themselves when
    ``in_place`` (rows must then not overlap).  Differentiable in query and
    key, backward and forward, either one more launch; a ``cos_sin`` that
    requires a gradient is refused.
    """
    shape, dtype, device = query.shape, query.dtype, query.device
    lead, dim = shape[:-2], shape[-1]
    if len(shape) not in (3, 4):
        raise ValueError("query must have shape ([batch,] tokens, heads, head_dim)")
    if not query.is_cuda:
        require_cuda_tensor(query, "query")
    if dtype not in _DTYPES:
        raise TypeError("apply_rotary takes BF16 or FP32 queries and keys")
    if dim % 2 or not 2 <= dim <= 1024:
        raise ValueError("head_dim must be even and at most 1024")
    if key is not None:
        other = key.shape
        if other[:-2] != lead or other[-1] != dim or key.device != device:
            raise ValueError("key must match the query but for its heads")
        if key.dtype != dtype:
            raise TypeError("query and key must have the same dtype")
    if positions.shape != lead or positions.device != device:
        raise ValueError("positions must be ([batch,] tokens) on the query's device")
    if positions.dtype not in _POSITIONS:
        raise TypeError("positions must be int32 or int64")
    check_table(cos_sin, dim, device)
    if (cos_sin.requires_grad and torch.is_grad_enabled()) or _is_dual(cos_sin):
        raise ValueError("apply_rotary has no gradient for cos_sin: detach it")
    if (torch.is_grad_enabled() and (query.requires_grad
                                     or (key is not None and key.requires_grad))
            or _is_dual(query) or _is_dual(key)):
        if in_place:
            raise ValueError("rows that require a gradient or carry a tangent cannot be rotated "
                             "in place")
        out = _Rotary.apply(query, key, positions, cos_sin, interleaved, inverse)
        return out if key is not None else (out, None)
    if in_place:
        for rows in (query, key):
            if rows is not None and any(s == 0 and n > 1
                                        for s, n in zip(rows.stride(), rows.shape)):
                raise ValueError("overlapping rows cannot be rotated in place")
    out = _launch(query, key, positions, cos_sin, interleaved, inverse, in_place)
    if in_place:
        mark_written(query, key)
    return out
