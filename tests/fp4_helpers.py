"""Pools of 4 bits from their definition, in 64 bits: tables of the numbers, nearest by comparison."""

import torch

#: The sizes of codes 0..7 and the e4m3 numbers of scale bytes 0..0x7e.
LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
SCALES = torch.tensor([(b % 8) / 8 * 2.0 ** -6 if b < 8 else (1 + b % 8 / 8) * 2.0 ** (b // 8 - 7)
                       for b in range(0x7f)], dtype=torch.float64)
NAN_SCALE = 0x7f


def nearest(x, table):
    """Index of the table's entry nearest to x >= 0, ties to the even index, beyond the last: the last."""
    table = table.to(x.device)
    mids = (table[:-1] + table[1:]) / 2
    i = torch.searchsorted(mids, x.contiguous())  # mids below x
    tie = (i < len(mids)) & (x == mids[i.clamp(max=len(mids) - 1)])
    return i + (tie & (i % 2 == 1)).long()


def quantise(x):
    """(..., dim) fp32 -> (codes (..., dim / 2), scales (..., dim / 16)) uint8."""
    block = x.double().unflatten(-1, (-1, 16))
    most = block.abs().amax(-1)  # NaN where there is one
    bad = ~most.isfinite()
    most = most.masked_fill(bad, 0.0)
    scale = nearest(most / torch.full_like(most, 6.0), SCALES)
    by = SCALES.to(x.device)[scale]
    size = block.abs() / torch.where(by == 0, torch.inf, by)[..., None]
    code = nearest(size.nan_to_num(0.0), LEVELS) + 8 * torch.signbit(block)
    code = code.masked_fill(bad[..., None], 0).flatten(-2)
    scale = scale.masked_fill(bad, NAN_SCALE)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale.to(torch.uint8)


def values(codes, scales):
    """The numbers they stand for, fp64 (exact)."""
    code = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    level = LEVELS.to(codes.device)[code % 8]
    level = torch.where(code >= 8, -level, level).unflatten(-1, (-1, 16))
    table = torch.cat([SCALES, torch.tensor([torch.nan], dtype=torch.float64)]).to(codes.device)
    return (level * table[scales.long()][..., None]).flatten(-2)


def parts(pool):
    """Views (pages, heads, block, dim / 2) and (pages, heads, block, dim / 16) of a pool's bytes."""
    pages, heads, block, row = pool.shape
    dim = row * 16 // 9
    flat = pool.view(pages, heads, -1) if pool.is_contiguous() else pool.flatten(2)
    return (flat[..., : block * dim // 2].unflatten(-1, (block, -1)),
            flat[..., block * dim // 2:].unflatten(-1, (block, -1)))


def fill(pool, x):
    """Holds (pages, heads, block, dim) numbers in a contiguous pool; returns what it stands for."""
    held = quantise(x)
    for part, new in zip(parts(pool), held):
        part.copy_(new)
    return values(*held)
