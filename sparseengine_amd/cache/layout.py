"""How keys and values lie inside a page, seen from Python.

A cache layer is ``[pages, 2 (keys, values), kv_heads, page_size, head_dim]``; the last two sizes
give a page's geometry, not the order of its elements.  Inside a kv head's page plane the elements
lie in groups of eight, so that sixteen lanes of a matrix-core operand load read one contiguous
stretch (``key_place`` / ``value_place`` in csrc/common.h):

    keys    [head_dim / 8][page_size][8]     eight dims of one key side by side, keys next to each other
    values  [page_size / 8][head_dim][8]     eight keys of one dim side by side, dims next to each other

``keys_view`` and ``values_view`` give strided views in which a key and a dim can be addressed; the
kernels never use them, tests and the kernel twins do.  ``page_size`` and ``head_dim`` are multiples
of 8.
"""
from __future__ import annotations

import torch


def keys_view(cache: torch.Tensor) -> torch.Tensor:
    """``[pages, kv_heads, page_size, head_dim / 8, 8]``: element ``[p, h, key, d // 8, d % 8]``."""
    pages, _, kv_heads, page_size, head_dim = cache.shape
    return cache[:, 0].reshape(pages, kv_heads, head_dim // 8, page_size, 8).permute(0, 1, 3, 2, 4)


def values_view(cache: torch.Tensor) -> torch.Tensor:
    """``[pages, kv_heads, page_size / 8, 8, head_dim]``: element ``[p, h, key // 8, key % 8, d]``."""
    pages, _, kv_heads, page_size, head_dim = cache.shape
    return cache[:, 1].reshape(pages, kv_heads, page_size // 8, head_dim, 8).permute(0, 1, 2, 4, 3)


def read_keys(cache: torch.Tensor, pages: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Keys at (page, offset) pairs: ``[n, kv_heads, head_dim]``."""
    return keys_view(cache)[pages, :, offsets].reshape(pages.numel(), cache.shape[2], cache.shape[4])


def read_values(cache: torch.Tensor, pages: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Values at (page, offset) pairs: ``[n, kv_heads, head_dim]``."""
    return values_view(cache)[pages, :, offsets // 8, offsets % 8]


def write_keys(cache: torch.Tensor, pages: torch.Tensor, offsets: torch.Tensor, keys: torch.Tensor) -> None:
    """``keys``: ``[n, kv_heads, head_dim]``."""
    keys_view(cache)[pages, :, offsets] = keys.reshape(pages.numel(), cache.shape[2], cache.shape[4] // 8, 8)


def write_values(cache: torch.Tensor, pages: torch.Tensor, offsets: torch.Tensor, values: torch.Tensor) -> None:
    """``values``: ``[n, kv_heads, head_dim]``."""
    values_view(cache)[pages, :, offsets // 8, offsets % 8] = values.reshape(pages.numel(), cache.shape[2], cache.shape[4])


# ---------------------------------------------------------------------------------------------- 4 bits
# A 4-bit layer is uint8 [pages, 2, kv_heads, page_size, head_dim * 17 / 32]; a kv head's part of a page holds two
# codes to a byte, then one factor byte for every 32 neighbouring dims (G = head_dim / 32; csrc/fp4.h has the format
# and the reasons):
#
#     keys    codes [G][page_size][16]             factors [G][page_size]
#     values  codes [page_size / 8][16][G][8]      factors [page_size / 8][G][8]
#
# A code stands for FP4_LEVELS[code % 8], bit 3 is its sign; a factor byte e stands for 2 ** (e - 127), 255 for a
# group that is not a number.  head_dim and page_size are multiples of 32.
FP4_GROUP = 32
FP4_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FP4_NAN = 255


def fp4_row_bytes(head_dim: int) -> int:
    """Bytes of a key or a value in 4 bits, its factors included."""
    if head_dim <= 0 or head_dim % FP4_GROUP:
        raise ValueError(f"4-bit keys and values take head sizes in steps of {FP4_GROUP}, got {head_dim}")
    return head_dim * 17 // 32


def fp4_quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``[..., head_dim]`` -> codes uint8 ``[..., head_dim]`` and factors uint8 ``[..., head_dim / 32]``: the smallest
    factor from 2 ** -125 to 2 ** 125 with ``max |x| <= 7 * factor``, the nearest codes, ties to the even code."""
    groups = x.float().reshape(*x.shape[:-1], x.shape[-1] // FP4_GROUP, FP4_GROUP)
    finite = torch.isfinite(groups).all(-1)
    size = torch.where(finite.unsqueeze(-1), groups.abs(), torch.zeros((), device=x.device))
    top = size.amax(-1)
    mantissa, exponent = torch.frexp(top)                # mantissa in [0.5, 1): 7 = 0.875 * 2 ** 3
    e = torch.where(mantissa <= 0.875, exponent - 3, exponent - 2)
    e = torch.where(top > 0, e, torch.full_like(e, -125)).clamp(-125, 125)
    y = torch.ldexp(size, -e.unsqueeze(-1))
    code = sum((y > edge if even else y >= edge).to(torch.uint8)
               for edge, even in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)))
    code = code + torch.signbit(groups).to(torch.uint8) * 8
    factors = torch.where(finite, e + 127, torch.full_like(e, FP4_NAN)).to(torch.uint8)
    return code.reshape(x.shape), factors


def fp4_values(codes: torch.Tensor, factors: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """What codes ``[..., head_dim]`` under factors ``[..., head_dim / 32]`` stand for."""
    levels = torch.tensor(FP4_LEVELS + tuple(-v for v in FP4_LEVELS), dtype=dtype, device=codes.device)
    scale = torch.where(factors == FP4_NAN, torch.full((), float("nan"), dtype=dtype, device=codes.device),
                        torch.exp2(factors.to(dtype) - 127))
    return levels[codes.long()] * scale.repeat_interleave(FP4_GROUP, -1)


def _fp4_parts(cache: torch.Tensor, which: int):
    """Views of a layer's keys (0) or values (1): code bytes ``[pages, kv_heads, page_size, G, 16]`` for keys, ``[pages,
    kv_heads, page_size / 8, 8, G, 16]`` for values, and the factors without the last size."""
    pages, _, kv_heads, page, row = cache.shape
    G = row // 17
    part = cache.view(pages, 2, kv_heads, page * row)[:, which]
    codes, factors = part[..., :page * G * 16], part[..., page * G * 16:]
    if which == 0:
        return (codes.view(pages, kv_heads, G, page, 16).permute(0, 1, 3, 2, 4),
                factors.view(pages, kv_heads, G, page).permute(0, 1, 3, 2))
    return (codes.view(pages, kv_heads, page // 8, 16, G, 8).permute(0, 1, 2, 5, 4, 3),
            factors.view(pages, kv_heads, page // 8, G, 8).permute(0, 1, 2, 4, 3))


def fp4_read(cache: torch.Tensor, which: int, pages: torch.Tensor, offsets: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """Keys (``which`` 0) or values (1) at (page, offset) pairs: ``[n, kv_heads, head_dim]``."""
    codes, factors = _fp4_parts(cache, which)
    at = (pages, slice(None), offsets) if which == 0 else (pages, slice(None), offsets // 8, offsets % 8)
    two, f = codes[at], factors[at]                                  # [n, kv_heads, G, 16], [n, kv_heads, G]
    return fp4_values(torch.stack([two & 15, two >> 4], -1).flatten(2), f, dtype)


def fp4_write(cache: torch.Tensor, which: int, pages: torch.Tensor, offsets: torch.Tensor, x: torch.Tensor) -> None:
    """``x``: ``[n, kv_heads, head_dim]``, put into 4 bits."""
    codes, factors = _fp4_parts(cache, which)
    code, factor = fp4_quantise(x)
    two = code[..., 0::2] | code[..., 1::2] << 4
    at = (pages, slice(None), offsets) if which == 0 else (pages, slice(None), offsets // 8, offsets % 8)
    codes[at] = two.view(*two.shape[:2], -1, 16)
    factors[at] = factor
