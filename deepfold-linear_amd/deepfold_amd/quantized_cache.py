"""A rolling cache held in 8 or 4 bits: what ``window_cache_fill``, ``window_cache_read`` and ``window_decode_attn`` take
in place of a bf16 or fp32 cache.

32 elements of a row form a group (the last one of a row filled up with zeros) that shares a power of two,
2 ** (E - 127) with the exponent byte E; an element stands for its code times that.  8 bits: the code is an integer from
-127 to 127.  4 bits: one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, the even element in a byte's low half.  E is the
lowest, from 1 on, with which the group's largest magnitude is below 127.5 (8 bits) or at most 7 (4 bits) times the power,
so every element is off by at most half a step: of normally distributed rows 0.7 % of their size in 8 bits, 12 % in 4.
(E is at most 248 and 252, so that all values are finite: of groups that reach 2 ** 127 the largest take the last code.)
A group that holds an infinity or NaN reads as NaN.  A row of 128 elements takes 132 or 68 bytes, where bf16 takes 256.

These are element formats that gfx950 converts in one instruction, and powers of two keep every step but the rounding
to a code exact: the codes are the same whoever forms them.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

GROUP = 32


class QuantizedCache(NamedTuple):
    """Keys or values of a rolling cache in few bits (module docstring); ``quantized_cache`` makes one.

    codes (B,Hk,slots,groups * 4 * bits) uint8, the rows 16-byte aligned; exponents (B,Hk,groups,n) uint8, n a multiple of 4
    from slots on (what lies behind the last slot is of no meaning); any strides over B and heads."""

    codes: torch.Tensor
    exponents: torch.Tensor
    bits: int


def groups_of(d: int) -> int:
    return -(-d // GROUP)


def quantized_cache(B: int, Hk: int, slots: int, D: int, *, bits: int, device=None) -> QuantizedCache:
    """An empty cache of ``slots`` (n_sink + window) rows of D elements in 8 or 4 bits, for keys or for values."""
    if bits not in (4, 8):
        raise ValueError(f"quantized_cache: bits={bits} must be 4 or 8")
    if min(B, Hk, slots, D) < 1:
        raise ValueError(f"quantized_cache: sizes must be positive, got {(B, Hk, slots, D)}")
    device = "cuda" if device is None else device
    groups = groups_of(D)
    return QuantizedCache(torch.zeros(B, Hk, slots, groups * 4 * bits, dtype=torch.uint8, device=device),
                          torch.zeros(B, Hk, groups, -(-slots // 16) * 16, dtype=torch.uint8, device=device), bits)
