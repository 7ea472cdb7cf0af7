"""Rotary positions on the sm_100a kernel: interleaved and half layouts, part of the
head, scaled for long contexts.

A head's first rotary_dim elements form pairs, (i, i + rotary_dim / 2) or, interleaved,
(2i, 2i + 1); pair i of the token at position t is rotated by t * inv_freq[i] and
multiplied by `magnitude`. Angles are formed and reduced in 64 bits, so far positions
lose nothing. The other elements are copied.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .._ext import C


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none",
                       factor: float = 1.0, original_length: int = 0, fast_turns: float = 32.0,
                       slow_turns: float = 1.0, device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq, magnitude) for apply_rotary: float64 [rotary_dim / 2], and a number.

    scaling "none":   inv_freq[i] = base^(-2i / rotary_dim)
            "linear": all of them over `factor`: positions are interpolated
            "base":   a larger base, base * factor^(d / (d - 2)), d = rotary_dim, which
                      leaves the fastest pair and interpolates the slowest one by `factor`
            "ramp":   by frequency: pairs that turn more than `fast_turns` times within
                      original_length positions stay, those with fewer than `slow_turns`
                      are over `factor`, and between them the share grows linearly with i;
                      magnitude 1 + 0.1 ln(factor)
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if base <= 1.0 or factor < 1.0:
        raise ValueError("base must be above 1 and factor at least 1")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("scaling 'base' needs rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    magnitude = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "ramp":
        if original_length < 1 or not fast_turns > slow_turns > 0:
            raise ValueError("scaling 'ramp' needs original_length and fast_turns > slow_turns > 0")

        def pair_of(turns):  # the (real) index of the pair that turns so often
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(pair_of(fast_turns)), 0)
        high = min(math.ceil(pair_of(slow_turns)), rotary_dim - 1)
        share = (torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)
        share = share.clamp(0, 1)
        inv = inv * (1 - share) + inv / factor * share
        magnitude = 1.0 + 0.1 * math.log(factor)
    elif scaling not in ("none", "base"):
        raise ValueError(f"scaling must be 'none', 'linear', 'base' or 'ramp', got {scaling!r}")
    return inv.to(device) if device is not None else inv, magnitude


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 inv_freq: torch.Tensor, interleaved: bool = False, magnitude: float = 1.0):
    """q and k (k may be None) with rotary positions; differentiable (once, in reverse
    mode) in q and k.

    q, k: [tokens, heads, head_dim] or [batch, tokens, heads, head_dim], bfloat16, float16
    or float32, head_dim up to 256, of one dtype; they may be strided, the results are
    contiguous. positions: int32 or int64 [tokens], or [batch, tokens]. inv_freq:
    float64 [rotary_dim / 2] (rotary_frequencies). Returns (q', k'), or q' alone."""
    qo, ko = C().apply_rotary(q, k, positions, inv_freq, interleaved, magnitude)
    return qo if ko is None else (qo, ko)
