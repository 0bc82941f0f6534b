"""Frequencies of a position rotation, for contexts of the length a model was
trained on and longer ones. No counterpart in the reference, whose runtime leaves
attention to the framework."""

from __future__ import annotations

import math

import torch

METHODS = ("none", "linear", "base", "parts")


def rotary_frequencies(rotary: int, base: float = 10000.0, method: str = "none", factor: float = 1.0, context: int = 8192,
                       slow: float = 1.0, fast: float = 32.0, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq FP32 [rotary / 2], scale) for `PagedKvCache.append` and `rotate_heads`: base^(-2 i / rotary), and for
    a context `factor` times the `context` tokens a model was trained on

      "linear"  all divided by factor (positions interpolated)
      "base"    base times factor^(rotary / (rotary - 2)): the slowest divided by factor, the fastest as it was
      "parts"   those that turn less than `slow` times over `context` divided by factor, those that turn more than `fast`
                times as they were, what lies between linearly in its turns; and sine and cosine times 0.1 ln(factor) +
                1, the scale (1.0 with the others)

    In 64 bits, rounded once."""
    if int(rotary) != rotary or rotary < 8 or rotary % 8:
        raise ValueError(f"rotary must be a multiple of 8, got {rotary}")
    if method not in METHODS:
        raise ValueError(f"method must be one of {METHODS}, got {method!r}")
    if not (base > 1 and math.isfinite(base) and factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"base must be above 1 and factor 1 or more, got {base}, {factor}")
    if method == "parts" and not (context > 0 and 0 <= slow < fast):
        raise ValueError("context must be above 0 and slow below fast")
    if method == "base":
        power = rotary / (rotary - 2)
        if math.log(base) + power * math.log(factor) > 709.0:
            raise ValueError(f"base times factor^{power:.3g} must be below e^709, got {base}, {factor}")
        base *= factor ** power
    freq = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    scale = 1.0
    if method == "linear":
        freq = freq / factor
    elif method == "parts":
        turns = context * freq / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / factor)
        scale = 0.1 * math.log(factor) + 1.0
    return freq.float().to(device), scale
