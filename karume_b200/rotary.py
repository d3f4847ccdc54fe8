"""Rotation angles for kq_rope, kq_cache_append and kq_cache_attention: the frequencies of a decoder's rotary positions,
scaled for long contexts where it was trained to be, and the (cos, sin) table of them.  Host arithmetic in 64 bits; the
kernels read the f32 table, so queries and keys meet with the same angles whatever kernel rotates them."""
from __future__ import annotations

import math

import numpy as np


def rope_frequencies(rotary: int, base: float = 10000.0, scaling: "dict | None" = None):
    """(frequencies f64 [rotary / 2], amplitude) of a rotation over `rotary` values: f_i = base^(-2 i / rotary).

    scaling, for a context `factor` times the trained one:
      {"kind": "linear", "factor"}                 every frequency divided by factor (positions interpolated)
      {"kind": "base", "factor"}                   the base raised so that the slowest pair is divided by factor and the
                                                   fastest stays: base * factor^(rotary / (rotary - 2))
      {"kind": "ramp", "factor", "trained", "slow", "fast", "over", "amplitude"}
          pairs that turn at most `slow` times over the `trained` positions are divided by factor, those that turn at least
          `fast` times stay, in between the two are mixed linearly over the number of turns (over="turns") or over the
          pair's index (over="index", its ends rounded outwards to whole pairs); amplitude multiplies cos and sin
          (default: 1 for "turns", 1 + 0.1 ln factor for "index").
    """
    if rotary < 2 or rotary % 2:
        raise ValueError(f"rotary {rotary} must be even and positive")
    i = np.arange(rotary // 2, dtype=np.float64)
    f = float(base) ** (-2.0 * i / rotary)
    if scaling is None:
        return f, 1.0
    kind, factor = scaling["kind"], float(scaling["factor"])
    if not factor >= 1.0:
        raise ValueError(f"factor {factor} must be at least one")
    if kind == "linear":
        return f / factor, 1.0
    if kind == "base":
        return (float(base) * factor ** (rotary / max(rotary - 2, 1))) ** (-2.0 * i / rotary), 1.0
    if kind != "ramp":
        raise ValueError(f"scaling kind {kind!r}: 'linear', 'base' or 'ramp'")
    trained, slow, fast = float(scaling["trained"]), float(scaling["slow"]), float(scaling["fast"])
    if not fast > slow > 0:
        raise ValueError("a ramp needs fast > slow > 0 turns")
    if scaling.get("over", "turns") == "turns":
        keep = np.clip((trained * f / (2.0 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        amplitude = float(scaling.get("amplitude", 1.0))
    elif scaling["over"] == "index":
        def pair(turns):  # the index at which a pair turns so often over the trained positions
            return rotary * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rotary - 1)
        keep = 1.0 - np.clip((i - first) / max(last - first, 1e-3), 0.0, 1.0)
        amplitude = float(scaling.get("amplitude", 1.0 + 0.1 * math.log(factor)))
    else:
        raise ValueError(f"over {scaling['over']!r}: 'turns' or 'index'")
    return f / factor * (1.0 - keep) + f * keep, amplitude


def rope_table(positions: int, rotary: int, base: float = 10000.0, scaling: "dict | None" = None) -> np.ndarray:
    """f32 [positions, rotary / 2, 2]: amplitude * (cos, sin)(position * frequency), computed in 64 bits."""
    f, amplitude = rope_frequencies(rotary, base, scaling)
    angle = np.arange(positions, dtype=np.float64)[:, None] * f
    return (amplitude * np.stack([np.cos(angle), np.sin(angle)], -1)).astype(np.float32)
