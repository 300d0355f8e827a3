"""Rotary frequencies for ``kudacuda_rope`` and ``kudacuda_rope_paged_append``.

The kernels take any table of frequencies (float64, one per pair of dims) and an
amplitude, so every way to stretch a model's positions over a longer context is a
table made here once: plain, position interpolation (``linear``), a larger base
(``ntk``) and interpolation by wavelength (``yarn``).
"""

from __future__ import annotations

import math

import numpy as np

SCALINGS = ("none", "linear", "ntk", "yarn")


def rope_frequencies(rotary_dim: int, theta: float = 1.0e6, *, scaling: str = "none", factor: float = 1.0,
                     original_positions: int = 32768, slow: float = 1.0,
                     fast: float = 32.0) -> tuple[np.ndarray, float]:
    """(inv_freq float64 [rotary_dim / 2], amplitude): pair i of a token at position p turns by p * inv_freq[i].

    ``factor`` is how many times longer the context becomes.  ``linear`` divides
    every frequency by it.  ``ntk`` raises the base so that the slowest pair is
    divided by it and the fastest is kept.  ``yarn`` (Peng et al., 2023) keeps the
    pairs that turn more than ``fast`` times over ``original_positions``, divides
    those that turn less than ``slow`` times, goes from one to the other linearly in
    the pair's number between (from the last whole number before the one limit to the
    first behind the other: what models of that configuration run, where the paper's
    text goes linearly in the turns), and multiplies the rows by 0.1 ln(factor) + 1."""

    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError("rotary_dim must be even and at least 2")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if not (math.isfinite(factor) and factor >= 1.0 and theta > 0.0):
        raise ValueError("factor must be at least 1 and theta positive")
    exponent = np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim
    inv_freq = theta ** -exponent
    if scaling == "linear":
        return inv_freq / factor, 1.0
    if scaling == "ntk":
        # theta' ^ e with e the last pair's exponent is factor * theta ^ e
        last = exponent[-1]
        return inv_freq if last == 0 else (theta * factor ** (1.0 / last)) ** -exponent, 1.0
    if scaling == "yarn":
        if not (0.0 < slow < fast and original_positions > 0 and theta > 1.0):
            raise ValueError("yarn needs 0 < slow < fast, original_positions and theta > 1")

        def pair(turns: float) -> float:
            # theta ^ (-2 i / rotary_dim) * original_positions = 2 pi turns
            return rotary_dim * math.log(original_positions / (2.0 * math.pi * turns)) / (2.0 * math.log(theta))

        first = max(math.floor(pair(fast)), 0)
        last = min(math.ceil(pair(slow)), rotary_dim - 1)
        # (nothing between the limits: the pairs up to the first are kept)
        ramp = np.clip((np.arange(rotary_dim // 2) - first) / max(last - first, 0.001), 0.0, 1.0)
        return inv_freq * (1.0 - ramp + ramp / factor), 0.1 * math.log(factor) + 1.0
    return inv_freq, 1.0
