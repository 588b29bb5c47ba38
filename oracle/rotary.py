"""Rotary positions in 64 bits, as a product of complex numbers."""

from __future__ import annotations

import numpy as np


def rotated(x: np.ndarray, positions: np.ndarray, frequencies: np.ndarray, interleaved: bool, factor: float) -> np.ndarray:
    """``x [tokens, heads, D]`` with its first ``2 len(frequencies)`` elements turned."""
    half = len(frequencies)
    turn = factor * np.exp(1j * (positions.astype(np.float64)[:, None] * frequencies[None]))[:, None]
    out = x.astype(np.float64).copy()
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = (out[..., one] + 1j * out[..., two]) * turn
    out[..., one], out[..., two] = z.real, z.imag
    return out
