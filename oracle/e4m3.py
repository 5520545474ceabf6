"""A cache of 8-bit floats with a power of two as the scale of each block and head, in float64 NumPy.

e4m3: one sign, four exponent and three mantissa bits, bias 7, no infinities, largest 448. The reference's cache is
float32 (src/paged_kv_serving/engine/runner.py:112-114, 195-196); slots and blocks are as there.
"""

from __future__ import annotations

import numpy as np

__all__ = ["LARGEST", "LOW_SCALE", "append", "block_scale", "nearest", "values"]

LARGEST = 448.0
LOW_SCALE = 2.0**-100


def nearest(x) -> np.ndarray:
    """The e4m3 number nearest to each number, ties to the one with an even last bit; what is not finite, NaN."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        exponent = np.frexp(np.where(np.isfinite(x), x, 0.0))[1] - 1  # 2^exponent <= |x| < 2^(exponent + 1)
        step = np.exp2(np.maximum(exponent, -6) - 3.0)  # below 2^-6 the steps stay 2^-9
        out = np.round(x / step) * step  # np.round: ties to even
    return np.where(np.abs(out) <= LARGEST, out, np.nan)


def block_scale(most: float) -> float:
    """The smallest power of two, LOW_SCALE at least, times which LARGEST is no less than ``most``."""
    scale = LOW_SCALE
    while LARGEST * scale < most:
        scale *= 2.0
    return scale


def append(codes: np.ndarray, scales: np.ndarray, new, slots) -> None:
    """``new [T, kv_heads, dim]`` into ``codes [blocks, block, kv_heads, dim]`` (their values as numbers) and
    ``scales [blocks, kv_heads]``, in place, block after block."""
    new, (blocks, size) = np.asarray(new, np.float64), codes.shape[:2]
    slots = np.asarray(slots)
    inside = (slots >= 0) & (slots < blocks * size)
    for block in np.unique(slots[inside] // size):
        tokens = np.flatnonzero(inside & (slots // size == block))
        before = int((slots[tokens] % size).min())
        for head in range(codes.shape[2]):
            rows = new[tokens, head]
            scale = block_scale(np.abs(rows[np.isfinite(rows)]).max(initial=0.0))
            if before > 0:
                held = scales[block, head]
                scale = max(scale, held)
                if scale != held:
                    codes[block, :before, head] = nearest(codes[block, :before, head] * (held / scale))
            scales[block, head] = scale
            codes[block, slots[tokens] % size, head] = nearest(rows / scale)


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """What codes stand for."""
    return codes * np.asarray(scales, np.float64)[:, None, :, None]
