"""The block-scaled 8-bit cache by its definition -- test infrastructure only.

Codes are e4m3 (``oracle.numerics``); every block and head has a key and a value scale, a power of
two 2^e with -40 <= e <= 80 or 0 for a block of nothing but zeros. Pinned in
``tests/test_block_scaled_host.py``.
"""

from __future__ import annotations

import math

import numpy as np

from oracle.numerics import e4m3_to_f32, f32_to_e4m3

__all__ = ["decode", "empty", "least_scale", "store"]

LEAST, MOST = -40, 80


def least_scale(amax: float) -> float:
    """The least 2^e, -40 <= e <= 80, with ``amax <= 448 * 2^e`` (the largest where none has); 0 for 0."""
    if amax == 0.0:
        return 0.0
    e = LEAST
    while e < MOST and amax > math.ldexp(448.0, e):
        e += 1
    return math.ldexp(1.0, e)


def empty(num_blocks: int, block_size: int, kv_heads: int, head_dim: int) -> tuple[np.ndarray, np.ndarray]:
    """A fresh cache of one tensor: NaN codes [blocks, positions, heads, elements], scales [blocks, heads] of 0."""
    return (np.full((num_blocks, block_size, kv_heads, head_dim), 0x7F, dtype=np.uint8),
            np.zeros((num_blocks, kv_heads), dtype=np.float64))


def _encode(x: np.ndarray, scale: float) -> np.ndarray:
    """e4m3(x / scale): magnitudes above 448 saturate, what is not finite is NaN."""
    y = np.clip(x.astype(np.float64) / (scale or 1.0), -448.0, 448.0)
    # a quotient below 2^-40 rounds to code 0 whatever it is; float32 holds the rest exactly
    return f32_to_e4m3(np.where(np.isfinite(x), y, np.nan).astype(np.float32))


def store(rows: np.ndarray, slots: np.ndarray, codes: np.ndarray, scales: np.ndarray) -> None:
    """Write ``rows`` [N, heads, elements] (float32) into slots of one tensor's cache, in place."""
    num_blocks, block_size, heads, _ = codes.shape
    by_block: dict[int, list[tuple[int, int]]] = {}
    for i, slot in enumerate(np.asarray(slots).tolist()):
        if block_size <= slot < num_blocks * block_size:
            by_block.setdefault(slot // block_size, []).append((slot % block_size, i))
    for block, written in by_block.items():
        first = min(offset for offset, _ in written)
        for h in range(heads):
            x = np.stack([rows[i, h] for _, i in written])
            finite = np.abs(x[np.isfinite(x)])
            old = float(scales[block, h]) if first else 0.0
            new = max(old, least_scale(float(finite.max()) if finite.size else 0.0))
            if new > old > 0.0:
                held = e4m3_to_f32(codes[block, :first, h]) * np.float32(old / new)
                codes[block, :first, h] = f32_to_e4m3(held)
            for (offset, _), row in zip(written, x):
                codes[block, offset, h] = _encode(row, new)
            scales[block, h] = new


def decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """What the cache is worth: float64 [blocks, positions, heads, elements]."""
    return e4m3_to_f32(codes).astype(np.float64) * scales[:, None, :, None]
