"""Rotary positions and attention over latent caches, by their definitions, in float64."""

from __future__ import annotations

import numpy as np

__all__ = ["attention", "chunk_attention", "positions_and_slots", "rotate"]


def rotate(x: np.ndarray, positions: np.ndarray, turns: np.ndarray, interleaved: bool, magnitude: float) -> np.ndarray:
    """Rows ``x`` [N, heads, width] with their first ``2 * len(turns)`` elements turned: pair i of row n
    by ``positions[n] * turns[i]`` full turns, as complex numbers."""
    x = np.array(x, dtype=np.float64)
    pairs = len(turns)
    first = np.arange(pairs) * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    fraction = np.remainder(np.asarray(positions, dtype=np.float64)[:, None] * np.asarray(turns)[None, :], 1.0)
    turned = (x[..., first] + 1j * x[..., second]) * (magnitude * np.exp(2j * np.pi * fraction))[:, None, :]
    x[..., first], x[..., second] = turned.real, turned.imag
    return x


def positions_and_slots(rows, lengths, table: np.ndarray, block: int) -> tuple[np.ndarray, np.ndarray]:
    """Every row's position and slot; 0 for a request without tokens."""
    positions, slots = [], []
    for b, (count, length) in enumerate(zip(rows, lengths)):
        for j in range(count):
            t = length - count + j if length else 0
            positions.append(t)
            slots.append(int(table[b, t // block]) * block + t % block if length else 0)
    return np.array(positions, dtype=np.int64), np.array(slots, dtype=np.int64)


def _weights(scores: np.ndarray) -> np.ndarray:
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.exp(scores - scores.max(axis=-1, keepdims=True))
        return e / e.sum(axis=-1, keepdims=True)


def _attend(q, keys, values, count, length, scale):
    """One head: q [count, w], keys [length, w], values [length, d] -> out, sum of weighted magnitudes of
    the values, and the largest |q||k| summed over a row's visible scores. Row j sees positions up to
    ``length - count + j``, and nothing of the others reaches it."""
    out = np.zeros((count, values.shape[1]))
    size, reach = np.zeros_like(out), np.zeros((count, 1))
    with np.errstate(invalid="ignore", over="ignore"):
        for j in range(count):
            seen = length - count + j + 1
            p = _weights(scale * (keys[:seen] @ q[j]))
            out[j], size[j] = p @ values[:seen], p @ np.abs(values[:seen])
            reach[j] = abs(scale) * (np.abs(keys[:seen]) @ np.abs(q[j])).max()
    return out, size, reach


def _requests(cache, table, rows, lengths):
    block, first = cache.shape[1], 0
    for b, (count, length) in enumerate(zip(rows, lengths)):
        if count and length:
            t = np.arange(length)
            yield first, count, length, np.asarray(cache[table[b, t // block], t % block], dtype=np.float64)
        first += count


def attention(q, cache, table, rows, lengths, scale, latent):
    """Absorbed form: out [N, heads, latent], and for error bounds the sums of weighted magnitudes (the
    same shape) and each row's largest sum of |q||k| times the scale [N, heads, 1]."""
    q = np.asarray(q, dtype=np.float64)
    out = np.zeros((*q.shape[:2], latent))
    size, reach = np.zeros_like(out), np.zeros((*q.shape[:2], 1))
    for first, count, length, x in _requests(cache, table, rows, lengths):
        for h in range(q.shape[1]):
            at = slice(first, first + count)
            out[at, h], size[at, h], reach[at, h] = _attend(q[at, h], x, x[:, :latent], count, length, scale)
    return out, size, reach


def chunk_attention(q, keys, values, cache, table, rows, lengths, scale):
    """Expanded form: the same three with ``keys`` [heads, nope, latent], ``values`` [heads, value, latent]."""
    q, keys, values = (np.asarray(x, dtype=np.float64) for x in (q, keys, values))
    latent = keys.shape[2]
    out = np.zeros((*q.shape[:2], values.shape[1]))
    size, reach = np.zeros_like(out), np.zeros((*q.shape[:2], 1))
    for first, count, length, x in _requests(cache, table, rows, lengths):
        for h in range(q.shape[1]):
            at = slice(first, first + count)
            with np.errstate(invalid="ignore"):
                k, v = x[:, :latent] @ keys[h].T, x[:, :latent] @ values[h].T
            out[at, h], size[at, h], reach[at, h] = _attend(q[at, h], np.concatenate((k, x[:, latent:]), axis=1), v,
                                                            count, length, scale)
    return out, size, reach
