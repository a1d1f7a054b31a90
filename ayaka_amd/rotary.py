"""Rotary positions: which pairs of a head's elements turn, and how far per position.

Pair ``i`` of the first ``dim`` elements of a head turns by ``position * base ** (-2 i / dim)`` radians,
or by a frequency that a scaling changed for contexts longer than the model was trained on:

* :class:`LinearScaling` divides every frequency by ``factor``;
* :class:`BandScaling` keeps pairs whose wavelength is under ``original_length / high``, divides those
  over ``original_length / low`` by ``factor`` and blends between (the "llama3" rule);
* :class:`YarnScaling` keeps pairs that turn more than ``fast`` times within ``original_length``, divides
  those that turn less than ``slow`` times, with a ramp over the pairs between, and multiplies
  cosines and sines by ``magnitude`` (0.1 ln(factor) + 1 where not given).

:func:`rotary` makes the record that ``kvcache.rotate``, ``store_rotated`` and ``store_latent`` take.
Importing this module does not import torch.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import TYPE_CHECKING, NamedTuple

if TYPE_CHECKING:
    import torch
    from torch import Tensor

__all__ = ["BandScaling", "LinearScaling", "Rotary", "YarnScaling", "rotary"]


def _require_positive(name: str, value: float) -> None:
    if not (math.isfinite(value) and value > 0):
        raise ValueError(f"{name} must be positive and finite, got {value!r}")


@dataclass(frozen=True, slots=True)
class LinearScaling:
    factor: float

    def __post_init__(self) -> None:
        _require_positive("factor", self.factor)

    def frequencies(self, plain: list[float], dim: int, base: float) -> list[float]:
        return [f / self.factor for f in plain]


@dataclass(frozen=True, slots=True)
class BandScaling:
    factor: float
    original_length: int
    low: float = 1.0
    high: float = 4.0

    def __post_init__(self) -> None:
        for name in ("factor", "original_length", "low"):
            _require_positive(name, getattr(self, name))
        if not self.high > self.low:
            raise ValueError(f"high must be above low, got {self.high!r} and {self.low!r}")

    def frequencies(self, plain: list[float], dim: int, base: float) -> list[float]:
        out = []
        for f in plain:
            turns = self.original_length * f / (2 * math.pi)  # within the original length
            keep = min(1.0, max(0.0, (turns - self.low) / (self.high - self.low)))
            out.append(f * (keep + (1.0 - keep) / self.factor))
        return out


@dataclass(frozen=True, slots=True)
class YarnScaling:
    factor: float
    original_length: int
    fast: float = 32.0
    slow: float = 1.0
    magnitude: float | None = None

    def __post_init__(self) -> None:
        for name in ("factor", "original_length", "slow"):
            _require_positive(name, getattr(self, name))
        if not self.fast > self.slow:
            raise ValueError(f"fast must be above slow, got {self.fast!r} and {self.slow!r}")

    def frequencies(self, plain: list[float], dim: int, base: float) -> list[float]:
        def pair_turning(turns: float) -> float:
            return dim * math.log(self.original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(0, math.floor(pair_turning(self.fast)))
        high = min(dim - 1, math.ceil(pair_turning(self.slow)))
        span = max(high - low, 0.001)
        out = []
        for i, f in enumerate(plain):
            stretch = min(1.0, max(0.0, (i - low) / span))
            out.append(f * (1.0 - stretch + stretch / self.factor))
        return out


class Rotary(NamedTuple):
    """A rotation of ``2 * len(turns)`` elements: ``turns`` float64 [pairs] on the device, full turns
    per position of each pair; ``interleaved`` pairs elements 2i and 2i + 1, else i and i + pairs;
    cosines and sines are multiplied by ``magnitude``. Make one with :func:`rotary`."""

    turns: Tensor
    interleaved: bool
    magnitude: float


def rotary(
    dim: int,
    *,
    base: float = 10000.0,
    interleaved: bool = False,
    scaling: LinearScaling | BandScaling | YarnScaling | None = None,
    device: "torch.device | str",
) -> Rotary:
    """The rotation of the first ``dim`` elements of a head."""
    import torch

    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and positive, got {dim}")
    if not (math.isfinite(base) and base > 1):
        raise ValueError(f"base must be above 1 and finite, got {base!r}")
    frequencies = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    magnitude = 1.0
    if scaling is not None:
        frequencies = scaling.frequencies(frequencies, dim, base)
        if isinstance(scaling, YarnScaling):
            magnitude = 0.1 * math.log(scaling.factor) + 1.0 if scaling.magnitude is None else scaling.magnitude
            if scaling.magnitude is None and scaling.factor <= 1.0:
                magnitude = 1.0
    turns = torch.tensor([f / (2 * math.pi) for f in frequencies], dtype=torch.float64, device=device)
    return Rotary(turns, bool(interleaved), float(magnitude))
