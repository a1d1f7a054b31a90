"""Attention over latent caches whose values, scores and weights span wide ranges, against float64.

The bounds are :class:`Scene`'s (``tests/test_gpu_latent.py``) where it checks. What a test derives
itself stands at the test.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, ForwardMode
from ayaka_amd.hip import latent as hip_latent
from tests.test_gpu_latent import DEV, TYPES, Scene

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


@pytest.fixture(params=[1, 2, 5])
def parts(request, monkeypatch) -> int:
    """The parts that chunks' contexts are cut into."""
    monkeypatch.setattr(hip_latent, "_chunk_splits", lambda *_: request.param)
    return request.param


def resize(s: Scene, request: int, sizes) -> None:
    """The latents and key parts of each 128 positions of a request, multiplied."""
    t = np.arange(s.lengths[request])
    by = torch.tensor(np.asarray(sizes, dtype=np.float64)[t // 128]).to(DEV)
    at = torch.as_tensor(s.table[request, t // s.block]), torch.as_tensor(t % s.block)
    s.cache[at] = (s.cache[at].double() * by[:, None]).to(s.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [
    [1.0, 64.0, 2.0 ** -8, 2.0 ** 9, 1.0, 2.0 ** -20, 32.0, 0.0],
    [1.0, 0.0, 1.0, 1.0, 0.0, 1.0, 0.0, 1.0],   # tiles of zeros, first, between and last
    [0.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 0.0],
    [2.0 ** 11, 1.0, 2.0 ** -11, 2.0 ** -13, 1.0, 2.0 ** -9, 2.0 ** -12, 1.0],
])
def test_every_position_counts_in_the_sum_of_weights(ops, parts, dtype, sizes) -> None:
    """Tiles of 128 positions whose values are far below others', or zeros, weigh as much as any."""
    s = Scene(ops, [(3, 900)], form="chunks", heads=2, dtype=dtype, seed=51, q_scale=0.05)
    resize(s, 0, sizes)
    s.check()
