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


def score(s: Scene, request: int, bits) -> None:
    """Scores of one request by its rotary parts alone: position t's weight is 2 ** bits[t] of the one of a
    position of 0 bits (as near as the element type holds it)."""
    s.scale = 1 / 64
    s.q[..., 128 if s.form == "chunks" else s.latent:] = 0
    s.q[..., 128 if s.form == "chunks" else s.latent] = 1
    if s.form == "chunks":
        s.weights.keys.zero_()
    else:
        s.q[..., :s.latent] = 0
    t = np.arange(s.lengths[request])
    at = torch.as_tensor(s.table[request, t // s.block]), torch.as_tensor(t % s.block)
    s.cache[(*at, s.latent)] = torch.tensor(np.asarray(bits, dtype=np.float64) * math.log(2) * 64).to(s.dtype).to(DEV)


@pytest.mark.parametrize("loud_at", [0, 3, 6])
@pytest.mark.parametrize("share", ["none", "as much"])
@pytest.mark.parametrize("dtype,quiet,loud", [("fp16", -6, 13), ("bf16", -12, 12), ("bf16", -20, 20), ("bf16", -60, 70)])
def test_values_that_weigh_nothing_cost_others_nothing(ops, parts, dtype, quiet, loud, share, loud_at) -> None:
    """A tile far louder than the others, whose scores leave it no share of the output, or one like theirs."""
    s = Scene(ops, [(3, 900), (140, 700)], form="chunks", heads=2, dtype=dtype, seed=52)
    rng = np.random.default_rng(53)
    for request, length in enumerate(s.lengths):
        tile = np.arange(length) // 128
        sizes = np.where(np.arange(tile[-1] + 1) == loud_at % (tile[-1] + 1), 2.0 ** loud, 2.0 ** quiet)
        resize(s, request, sizes)
        bits = rng.uniform(-12, 0, length)
        score(s, request, np.where(sizes[tile] == 2.0 ** loud, bits + (-300 if share == "none" else quiet - loud), bits))
    s.check()


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("form,dtype", [("absorbed", "fp16"), ("chunks", "fp16"), ("chunks", "bf16")])
def test_a_long_flat_tail(ops, monkeypatch, form, dtype, first) -> None:
    """One position of nearly all the weight, and 131071 of 2^-26 of it each, which make a share of 2^-9. Contexts
    are not cut: a workgroup has the whole of one (in absorbed form one of as many requests as there are compute
    units, over the same blocks).

    A weight is held to 2^-11 of itself, or 2^-32 of the position's that set the running maximum, which is no more
    than the largest, numerator and denominator alike: 2 n (2^-26 2^-11 + 2^-32) = 2^-13 (1 + 2^-5) of the values' size 1
    (the tail's values are 1 and the other's 0). Beside it the output's rounding, a half step of 2^-9, and (n / 32 + 40) 2^-24 of
    the sums."""
    n, block = 1 << 17, 64
    monkeypatch.setattr(hip_latent, "_chunk_splits", lambda *_: 1)
    requests = 256 if form == "absorbed" else 1
    s = Scene(ops, [(1, 5)] * requests, form=form, dtype=dtype, heads=1, latent=256, block=block, seed=54)
    s.lengths, s.rows = [n] * requests, [1] * requests
    s.table = np.tile(1 + np.arange(n // block), (requests, 1))
    s.cache = torch.zeros(1 + n // block, block, 320, dtype=s.dtype, device=DEV)
    s.cache[..., :256] = 1
    s.meta = ops.attention.plan(ForwardMode.DECODE, torch.tensor(s.rows, device=DEV), torch.tensor(s.lengths, device=DEV),
                                torch.tensor(s.table, device=DEV), block)
    bits = np.random.default_rng(55).uniform(-26.5, -25.5, n)
    most = 0 if first else n - 1
    bits[most] = 0
    score(s, 0, bits)
    s.cache[int(s.table[0, most // block]), most % block, :256] = 0
    if form == "chunks":
        s.weights.values.zero_()
        s.weights.values[..., 0] = 1
    p = np.exp(s.cache[1:][..., 256].reshape(-1).double().cpu().numpy() / 64)
    p[most] = 1
    want = 1 - 1 / p.sum()
    bound = 2.0 ** -13 * (1 + 2.0 ** -5) + want * torch.finfo(s.dtype).eps / 2 + (n / 32 + 40) * 2.0 ** -24 * want
    assert abs(want - 2.0 ** -9) < 2.0 ** -13
    assert float((s.run().double() - want).abs().max()) <= bound


@pytest.mark.parametrize("form", ["absorbed", "chunks"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("step", [16, 32])
def test_scores_a_few_steps_of_their_own_apart(ops, form, dtype, step) -> None:
    """Scores of 2^27, whose neighbours in fp32 are 16 apart: what a score passes by is compared as it is.
    The rows are the last position's values, to 97 weights of 2^-16 (values within 8)."""
    s = Scene(ops, [(1, 98)], form=form, dtype=dtype, heads=2, seed=56)
    at = torch.as_tensor(s.table[0, np.arange(98) // 16]), torch.as_tensor(np.arange(98) % 16)
    if form == "chunks":
        s.weights.keys.zero_()
    s.q.zero_()
    rope = s.latent if form == "absorbed" else 128
    s.q[..., rope], s.q[..., rope + 1] = 2.0 ** 14, 1.0
    s.cache[(*at, s.latent)] = 2.0 ** 13
    s.cache[(*at, s.latent + 1)] = torch.where(torch.arange(98) == 97, 16.0 + step, 16.0).to(s.dtype).to(DEV)
    s.scale = float(np.float32(math.log(2)))  # a power of two a unit of score
    assert np.float32(s.scale) * np.float32(1.4426950408889634) in (np.float32(1), np.nextafter(np.float32(1), np.float32(0)))
    values = s.cache[(*at, slice(0, s.latent))].double().cpu().numpy()
    if form == "chunks":
        values = np.einsum("tc,hvc->htv", values, s.weights.values.double().cpu().numpy())
    else:
        values = np.broadcast_to(values, (2, 98, s.latent))
    got, want = s.run().double().cpu().numpy()[0], values[:, 97]
    assert np.abs(values).max() <= 8
    # the other weights, and half steps: of the output, the value, the weight and its sum
    bound = 97 * 2.0 ** -16 * 16 * (step == 16) + (torch.finfo(s.dtype).eps / 2 + 3 * 2.0 ** -11) * (np.abs(want) + 2.0 ** -14)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("at", [17, 300, 391])
def test_values_past_the_range_of_fp32_stay_with_the_rows_that_see_them(ops, parts, at) -> None:
    """Latents that the keys' matrix passes over and the values' takes past the largest fp32."""
    steps = [(400, 400), (1, 64)]
    s, clean = (Scene(ops, steps, form="chunks", heads=3, seed=57) for _ in range(2))
    for x in (s, clean):
        x.cache[..., 3] = 0
        x.weights.keys[..., 3] = 0
        x.weights.values[..., 3] = 0
        x.weights.values[:, ::5, 3] = 1e30
    s.cache[int(s.table[0, at // 16]), at % 16, 3] = 1e20
    got, ref = s.run(), clean.run()
    assert bool(ref.isfinite().all())
    blind = [*range(at), 400]
    assert torch.equal(got[blind], ref[blind])
    assert not bool(got[at:400, :, ::5].isfinite().any())
    assert torch.equal(got[at:400, :, 1::5], got[at:400, :, 1::5].nan_to_num(7.0, 7.0, 7.0))


def test_loud_queries_across_loud_keys(ops, parts) -> None:
    """Queries and keys of 2^80 whose products are zeros: every position weighs the same."""
    s = Scene(ops, [(3, 300), (130, 200)], form="chunks", heads=2, seed=58)
    s.weights.keys.zero_()
    s.weights.keys[:, 1, 1] = 1
    s.weights.values[..., 1] = 0
    s.cache[..., 1] = 2.0 ** 80
    s.cache[..., s.latent:] = 0
    s.q.zero_()
    s.q[..., 0] = 2.0 ** 80
    s.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("louder", [2.0 ** -6, 2.0, 64.0])
def test_scales_of_positions_not_seen_change_no_bits(ops, parts, dtype, louder) -> None:
    """A position that sets its tile's scales, seen by some rows: the others' outputs keep every bit. (Elements from 2^-27
    of a tile's largest on are not rounded otherwise under another power of two.)"""
    steps = [(150, 400), (1, 64)]
    s, clean = (Scene(ops, steps, form="chunks", dtype=dtype, heads=3, seed=48) for _ in range(2))
    at = (int(s.table[0, 330 // 16]), 330 % 16, slice(0, s.latent))
    s.cache[at] *= louder
    for x in (s, clean):
        if louder < 1:  # there it is the clean one that is louder
            x.cache[at] *= 8
    got, ref = s.run(), clean.run()
    assert torch.equal(got[:80], ref[:80]) and torch.equal(got[150], ref[150])
    assert not torch.equal(got[80:150], ref[80:150])
    s.check(got)
