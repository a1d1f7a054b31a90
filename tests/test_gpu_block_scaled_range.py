"""Attention over block-scaled caches whose value scales span the whole range, against float64.

The weights' sum is carried by the positions with the largest scores, whatever their blocks' value
scales: here one block lies at 2^80, the others at 2^-40, and most of the sum (or a share of it far
above a rounding) belongs to positions whose value-scaled weights are below the smallest normal
float32 next to the loud block's.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType
from ayaka_amd.hip import attention as hip_attention
from oracle.numerics import e4m3_to_f32, f32_to_bits, f32_to_e4m3
from tests.test_gpu_block_scaled_attention import Step, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


class Quiet(Step):
    """Contexts in which every block's values are worth 2^-40 of their codes but one's, worth 2^80.

    A position's score is its key's first element (queries are one there and zero elsewhere, key
    scales are 1): ``loud`` in the loud block, drawn from ``quiet`` in the others. ``at`` places the
    loud block: the first of every context, its middle one or its last.
    """

    def __init__(self, steps, quiet, *, loud=0.0, at="first", low=-40, high=80, **kw) -> None:
        super().__init__(steps, **kw)
        rng = np.random.default_rng(1)
        self.scale = 1.0
        q = np.zeros((sum(self.rows), kw.get("heads", 4), self.codes[0].shape[-1]), np.float32)
        q[..., 0] = 1.0
        self.q_bits = f32_to_bits(q, self.dtype)
        for b, length in enumerate(self.lengths):
            ids = self.table[b, : -(-length // self.block)]
            if not len(ids):
                continue
            place = {"first": 0, "middle": len(ids) // 2, "last": len(ids) - 1}[at]
            self.scales[ids, :, 0] = 1.0
            self.scales[ids, :, 1] = 2.0 ** low
            self.scales[ids[place], :, 1] = 2.0 ** high
            score = rng.choice(np.asarray(quiet, np.float32), (len(ids), self.block, self.kv_heads))
            score[place] = loud
            keys = np.zeros((*score.shape, self.codes[0].shape[-1]), np.float32)
            keys[..., 0] = score
            # (the slots behind the context stay NaN codes)
            held = (np.arange(len(ids) * self.block) < length).reshape(len(ids), self.block)
            codes = self.codes[0][ids]
            codes[held] = f32_to_e4m3(keys)[held]
            self.codes[0][ids] = codes
        self._known = None

    def reference(self):
        if self._known is None:
            self._known = super().reference()
        return self._known


def test_the_scores_are_the_keys_first_elements() -> None:
    # e4m3 holds these scores as they are, so the cases are what they say
    scores = np.array([0.0, -4.0, -4.5, -5.0, -6.0, -10.0, -12.0, 3.0], np.float32)
    assert np.array_equal(e4m3_to_f32(f32_to_e4m3(scores)), scores)


@pytest.mark.parametrize("block", [16, 12, 7])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_decode(ops, at, head_dim, block) -> None:
    step = Quiet([(1, 700), (1, 40), (1, 0)], [-4.5, -5.0, -6.0], at=at, heads=4, head_dim=head_dim, block=block,
                 mode="decode")
    run(ops, step)
    for waves in (1, 2, 4, 8):
        run(ops, step, label=at, partitions=0, waves=waves)
    for size, merge in ((64, "in-kernel"), (64, "reduce-kernel"), (320, None)):
        run(ops, step, label=at, partitions=-(-701 // size), partition_size=size, merge=merge)


@pytest.mark.parametrize("merge", ["in-kernel", "reduce-kernel"])
@pytest.mark.parametrize("length,quiet", [(2600, [-9.0, -10.0]), (9000, [-10.0, -12.0])])
def test_a_sum_of_many_far_smaller_weights(ops, length, quiet, merge) -> None:
    # up to 17 bits below the loud block's each, and together a share that no rounding hides; over 41
    # and 141 partitions, where the reduce kernel takes 8 at a time (above: 1 and 4)
    for at in ("first", "last"):
        step = Quiet([(1, length)], quiet, at=at, heads=4, head_dim=128, mode="decode")
        run(ops, step, label=at, partitions=-(-length // 64), partition_size=64, merge=merge)


@pytest.mark.parametrize("high,low", [(80, -40), (56, -40), (41, -40), (40, -40), (80, -17)])
def test_scores_above_the_loud_blocks(ops, high, low) -> None:
    # the quiet positions hold nearly all of the weight, and some of it lies 20 bits below their own most
    for mode, rows in (("decode", 1), ("mixed", 3), ("mixed", 40)):
        run(ops, Quiet([(rows, 300)], [14.0, 11.0, 0.0], at="middle", high=high, low=low, heads=8, head_dim=128,
                       mode=mode))


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_windows(ops, at, head_dim) -> None:
    step = Quiet([(4, 300), (2, 517), (1, 0)], [-4.5, -5.0, -6.0], at=at, heads=8, head_dim=head_dim)
    for size in (0, 64, 256):
        run(ops, step, label=at, prefill=True, window=True, partitions=0 if size == 0 else None,
            partition_size=size or None)


@pytest.mark.parametrize("block", [16, 12, 7])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_multi_row(ops, at, head_dim, block) -> None:
    step = Quiet([(37, 300), (3, 90), (2, 0)], [-4.5, -5.0, -6.0], at=at, heads=4, head_dim=head_dim, block=block)
    run(ops, step)
    full = hip_attention.PREFILL_PAIRS[head_dim]
    for pairs in ((2 * full,) if head_dim != 64 else ()) + (full, full // 2, full // 4):
        run(ops, step, label=at, prefill=True, window=False, tile_pairs=pairs, partitions=0)
        run(ops, step, label=at, prefill=True, window=False, tile_pairs=pairs, partition_size=64)


def test_many_table_segments(ops) -> None:
    # blocks of one position: the loud one is in a segment of its own, before or behind the others
    for at in ("first", "last"):
        for rows in (1, 3, 40):
            step = Quiet([(rows, 2100)], [-5.0, -6.0], at=at, heads=8, head_dim=128, block=1,
                         mode="decode" if rows == 1 else "mixed")
            run(ops, step, label=at)
            run(ops, step, label=at, **(dict(partitions=0) if rows == 1 else
                                        dict(prefill=True, window=rows == 3, partitions=0)))


# --- scales that the write does not make ----------------------------------------------------------------


@pytest.mark.parametrize("mode,rows", [("decode", 1), ("mixed", 3), ("mixed", 40)])
def test_a_scale_that_is_not_above_zero_counts_as_zero(ops, mode, rows) -> None:
    # as the write counts it: keys of such a block score 0 whatever their codes, values are codes of zero
    for block in (16, 12, 7):
        step = Step([(rows, 300)], heads=8, head_dim=128, block=block, mode=mode, seed=5)
        ids = step.table[0, 1:4]
        step.codes[1][ids] = 0
        step.scales[ids, :, 0] = 0.0
        # (a value scale of 0 is read as 2^-40: the oracle's tolerance divides by it)
        step.scales[ids, :, 1] = 2.0 ** -40
        q, buffers, meta, out = step.device(ops)
        outs = []
        for key, value in ((0.0, 2.0 ** -40), (0.0, 0.0), (-4.0, -2.0 ** 30), (-0.0, -0.0), (-np.inf, -np.nan)):
            buffers.codec.scales[torch.from_numpy(ids).to(buffers.k.device)] = torch.tensor(
                np.array([key, value], np.float32), device=buffers.k.device)
            out.fill_(float("nan"))
            ops.attention.attend(q, buffers, meta, out, scale=step.scale)
            step.check(out, f"scales {key} and {value}")
            outs.append(out.clone())
        assert all(torch.equal(o, outs[0]) for o in outs)


def test_scales_between_and_beyond_the_powers_count_as_the_one_below(ops) -> None:
    step = Step([(1, 100)], heads=4, head_dim=64, mode="decode", seed=6)
    q, buffers, meta, out = step.device(ops)
    ids = torch.from_numpy(step.table[0, :7]).to(buffers.k.device)
    outs = []
    for pair in ((0.25, 2.0 ** -40), (0.3, 2.0 ** -45), (0.49999, 1e-38)):
        buffers.codec.scales[ids] = torch.tensor(pair, device=buffers.k.device)
        ops.attention.attend(q, buffers, meta, out, scale=step.scale)
        outs.append(out.clone())
    for pair in ((0.25, 2.0 ** 80), (0.25, 2.0 ** 90), (0.25, float("inf")), (0.25, float("nan"))):
        buffers.codec.scales[ids] = torch.tensor(pair, device=buffers.k.device)
        ops.attention.attend(q, buffers, meta, out, scale=step.scale)
        outs.append(out.clone())
    assert all(torch.equal(o, outs[0]) for o in outs[1:3]) and all(torch.equal(o, outs[3]) for o in outs[4:])
