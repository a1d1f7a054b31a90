"""The block-scaled KV write on steps large enough for each of its launch shapes, bit for bit.

The launch deals rows to waves by the step's size (rows x heads x 2) and its blocks' size: these
steps reach every one, with runs of every length side by side, begun blocks whose scales grow,
padding between the runs and values that are not finite in runs that several waves share.
"""

from __future__ import annotations

import numpy as np
import pytest

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType
from tests.test_gpu_block_scaled import Cache, device_rows, values, with_slots

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


def runs(rng: np.random.Generator, total: int, block: int) -> tuple[np.ndarray, np.ndarray, int]:
    """Slots of at least ``total`` rows, run by run, the slots of what the begun blocks hold before, and
    the blocks in the pool. A run is of one block: a third of them a single row, a third up to 16, the
    others as much as the block holds, half of all from an offset inside it; rows of the padding block
    and of slots outside the pool lie between some, and some runs' rows are not in order."""
    spans = []
    while sum(count for _, count in spans) < total:
        kind = int(rng.integers(3))
        count = 1 if kind == 0 else int(rng.integers(1, min(16, block) + 1)) if kind == 1 else block
        first = int(rng.integers(0, block)) if rng.integers(2) else 0
        spans.append((first, min(count, block - first)))
    blocks = 1 + len(spans)
    new: list[int] = []
    held: list[int] = []
    for block_id, (first, count) in zip((1 + rng.permutation(len(spans))).tolist(), spans):
        offsets = first + np.arange(count)
        if rng.integers(8) == 0:
            rng.shuffle(offsets)
        new += (block_id * block + offsets).tolist()
        held += (block_id * block + np.arange(first)).tolist()
        if rng.integers(16) == 0:
            new += [0, -1, blocks * block + 3][: int(rng.integers(1, 4))]
    return np.array(new, np.int64), np.array(held, np.int64), blocks


# (rows, block size, key/value heads, head width): the waves one row each would take are rows x heads x 2,
# and the launch changes at 8192 and 32768 of them, at blocks of 16 and (above 32768) of 32
LAUNCHES = [(5000, 16, 1, 64), (17500, 16, 1, 64), (9000, 5, 2, 64), (3000, 24, 1, 64), (6000, 24, 1, 64),
            (17500, 24, 1, 64), (9000, 32, 2, 64), (6000, 64, 1, 64), (17500, 64, 1, 64), (6000, 100, 3, 64),
            (17500, 1000, 1, 64), (8700, 64, 2, 128), (8700, 48, 2, 256), (8700, 16, 2, 256)]


@pytest.mark.parametrize("layout,dtype", [("nhd", "bf16"), ("hnd", "fp16")])
@pytest.mark.parametrize("rows,block,kv_heads,head_dim", LAUNCHES)
def test_every_launch_is_the_oracles_bit_for_bit(ops, rows, block, kv_heads, head_dim, layout, dtype) -> None:
    rng = np.random.default_rng(rows + block)
    new, held, blocks = runs(rng, rows, block)
    cache = Cache(blocks, block, kv_heads, head_dim, layout)
    for at, slots in enumerate((held, new)):
        # what the blocks hold first is small, so that most scales grow in the step that follows
        x = [values(rng, len(slots), kv_heads, head_dim) * (0.02 if at == 0 else 1.0) for _ in range(2)]
        if at == 1:
            for which in range(2):
                for value in (np.nan, np.inf, -np.inf):
                    bad = rng.integers(0, len(slots), len(slots) // 200)
                    x[which][bad, rng.integers(0, kv_heads, len(bad)), rng.integers(0, head_dim, len(bad))] = value
        ops.kvcache.store(*(device_rows(t, dtype) for t in x), cache.buffers, with_slots(slots, block))
        cache.store_host(*x, slots, dtype)
        cache.check(f"step {at}, {len(slots)} rows")


def test_runs_of_nothing_finite_and_of_zeros_shared_by_waves(ops) -> None:
    # whole runs of 33 to 64 rows: no finite value, zeros alone, one finite value beside NaN, over old scales
    # that are zero, smaller and larger
    rng = np.random.default_rng(3)
    block, runs_of = 64, 280
    cache = Cache(1 + runs_of, block, 1, 64, "nhd")
    ids = 1 + rng.permutation(runs_of)
    first = rng.choice([0, 20], runs_of)
    held = np.concatenate([i * block + np.arange(f) for i, f in zip(ids, first)])
    new = np.concatenate([i * block + np.arange(f, block) for i, f in zip(ids, first)])
    owner = np.repeat(np.arange(runs_of), block - first)
    before = np.repeat(rng.choice([0.0, 1e-3, 1e3], runs_of), first)
    x = [rng.standard_normal((len(held), 1, 64)).astype(np.float32) * before[:, None, None].astype(np.float32)
         for _ in range(2)]
    ops.kvcache.store(*(device_rows(t, "bf16") for t in x), cache.buffers, with_slots(held, block))
    cache.store_host(*x, held, "bf16")
    cache.check("held")
    kind = rng.integers(0, 4, runs_of)[owner]
    y = []
    for _ in range(2):
        t = rng.standard_normal((len(new), 1, 64)).astype(np.float32)
        t[kind == 0] = np.nan
        t[kind == 1] = 0.0
        t[kind == 2] = np.inf
        last = np.flatnonzero(np.diff(owner, append=-1))
        t[last[kind[last] == 2], 0, 7] = -3.25
        y.append(t)
    ops.kvcache.store(*(device_rows(t, "bf16") for t in y), cache.buffers, with_slots(new, block))
    cache.store_host(*y, new, "bf16")
    cache.check("new")
