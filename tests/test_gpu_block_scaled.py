"""The block-scaled 8-bit cache on the GPU: its write and block moves bit for bit against the oracle."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ayaka_amd.attention import AttentionMetadata
from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, ForwardMode, KVLayoutKind
from ayaka_amd.errors import BackendError
from ayaka_amd.kvcache import FP8_E4M3_CODEC, KVBuffers, fp8_e4m3_block_codec
from oracle import block_scaled
from oracle.numerics import bits_to_f32, f32_to_bits

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}
LAYOUTS = {"nhd": KVLayoutKind.NHD, "hnd": KVLayoutKind.HND}


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


def device_rows(x: np.ndarray, dtype: str) -> torch.Tensor:
    return torch.from_numpy(f32_to_bits(x, dtype).view(np.int16)).view(TORCH[dtype]).to(DEV)


class Cache:
    """A block-scaled cache on the device and its oracle on the host, fresh: NaN codes, scales of 0."""

    def __init__(self, blocks: int, block: int, kv_heads: int, head_dim: int, layout: str) -> None:
        self.layout = layout
        self.host = [block_scaled.empty(blocks, block, kv_heads, head_dim) for _ in range(2)]
        shape = (blocks, block, kv_heads, head_dim) if layout == "nhd" else (blocks, kv_heads, block, head_dim)
        k, v = (torch.full(shape, 0x7F, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
        self.scales = torch.zeros(blocks, kv_heads, 2, device=DEV)
        self.buffers = KVBuffers(k, v, LAYOUTS[layout], fp8_e4m3_block_codec(self.scales))

    def store_host(self, k: np.ndarray, v: np.ndarray, slots: np.ndarray, dtype: str) -> None:
        for x, (codes, scales) in zip((k, v), self.host):
            block_scaled.store(bits_to_f32(f32_to_bits(x, dtype), dtype), slots, codes, scales)

    def check(self, label: str) -> None:
        for which, tensor in enumerate((self.buffers.k, self.buffers.v)):
            got = tensor.view(torch.uint8).cpu().numpy()
            if self.layout == "hnd":
                got = got.transpose(0, 2, 1, 3)
            codes, scales = self.host[which]
            nan = (codes & 0x7F) == 0x7F
            assert np.array_equal((got & 0x7F) == 0x7F, nan), f"{label}: NaN codes of tensor {which}"
            assert np.array_equal(got[~nan], codes[~nan]), f"{label}: codes of tensor {which}"
            assert np.array_equal(self.scales[:, :, which].cpu().numpy().astype(np.float64), scales), (
                f"{label}: scales of tensor {which}")


def with_slots(slots: np.ndarray, block: int) -> AttentionMetadata:
    """A step's record with these slots, as far as the KV write reads it."""
    n = len(slots)
    row = torch.arange(n, dtype=torch.int32, device=DEV)
    return AttentionMetadata(mode=ForwardMode.MIXED, block_size=block, rows_per_request=torch.ones_like(row),
                             request_of_row=row, positions=row, slot_mapping=torch.from_numpy(slots).to(DEV),
                             kv_lengths=torch.ones_like(row), block_table=None, plan=None)


def values(rng: np.random.Generator, *shape: int) -> np.ndarray:
    """Rows whose sizes differ from row to row by up to 2^12, so that scales grow."""
    size = np.exp2(rng.integers(-6, 7, size=(*shape[:-1], 1)))
    return (rng.standard_normal(shape) * size).astype(np.float32)


STEPS = [  # (new rows, length before) per request and call
    [(5, 0), (1, 0), (17, 0)],
    [(1, 5), (1, 1), (1, 17)],
    [(1, 6), (30, 2), (1, 18)],
    [(9, 7), (1, 32), (2, 19)],
]


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("block", [1, 5, 16, 24, 100])
@pytest.mark.parametrize("dtype,kv_heads,head_dim", [("bf16", 2, 64), ("fp16", 3, 128), ("bf16", 1, 256)])
def test_a_sequence_of_writes_is_the_oracles_bit_for_bit(ops, layout, block, dtype, kv_heads, head_dim) -> None:
    rng = np.random.default_rng(block * 1000 + head_dim)
    width = -(-64 // block)
    blocks = 1 + 3 * width + 1
    cache = Cache(blocks, block, kv_heads, head_dim, layout)
    table = (1 + rng.permutation(blocks - 2)).reshape(3, width)
    for at, step in enumerate(STEPS):
        rows = [r for r, _ in step]
        lengths = [r + before for r, before in step]
        meta = ops.attention.plan(ForwardMode.MIXED, torch.tensor(rows, device=DEV), torch.tensor(lengths, device=DEV),
                                  torch.from_numpy(table).to(DEV), block)
        k, v = values(rng, sum(rows), kv_heads, head_dim), values(rng, sum(rows), kv_heads, head_dim)
        ops.kvcache.store(device_rows(k, dtype), device_rows(v, dtype), cache.buffers, meta)
        cache.store_host(k, v, meta.slot_mapping.cpu().numpy(), dtype)
        cache.check(f"step {at}")


def test_special_values(ops) -> None:
    # zeros, negative zeros, NaN, infinities, subnormals of every type, the largest finite values,
    # exact ties and the edges of a scale, as prompts and as later tokens
    special = [0.0, -0.0, np.nan, np.inf, -np.inf, 448.0, 449.0, -464.0, 2.0 ** -24, 2.0 ** -126, 2.0 ** -133, 1e-12,
               3e38, -2.5e30, 1e27, 65504.0, 17.0, 19.0, -1.0625, 1.1875]
    rng = np.random.default_rng(5)
    for dtype in ("bf16", "fp16"):
        cache = Cache(8, 4, 2, 64, "nhd")
        rows = np.zeros((12, 2, 64), np.float32)
        rows[1, :, :len(special)] = special
        rows[2, 0] = rng.standard_normal(64) * 1e-6
        rows[5:9, :, ::7] = np.nan
        rows[6, 1] = 1e30
        rows[9] = rng.standard_normal((2, 64)) * 300
        rows[10, 0, :5] = 3.3e38
        rows[11, 1] = np.inf
        with np.errstate(over="ignore"):
            slots = np.array([4, 5, 6, 7, 8, 9, 10, 11, 12, 16, 17, 20], dtype=np.int64)
            for lo, hi in ((0, 1), (1, 4), (4, 5), (5, 8), (8, 12)):
                part = rows[lo:hi]
                ops.kvcache.store(device_rows(part, dtype), device_rows(-part, dtype), cache.buffers,
                                  with_slots(slots[lo:hi], 4))
                cache.store_host(part, -part, slots[lo:hi], dtype)
                cache.check(f"{dtype} rows {lo}..{hi}")


def test_padding_rows_and_rows_outside_the_pool_are_dropped(ops) -> None:
    cache = Cache(6, 4, 2, 64, "nhd")
    cache.scales[0] = 3.0  # whatever block 0 holds stays
    for _, scales in cache.host:
        scales[0] = 3.0
    rng = np.random.default_rng(1)
    slots = np.array([0, 0, 3, -1, 6 * 4, 1 << 40, 9, 10, 0, 8, 2], dtype=np.int64)
    k, v = values(rng, len(slots), 2, 64), values(rng, len(slots), 2, 64)
    meta = with_slots(slots[:9], 4)
    ops.kvcache.store(device_rows(k[:9], "bf16"), device_rows(v[:9], "bf16"), cache.buffers, meta)
    cache.store_host(k[:9], v[:9], slots[:9], "bf16")
    cache.check("dropped rows")


def test_a_long_run_of_rows_in_one_block(ops) -> None:
    # more rows than a wave has lanes, from an offset inside the block
    cache = Cache(3, 400, 1, 128, "hnd")
    rng = np.random.default_rng(2)
    for slots in (np.arange(400, 470), np.arange(470, 800)):
        k, v = values(rng, len(slots), 1, 128), values(rng, len(slots), 1, 128)
        ops.kvcache.store(device_rows(k, "bf16"), device_rows(v, "bf16"), cache.buffers, with_slots(slots, 400))
        cache.store_host(k, v, slots, "bf16")
        cache.check(f"{len(slots)} rows")


def test_scales_a_caller_left_in_another_form_count_as_the_power_of_two_below(ops) -> None:
    cache = Cache(3, 4, 1, 64, "nhd")
    rng = np.random.default_rng(3)
    one = rng.standard_normal((1, 1, 64)).astype(np.float32)
    for stored, meant in ((1.5, 1.0), (float("inf"), 2.0 ** 80), (float("nan"), 2.0 ** 80), (-4.0, 0.0),
                          (1e-30, 2.0 ** -40)):
        codes, scales = cache.host[0]
        codes[1], cache.host[1][0][1] = 0x38, 0x38  # ones
        cache.buffers.k.view(torch.uint8)[1] = 0x38
        cache.buffers.v.view(torch.uint8)[1] = 0x38
        cache.scales[1] = stored
        scales[1] = cache.host[1][1][1] = meant
        ops.kvcache.store(device_rows(one, "bf16"), device_rows(one, "bf16"), cache.buffers,
                          with_slots(np.array([6]), 4))
        cache.store_host(one, one, np.array([6]), "bf16")
        cache.check(f"scale {stored}")


def test_large_steps(ops) -> None:
    rng = np.random.default_rng(4)
    rows, before = [700, 1, 333, 1, 1], [9, 70, 0, 15, 16]
    block, kv_heads, head_dim = 16, 8, 64
    lengths = [r + b for r, b in zip(rows, before)]
    need = [-(-n // block) for n in lengths]
    table = np.zeros((5, max(need)), np.int64)
    free = list(1 + rng.permutation(sum(need)))
    for b, n in enumerate(need):
        table[b, :n] = [free.pop() for _ in range(n)]
    cache = Cache(1 + sum(need), block, kv_heads, head_dim, "nhd")
    for counts, ends in ((before, before), (rows, lengths)):
        live = [i for i, c in enumerate(counts) if c]
        meta = ops.attention.plan(ForwardMode.MIXED, torch.tensor([counts[i] for i in live], device=DEV),
                                  torch.tensor([ends[i] for i in live], device=DEV),
                                  torch.from_numpy(table[live]).to(DEV), block)
        n = sum(counts)
        k, v = values(rng, n, kv_heads, head_dim), values(rng, n, kv_heads, head_dim)
        ops.kvcache.store(device_rows(k, "fp16"), device_rows(v, "fp16"), cache.buffers, meta)
        cache.store_host(k, v, meta.slot_mapping.cpu().numpy(), "fp16")
        cache.check(f"{n} rows")


def test_block_moves_take_the_scales_along(ops) -> None:
    rng = np.random.default_rng(6)
    cache = Cache(9, 4, 3, 64, "nhd")
    slots = np.arange(4, 36)
    k, v = values(rng, 32, 3, 64), values(rng, 32, 3, 64)
    ops.kvcache.store(device_rows(k, "bf16"), device_rows(v, "bf16"), cache.buffers, with_slots(slots, 4))
    cache.store_host(k, v, slots, "bf16")
    before = cache.scales.clone()
    src, dst = torch.tensor([2, 5], device=DEV), torch.tensor([7, 1], device=DEV)
    ops.kvcache.copy_blocks(cache.buffers, src, dst)
    for codes, scales in cache.host:
        codes[[7, 1]], scales[[7, 1]] = codes[[2, 5]], scales[[2, 5]]
    cache.check("copy")
    ids = torch.tensor([7, 3], dtype=torch.int32, device=DEV)
    out_k, out_v = (torch.empty(2, 4, 3, 64, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2))
    out_scales = torch.full((2, 3, 2), -1.0, device=DEV)
    ops.kvcache.gather(cache.buffers, ids, out_k, out_v, out_scales)
    assert torch.equal(out_scales, before[[2, 3]])
    assert torch.equal(out_k.view(torch.uint8), cache.buffers.k.view(torch.uint8)[[7, 3]])
    ops.kvcache.zero_blocks(cache.buffers, ids)
    for codes, scales in cache.host:
        codes[[7, 3]], scales[[7, 3]] = 0, 0.0
    cache.check("zero")
    with pytest.raises(BackendError, match="out_scales goes with a block-scaled cache"):
        ops.kvcache.gather(cache.buffers, ids, out_k, out_v)
    plain = KVBuffers(cache.buffers.k, cache.buffers.v, KVLayoutKind.NHD, FP8_E4M3_CODEC)
    with pytest.raises(BackendError, match="out_scales goes with a block-scaled cache"):
        ops.kvcache.gather(plain, ids, out_k, out_v, out_scales)


def test_refusals_on_the_device(ops) -> None:
    cache = Cache(4, 4, 2, 64, "nhd")
    meta = with_slots(np.array([4, 5]), 4)
    rows = torch.zeros(2, 2, 64, device=DEV)
    with pytest.raises(BackendError, match="computes in float16, bfloat16"):
        ops.kvcache.store(rows, rows, cache.buffers, meta)
    other = cache.buffers._replace(codec=fp8_e4m3_block_codec(torch.zeros(4, 2, 2)))
    half = rows.to(torch.bfloat16)
    with pytest.raises(BackendError, match="scales is on cpu"):
        ops.kvcache.store(half, half, other, meta)
    with pytest.raises(BackendError, match="make the codec with fp8_e4m3_block_codec"):
        ops.kvcache.store(half, half, cache.buffers._replace(codec="fp8_e4m3_block"), meta)
