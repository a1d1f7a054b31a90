"""Attention whose every score is far from zero: still a mean of the values.

All keys of a context are alike, so its weights are equal whatever the score: the output is bit for
bit the one of a softmax scale of 0.
"""

from __future__ import annotations

import math

import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, ForwardMode, KVLayoutKind
from ayaka_amd.hip import attention as hip_attention
from ayaka_amd.kvcache import FP8_E4M3_CODEC, RAW_CODEC, KVBuffers, fp8_e4m3_block_codec, fp8_e4m3_codec

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _step(codec: str, dtype: torch.dtype, rows: list[int], lengths: list[int], heads: int, kv_heads: int, dim: int,
          score: float):
    """(q, buffers, metadata, out): every key is ``score`` along the queries' only element."""
    block, width = 16, 64
    g = torch.Generator(device=DEV).manual_seed(dim)
    blocks = 1 + len(rows) * width
    shape = (blocks, block, kv_heads, dim)
    q = torch.zeros(sum(rows), heads, dim, dtype=dtype, device=DEV)
    k = torch.zeros(shape, device=DEV)
    v = torch.randn(shape, generator=g, device=DEV)
    if codec == RAW_CODEC:
        q[..., 0], k[..., 0] = 16.0, score / 16.0
        buffers = KVBuffers(k.to(dtype), v.to(dtype), KVLayoutKind.NHD, RAW_CODEC)
    else:
        q[..., 0], k[..., 0] = 16384.0, -448.0 if score < 0 else 448.0
        by = abs(score) / 16384.0 / 448.0
        if codec == FP8_E4M3_CODEC:
            name = fp8_e4m3_codec(by, 1.0)
        else:
            scales = torch.ones(blocks, kv_heads, 2, device=DEV)
            scales[..., 0] = 2.0 ** math.floor(math.log2(by))
            name = fp8_e4m3_block_codec(scales)
        buffers = KVBuffers(k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn), KVLayoutKind.NHD, name)
    table = torch.arange(1, blocks, device=DEV).view(len(rows), width)
    mode = ForwardMode.DECODE if max(rows) == 1 else ForwardMode.MIXED
    ops = load_backend(["hip"], device="cuda", dtype=DType.FP32 if dtype == torch.float32 else DType.BF16)
    meta = ops.attention.plan(mode, torch.tensor(rows, device=DEV), torch.tensor(lengths, device=DEV), table, block)
    return ops, q, buffers, meta, torch.full_like(q, float("nan"))


@pytest.mark.parametrize("score", [-9e30, -3e10, 1e8, 3e10, 9e30])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("codec,dtype", [(RAW_CODEC, torch.bfloat16), (RAW_CODEC, torch.float32),
                                         (FP8_E4M3_CODEC, torch.bfloat16), ("fp8_e4m3_block", torch.bfloat16)])
def test_equal_scores_weigh_equally_however_far(codec, dtype, head_dim, score) -> None:
    pairs = hip_attention.PREFILL_PAIRS[head_dim]
    half = dtype != torch.float32
    for rows, lengths, heads in (([1, 1, 1], [700, 1, 17], 8), ([1, 1], [300, 33], 2), ([4, 2], [300, 2], 8),
                                 ([40, 3], [300, 90], 8)):
        ops, q, buffers, meta, out = _step(codec, dtype, rows, lengths, heads, 2, head_dim, score)
        if max(rows) == 1:
            forced = [dict(partitions=0), dict(partitions=11, partition_size=64),
                      dict(partitions=11, partition_size=64, merge="reduce-kernel")]
            if half:
                forced += [dict(partitions=0, waves=4)]
            if half and codec == RAW_CODEC:
                forced += [dict(partitions=0, qk="dpp"), dict(partitions=0, qk="mfma")]
            if not half:
                forced[1:2] = []
        elif not half:
            forced = []
        elif max(rows) <= 4:
            forced = [dict(partitions=0, prefill=True, window=True),
                      dict(partitions=None, partition_size=64, prefill=True, window=True)]
        else:
            forced = [dict(partitions=None, partition_size=64, prefill=True, window=False, tile_pairs=pairs)] + [
                dict(partitions=0, prefill=True, window=False, tile_pairs=n) for n in (pairs, pairs // 2, pairs // 4)]
        for launch in [None, *forced]:
            want = torch.full_like(out, float("nan"))
            for scale, to in ((0.0, want), (1.0, out)):
                if launch is None:
                    ops.attention.attend(q, buffers, meta, to, scale=scale)
                else:
                    hip_attention.attend_with(q, buffers, meta, to, scale=scale, **launch)
            torch.cuda.synchronize()
            assert want.float().abs().max() > 0.01
            assert torch.equal(out, want), (rows, launch)
