"""The block-scaled codec on the CPU: its oracle against torch, the codec object, every refusal."""

from __future__ import annotations

import copy
import pickle
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from ayaka_amd.enums import ForwardMode, KVLayoutKind
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import _checks, _lib
from ayaka_amd.hip import attention as hip_attention
from ayaka_amd.hip import kvcache as hip_kvcache
from ayaka_amd.kvcache import (
    FP8_E4M3_BLOCK_CODEC,
    FP8_E4M3_CODEC,
    KVBuffers,
    codec_scales,
    fp8_e4m3_block_codec,
)
from oracle import block_scaled
from oracle.numerics import e4m3_to_f32
from tests import test_kv_reach as kv_reach

HEADER = Path(__file__).resolve().parent.parent / "include" / "ayaka_hip_block_scaled.h"


def test_every_declared_function_is_exported_and_bound() -> None:
    names = re.findall(r"\b(ayk_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S))
    assert sorted(names) == sorted(_lib.BLOCK_SCALED_EXPORTS)
    lib = _lib.lib()
    for name in names:
        assert hasattr(lib, name), name


# --- the oracle -----------------------------------------------------------------------------------


def test_least_scale() -> None:
    # 448 * 2^e is still covered by 2^e; the next value above needs twice as much
    for e in (-40, -7, 0, 3, 79):
        assert block_scaled.least_scale(448.0 * 2.0 ** e) == 2.0 ** e
        assert block_scaled.least_scale(np.nextafter(448.0 * 2.0 ** e, np.inf)) == 2.0 ** (e + 1)
    assert block_scaled.least_scale(0.0) == 0.0
    assert block_scaled.least_scale(1e-38) == 2.0 ** -40
    assert block_scaled.least_scale(3e38) == 2.0 ** 80


def test_the_oracle_encodes_as_torch_casts() -> None:
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((8, 2, 64)) * 30.0).astype(np.float32)
    codes, scales = block_scaled.empty(3, 8, 2, 64)
    block_scaled.store(x, np.arange(8) + 8, codes, scales)
    for h in range(2):
        s = float(scales[1, h])
        assert 224.0 * s < np.abs(x[:, h]).max() <= 448.0 * s
        cast = torch.from_numpy(x[:, h] / np.float32(s)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        assert np.array_equal(codes[1, :, h], cast)
    assert (codes[0] == 0x7F).all() and (codes[2] == 0x7F).all() and not scales[[0, 2]].any()
    error = np.abs(block_scaled.decode(codes, scales)[1] - x)
    # half a step: 2^-4 of the value, or half the subnormals' step of 2^-9 * scale
    assert (error <= np.maximum(np.abs(x) * 2.0 ** -4, scales[1][None, :, None] * 2.0 ** -10)).all()


def test_growth_lowers_exponents_and_a_first_token_starts_afresh() -> None:
    codes, scales = block_scaled.empty(2, 4, 1, 64)
    one = np.full((1, 1, 64), 1.0, np.float32)
    block_scaled.store(one, np.array([4]), codes, scales)  # 1 <= 448 * 2^-8, and not 448 * 2^-9
    assert scales[1, 0] == 2.0 ** -8 and e4m3_to_f32(codes[1, 0]).max() == 256.0
    block_scaled.store(one * 1000.0, np.array([5]), codes, scales)
    assert scales[1, 0] == 4.0
    assert (block_scaled.decode(codes, scales)[1, 0] == 1.0).all()  # exactly as it was
    block_scaled.store(one, np.array([6]), codes, scales)  # a smaller token leaves the scale
    assert scales[1, 0] == 4.0 and (block_scaled.decode(codes, scales)[1, 2] == 1.0).all()
    block_scaled.store(one * 0.5, np.array([4]), codes, scales)  # the block's first token: a new block
    assert scales[1, 0] == 2.0 ** -9


def test_values_that_are_not_finite_leave_the_scale_alone() -> None:
    codes, scales = block_scaled.empty(2, 2, 1, 64)
    x = np.ones((2, 1, 64), np.float32)
    x[0, 0, 3], x[1, 0, 5] = np.inf, np.nan
    block_scaled.store(x, np.array([2, 3]), codes, scales)
    got = block_scaled.decode(codes, scales)[1, :, 0]
    assert scales[1, 0] == 2.0 ** -8
    assert np.isnan(got[0, 3]) and np.isnan(got[1, 5]) and np.isfinite(got).sum() == 2 * 64 - 2


# --- the codec object -------------------------------------------------------------------------------


def test_the_codec_is_its_name_and_carries_its_scales() -> None:
    scales = torch.zeros(5, 2, 2)
    codec = fp8_e4m3_block_codec(scales)
    assert codec == FP8_E4M3_BLOCK_CODEC and codec != FP8_E4M3_CODEC and hash(codec) == hash(FP8_E4M3_BLOCK_CODEC)
    assert codec.scales is scales and codec_scales(codec) == (1.0, 1.0) and "5, 2, 2" in repr(codec)
    with pytest.raises(AttributeError):
        codec.scales = torch.zeros(5, 2, 2)
    for other in (copy.deepcopy(codec), pickle.loads(pickle.dumps(codec))):
        assert other == codec and torch.equal(other.scales, scales)
    assert copy.copy(codec).scales is scales


@pytest.mark.parametrize("scales", [torch.zeros(5, 2), torch.zeros(5, 2, 3), torch.zeros(5, 2, 2, dtype=torch.float16),
                                    torch.zeros(5, 2, 4)[:, :, ::2]])
def test_the_codec_refuses_other_scales(scales: torch.Tensor) -> None:
    with pytest.raises(ValueError, match="float32 \\[num_blocks, kv_heads, 2\\]"):
        fp8_e4m3_block_codec(scales)


# --- refusals of the ops ------------------------------------------------------------------------------


def _buffers(codec: str, head_dim: int = 64) -> KVBuffers:
    k = torch.zeros(5, 4, 2, head_dim, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return KVBuffers(k, k.clone(), KVLayoutKind.NHD, codec)


def _meta():
    return hip_attention.plan(ForwardMode.DECODE, torch.tensor([1, 1]), torch.tensor([3, 2]),
                              torch.tensor([[1], [2]]), 4)


def test_a_cache_without_its_scales_is_refused(monkeypatch: pytest.MonkeyPatch) -> None:
    # the device check comes first on the CPU, so the scales' own check is called as it calls it
    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(BackendError, match="runs on a HIP device"):
        hip_kvcache.store(q, q, _buffers(fp8_e4m3_block_codec(torch.zeros(5, 2, 2))), _meta())
    with pytest.raises(BackendError, match="make the codec with fp8_e4m3_block_codec"):
        _checks.require_block_scales("op", _buffers(FP8_E4M3_BLOCK_CODEC))
    for shape in ((4, 2, 2), (5, 1, 2)):
        with pytest.raises(BackendError, match=r"scales must be float32 \[5, 2, 2\]"):
            _checks.require_block_scales("op", _buffers(fp8_e4m3_block_codec(torch.zeros(*shape))))
    with pytest.raises(BackendError, match=r"head widths \[64, 128, 256\], not 32"):
        _checks.require_block_scales("op", _buffers(fp8_e4m3_block_codec(torch.zeros(5, 2, 2)), 32))
    with pytest.raises(BackendError, match="8-byte aligned"):
        _checks.require_block_scales("op", _buffers(fp8_e4m3_block_codec(torch.zeros(21)[1:].view(5, 2, 2))))
    _checks.require_block_scales("op", _buffers(fp8_e4m3_block_codec(torch.zeros(5, 2, 2))))


def test_block_scaled_caches_hold_fp8_codes() -> None:
    buffers = _buffers(fp8_e4m3_block_codec(torch.zeros(5, 2, 2)))
    raw = buffers._replace(k=torch.zeros(5, 4, 2, 64), v=torch.zeros(5, 4, 2, 64))
    with pytest.raises(BackendError, match="stores the 'fp8_e4m3_block' codec as float8_e4m3fn"):
        _checks.require_buffers("op", raw)


def _store(**kw: object) -> int:
    args = dict(k=16, v=16, k_cache=8, v_cache=8, scales=8, slots=8, n_rows=1, kv_heads=2, head_dim=64, num_blocks=4,
                block_size=16, layout=0, dtype=1, stream=None)
    args.update(kw)
    return _lib.lib().ayk_store_block_scaled(*args.values())


@pytest.mark.parametrize("changes,code,message", [
    ({"n_rows": -1}, 1, b"n_rows is negative"),
    ({"kv_heads": 0}, 1, b"num_kv_heads 0"),
    ({"head_dim": 96}, 2, b"head_dim 96"),
    ({"block_size": 0}, 2, b"block_size 0"),
    ({"block_size": 65537}, 2, b"block_size 65537"),
    ({"dtype": 3}, 2, b"src_dtype 3"),
    ({"layout": 2}, 2, b"layout 2"),
    ({"num_blocks": 1 << 21, "block_size": 16}, 2, b"32-bit element offsets"),
    ({"num_blocks": 1 << 30, "block_size": 1 << 16, "kv_heads": 1 << 12, "head_dim": 256}, 2, b"32-bit element offsets"),
    ({"n_rows": 1 << 32}, 2, b"exceed one launch"),
    ({"scales": None}, 1, b"null"),
    ({"k": 24}, 1, b"not 16-byte aligned"),
    ({"v": 18}, 1, b"not 16-byte aligned"),
    ({"v_cache": 12}, 1, b"not 16-byte aligned"),
])
def test_the_library_refuses_bad_stores(changes: dict, code: int, message: bytes) -> None:
    assert _store(**changes) == code
    assert message in _lib.lib().ayk_last_error()


def test_no_rows_is_no_launch() -> None:
    assert _store(n_rows=0, k=None, scales=None) == 0


# --- the library's attention entry points ---------------------------------------------------------------


def _v1(**kw: object) -> int:
    args = dict(out=16, q=16, k=8, v=8, scales=8, table=1, stride=4, lengths=1, ror=None, pos=None, n_rows=1, heads=8,
                kv_heads=2, head_dim=128, num_blocks=10, block_size=16, max_blocks=4, layout=0, dtype=1, scale=1.0,
                flags=0, stream=None)
    args.update(kw)
    return _lib.lib().ayk_paged_attention_v1_block_scaled(*args.values())


@pytest.mark.parametrize("changes,code,message", [
    ({"scales": None}, 1, b"block_scales"),
    ({"scales": 12}, 1, b"not 8-byte aligned"),
    ({"dtype": 3}, 2, b"under fp16/bf16"),
    ({"flags": 1}, 2, b"16-bit caches only"),
    ({"head_dim": 96}, 2, b"head_dim 96"),
    ({"num_blocks": 1 << 30, "block_size": 1 << 16, "heads": 1 << 12, "kv_heads": 1 << 12, "head_dim": 256}, 2,
     b"32-bit element offsets"),
    ({"heads": 7}, 1, b"not a positive multiple"),
    ({"q": None}, 1, b"null"),
    ({"q": 8}, 1, b"not 16-byte aligned"),
    ({"out": 24}, 1, b"not 16-byte aligned"),
    ({"k": 4}, 1, b"not 16-byte aligned"),
])
def test_the_library_refuses_bad_attention(changes: dict, code: int, message: bytes) -> None:
    assert _v1(**changes) == code
    assert message in _lib.lib().ayk_last_error()


def test_multi_row_and_split_refusals() -> None:
    lib = _lib.lib()
    base = (16, 16, 8, 8, 8, 1, 4, 1)
    shape = (1, 8, 2, 128, 10, 16, 4, 0, 1, 1.0)
    assert lib.ayk_paged_attention_v2_block_scaled(*base, None, None, *shape, 100, 4, None, 0, None, 1, 1 << 20, None,
                                                   0, None) == 1
    assert b"ayk_paged_attention_v2_block_scaled: partition_size 100" in lib.ayk_last_error()
    assert lib.ayk_paged_attention_v2_block_scaled(*base, None, None, *shape, 64, 4, None, 0, None, 16, 16, None, 0,
                                                   None) == 4
    assert lib.ayk_paged_prefill_block_scaled(*base, None, None, 1, 1, 128, *shape, 0, None, 0, None) == 1
    assert b"request_of_row and positions are required" in lib.ayk_last_error()
    assert lib.ayk_paged_prefill_block_scaled(*base, 1, 1, 1, 1, 100, *shape, 0, None, 0, None) == 1
    assert b"tile_pairs 100" in lib.ayk_last_error()
    wide = (1, 34, 2, 128, 10, 16, 4, 0, 1, 1.0)
    assert lib.ayk_paged_attention_windows_block_scaled(*base, 1, 1, 1, 1, *wide, 0, None, 0, None) == 2
    assert b"17 query heads" in lib.ayk_last_error()


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_loads_stay_in_the_cache(head_dim: int) -> None:
    # the block-scaled launches form the fp8 launches' addresses: the host walk of each entry point
    rng = np.random.default_rng(head_dim)
    for case in range(12):
        block = kv_reach.BLOCK_SIZES[case % len(kv_reach.BLOCK_SIZES)]
        kv_heads, group = [(2, 4), (3, 1), (1, 8), (4, 2)][case % 4]
        lengths = kv_reach._lengths(rng, block, int(rng.integers(1, 5)))
        step = kv_reach.Step(rng, lengths, block, kv_heads, head_dim, True, case % 2)
        heads = kv_heads * group

        def common(rows, req, pos):
            args = kv_reach._common(step, heads, rows, req, pos)
            return (*args[:4], 8, *args[4:-4], args[-3])  # scales in, kv_dtype and the layer's scales out

        def check(call, label):
            kv_reach._check(step, kv_reach._walk(step, call), f"case {case} block {block} {label}")

        rows = len(lengths)
        check(lambda lib: lib.ayk_paged_attention_v1_block_scaled(*common(rows, None, None), 0, None), "v1")
        parts = -(-step.width * block // 64)
        nbytes = _lib.lib().ayk_paged_attention_v2_workspace_bytes(rows, heads, head_dim, parts)
        check(lambda lib: lib.ayk_paged_attention_v2_block_scaled(
            *common(rows, None, None), 64, parts, None, 0, None, kv_reach.FAKE, nbytes, None, 0, None), "v2")
        counts = [min(n, 16 // group) or 1 for n in lengths]
        req, pos = kv_reach._rows(step, counts)
        tiles = kv_reach._tiles(counts, max(counts), 1)
        args = common(len(req), req, pos)
        check(lambda lib: lib.ayk_paged_attention_windows_block_scaled(
            *args[:10], kv_reach._ptr(tiles), tiles.size // 4, *args[10:], 0, None, 0, None), "windows")
        pairs = _lib.lib().ayk_paged_prefill_tile_pairs(head_dim)
        check(lambda lib: lib.ayk_paged_prefill_block_scaled(
            *args[:10], kv_reach._ptr(tiles), tiles.size // 4, pairs, *args[10:], 0, None, 0, None), "multi-row")


def test_a_default_stream_of_another_device_is_refused(monkeypatch: pytest.MonkeyPatch) -> None:
    # the raw handle 0 names the current device's default stream, whichever device the tensors are on
    monkeypatch.setattr(_checks, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(_checks, "_current_device", lambda: 0)
    assert _checks.stream_handle(torch.device("cuda", 0)) == 0
    with pytest.raises(BackendError, match="tensors are on device 1 .* under torch.cuda.device"):
        _checks.stream_handle(torch.device("cuda", 1))
    monkeypatch.setattr(_checks, "_raw_stream", lambda index: 77)  # a stream of its own names its device
    assert _checks.stream_handle(torch.device("cuda", 1)) == 77


def test_the_refusal_of_other_codecs_names_this_one() -> None:
    with pytest.raises(BackendError, match="not 'int8' .*'fp8_e4m3_block', made with fp8_e4m3_block_codec"):
        _checks.require_buffers("op", _buffers("int8"))
