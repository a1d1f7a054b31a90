"""Rotary positions and latent caches on the CPU: the oracle, the frequencies, every refusal."""

from __future__ import annotations

import math
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from ayaka_amd.attention import AttentionMetadata
from ayaka_amd.enums import ForwardMode, KVLayoutKind
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import _lib
from ayaka_amd.hip import attention as hip_attention
from ayaka_amd.hip import kvcache as hip_kvcache
from ayaka_amd.hip._checks import require_rows
from ayaka_amd.kvcache import RAW_CODEC, KVBuffers, LatentBuffers, LatentWeights
from ayaka_amd.rotary import BandScaling, LinearScaling, Rotary, YarnScaling, rotary
from oracle import latent as oracle

HEADER = Path(__file__).resolve().parent.parent / "include" / "ayaka_hip_latent.h"


def test_every_declared_function_is_exported_and_bound() -> None:
    names = re.findall(r"\b(ayk_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S))
    assert sorted(set(names)) == sorted(_lib.LATENT_EXPORTS)
    lib = _lib.lib()
    for name in names:
        assert hasattr(lib, name), name


# --- the oracle -----------------------------------------------------------------------------------


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_the_cosine_sine_form(interleaved) -> None:
    rng = np.random.default_rng(0)
    x, positions, turns = rng.standard_normal((3, 2, 10)), np.array([0, 5, 70000]), np.array([0.1591, 0.01, 0.0003])
    got = oracle.rotate(x, positions, turns, interleaved, 1.5)
    for n, t in enumerate(positions):
        for i, turn in enumerate(turns):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 3)
            c, s = math.cos(2 * math.pi * t * turn), math.sin(2 * math.pi * t * turn)
            np.testing.assert_allclose(got[n, :, a], 1.5 * (x[n, :, a] * c - x[n, :, b] * s), atol=1e-9)
            np.testing.assert_allclose(got[n, :, b], 1.5 * (x[n, :, b] * c + x[n, :, a] * s), atol=1e-9)
    assert np.array_equal(got[..., 6:], x[..., 6:])


def test_scores_of_rotated_rows_depend_on_the_distance_alone() -> None:
    rng = np.random.default_rng(1)
    q, k, turns = rng.standard_normal((1, 1, 8)), rng.standard_normal((1, 1, 8)), np.array([0.159, 0.05, 0.01, 0.002])
    dot = [float((oracle.rotate(q, [a], turns, False, 1.0) * oracle.rotate(k, [b], turns, False, 1.0)).sum())
           for a, b in ((7, 3), (1004, 1000))]
    assert dot[0] == pytest.approx(dot[1], abs=1e-9)


def test_both_forms_of_latent_attention_are_one() -> None:
    rng = np.random.default_rng(2)
    cache, table = rng.standard_normal((6, 4, 16 + 8)), np.array([[3, 1, 5], [2, 4, 0]])
    rows, lengths = [3, 2], [11, 7]
    q = rng.standard_normal((5, 2, 6 + 8))
    keys, values = rng.standard_normal((2, 6, 16)), rng.standard_normal((2, 5, 16))
    want = oracle.chunk_attention(q, keys, values, cache, table, rows, lengths, 0.3)[0]
    absorbed = np.concatenate((np.einsum("nhi,hic->nhc", q[..., :6], keys), q[..., 6:]), axis=-1)
    out = oracle.attention(absorbed, cache, table, rows, lengths, 0.3, 16)[0]
    np.testing.assert_allclose(np.einsum("nhc,hvc->nhv", out, values), want, atol=1e-9)


# --- frequencies ----------------------------------------------------------------------------------


def _frequencies(**kw) -> list[float]:
    return (rotary(8, device="cpu", **kw).turns * 2 * math.pi).tolist()


def test_plain_and_linear_frequencies() -> None:
    assert _frequencies() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    assert _frequencies(scaling=LinearScaling(4.0)) == pytest.approx([0.25, 0.025, 0.0025, 0.00025], rel=1e-14)
    made = rotary(8, device="cpu", interleaved=True)
    assert made.turns.dtype == torch.float64 and made.interleaved is True and made.magnitude == 1.0


def test_band_frequencies() -> None:
    # within 2000 positions the pairs turn 318, 31.8, 3.18 and 0.318 times: two stay (over 4), the last is
    # divided (under 1), the third is blended by (3.18 - 1) / 3
    keep = (2000 * 0.01 / (2 * math.pi) - 1) / 3
    want = [1.0, 0.1, 0.01 * (keep + (1 - keep) / 8), 0.001 / 8]
    assert _frequencies(scaling=BandScaling(8.0, 2000)) == pytest.approx(want, rel=1e-14)


def test_yarn_frequencies_and_magnitude() -> None:
    # 8 ln(2000 / (2 pi r)) / (2 ln 10000): r 32 at 0.997, r 1 at 2.502 -> the ramp from pair 0 to pair 3
    want = [f * (1 - r + r / 16) for f, r in zip((1.0, 0.1, 0.01, 0.001), (0.0, 1 / 3, 2 / 3, 1.0))]
    made = rotary(8, device="cpu", scaling=YarnScaling(16.0, 2000))
    assert (made.turns * 2 * math.pi).tolist() == pytest.approx(want, rel=1e-14)
    assert made.magnitude == pytest.approx(0.1 * math.log(16.0) + 1.0)
    assert rotary(8, device="cpu", scaling=YarnScaling(16.0, 2000, magnitude=0.75)).magnitude == 0.75


@pytest.mark.parametrize("call", [
    lambda: rotary(7, device="cpu"), lambda: rotary(0, device="cpu"), lambda: rotary(8, base=1.0, device="cpu"),
    lambda: rotary(8, base=math.nan, device="cpu"), lambda: LinearScaling(0.0), lambda: LinearScaling(math.inf),
    lambda: BandScaling(2.0, 0), lambda: BandScaling(2.0, 100, low=4.0, high=4.0), lambda: YarnScaling(-1.0, 100),
    lambda: YarnScaling(2.0, 100, fast=1.0, slow=1.0),
])
def test_rotations_that_mean_nothing_are_refused(call) -> None:
    with pytest.raises(ValueError):
        call()


# --- buffers ----------------------------------------------------------------------------------------


def _latent(blocks=4, block=16, latent=512, rope=64, dtype=torch.bfloat16) -> LatentBuffers:
    return LatentBuffers(torch.zeros(blocks, block, latent + rope, dtype=dtype), latent)


def test_latent_buffers_say_what_they_are() -> None:
    b = _latent(5, 24, 256, 64)
    assert (b.num_blocks, b.block_size, b.latent_dim, b.rope_dim) == (5, 24, 256, 64)
    assert b.layout == KVLayoutKind.NLD and b.codec == RAW_CODEC
    assert b.k is b.cache and b.v.shape == (5, 24, 256) and b.v.data_ptr() == b.cache.data_ptr()


def _meta(n=2, block=16) -> AttentionMetadata:
    return hip_attention.plan(ForwardMode.DECODE, torch.ones(n, dtype=torch.int32), torch.full((n,), 3, dtype=torch.int32),
                              torch.arange(1, n + 1, dtype=torch.int32)[:, None], block)


def test_ops_for_caches_of_keys_and_values_refuse_latent_ones() -> None:
    meta, b = _meta(), _latent()
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(BackendError, match="NHD and HND layouts, not NLD"):
        hip_attention.attend(x, b, meta, x, scale=1.0)
    with pytest.raises(BackendError, match="NHD and HND layouts, not NLD"):
        hip_kvcache.store(x, x, b, meta)


def test_latent_ops_refuse_what_is_no_latent_cache() -> None:
    meta = _meta()
    kv = KVBuffers(torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64), KVLayoutKind.NHD, RAW_CODEC)
    q, out = torch.zeros(2, 8, 576, dtype=torch.bfloat16), torch.zeros(2, 8, 512, dtype=torch.bfloat16)
    with pytest.raises(BackendError, match="must be LatentBuffers"):
        hip_attention.attend_latent(q, kv, meta, out, scale=1.0)
    for b, message in (
        (_latent(dtype=torch.float64), "stores latents as float16"),
        (LatentBuffers(torch.zeros(4, 16, 576), 576), "rope_dim above 0"),
        (LatentBuffers(torch.zeros(4, 16, 2, 288), 512), "rope_dim above 0"),
        (LatentBuffers(torch.zeros(4, 576, 16).transpose(1, 2), 512), "contiguous"),
        (_latent(), "runs on a HIP device"),
    ):
        with pytest.raises(BackendError, match=message):
            hip_attention.attend_latent(q, b, meta, out, scale=1.0)
        with pytest.raises(BackendError, match=message):
            hip_kvcache.store_latent(q[:, 0, :512], q[:, 0, 512:], b, meta)
        with pytest.raises(BackendError, match=message):
            hip_kvcache.copy_blocks(b, torch.zeros(1, dtype=torch.int64), torch.ones(1, dtype=torch.int64))


def test_rows_to_write_into_may_not_share_memory() -> None:
    def check(t, written=True):
        require_rows("op", "x", t, tuple(t.shape), t.dtype, t.device, written=written)

    x = torch.zeros(6, 4, 8)
    for fine in (x, x.transpose(0, 1), x[:, :, :4], x[::2], torch.zeros(1, 1, 8).expand(1, 1, 8),
                 torch.zeros(6, 100)[:, :32].unflatten(1, (4, 8)), x[:0]):
        check(fine)
    shared = torch.zeros(1, 4, 8).expand(6, 4, 8)
    check(shared, written=False)
    for bad in (shared, torch.zeros(100).as_strided((6, 4, 8), (16, 4, 1)), torch.zeros(100).as_strided((6, 4, 8), (8, 8, 1))):
        with pytest.raises(BackendError, match="share memory"):
            check(bad)
    with pytest.raises(BackendError, match="next to each other"):
        check(x.transpose(1, 2))


def test_rotate_refusals() -> None:
    meta, turn = _meta(), rotary(64, device="cpu")
    with pytest.raises(BackendError, match="neither q nor k"):
        hip_kvcache.rotate(None, None, meta, turn)
    with pytest.raises(BackendError, match="on a HIP device"):
        hip_kvcache.rotate(torch.zeros(2, 4, 64), None, meta, turn)
    with pytest.raises(BackendError, match="float16, bfloat16 or float32"):
        hip_kvcache.rotate(torch.zeros(2, 4, 64, dtype=torch.float64), None, meta, turn)


# --- the C entries ----------------------------------------------------------------------------------


def _rotate_args(**kw) -> list:
    args = dict(q=16, q_row=64, q_head=64, q_out=16, q_out_row=64, q_out_head=64, k=16, k_row=64, k_head=64, k_out=16,
                k_out_row=64, k_out_head=64, v=None, v_row=0, v_head=0, k_cache=None, v_cache=None, positions=16, slots=None,
                turns=16, pairs=32, interleaved=0, magnitude=1.0, n_rows=2, heads=1, kv_heads=1, head_dim=64, num_blocks=0,
                block_size=0, layout=0, dtype=1, stream=None)
    args.update(kw)
    return list(args.values())


@pytest.mark.parametrize("changes,code,message", [
    ({"n_rows": -1}, 1, b"n_rows is negative"),
    ({"dtype": 2}, 2, b"dtype 2"),
    ({"heads": -1}, 1, b"num_heads is negative"),
    ({"kv_heads": -1}, 1, b"num_kv_heads is negative"),
    ({"head_dim": 63}, 2, b"not even"),
    ({"head_dim": 1026}, 2, b"in [2, 1024]"),
    ({"pairs": 33}, 1, b"33 pairs do not fit"),
    ({"pairs": -1}, 1, b"-1 pairs"),
    ({"magnitude": math.inf}, 1, b"magnitude must be finite"),
    ({"turns": None}, 1, b"turns is null"),
    ({"turns": 20}, 1, b"8-byte aligned"),
    ({"positions": None}, 1, b"positions or turns is null"),
    ({"q": None}, 1, b"null"),
    ({"k_out": None}, 1, b"null"),
    ({"q": 17}, 1, b"multiple of the element's size"),
    ({"k_cache": 16}, 1, b"given together"),
    ({"k_cache": 16, "v_cache": 16, "num_blocks": 4}, 2, b"block_size 0"),
    ({"k_cache": 16, "v_cache": 16, "num_blocks": 0, "block_size": 16}, 1, b"num_blocks 0"),
    ({"k_cache": 16, "v_cache": 16, "num_blocks": 1 << 28, "block_size": 16}, 2, b"exceed 2^31 slots"),
    ({"k_cache": 16, "v_cache": 16, "num_blocks": 4, "block_size": 16, "layout": 2}, 2, b"layout 2"),
    ({"k_cache": 16, "v_cache": 16, "num_blocks": 4, "block_size": 16}, 1, b"null"),
    ({"heads": 1 << 24}, 2, b"exceed one launch"),
])
def test_rotation_arguments_are_refused_without_a_launch(changes, code, message) -> None:
    lib = _lib.lib()
    assert lib.ayk_rotate_and_cache(*_rotate_args(**changes)) == code
    assert message in lib.ayk_last_error()


def test_rotation_of_no_rows_is_fine() -> None:
    assert _lib.lib().ayk_rotate_and_cache(*_rotate_args(n_rows=0, q=None, turns=None)) == 0


@pytest.mark.parametrize("changes,code,message", [
    ({"latent_dim": 511}, 2, b"latent_dim 511"),
    ({"rope_dim": 62}, 1, b"32 pairs do not fit a width of 62"),
    ({"rope_dim": 66}, 1, b"neither 0 nor half of rope_dim 66"),
    ({"pairs": 0}, 1, b"nothing to rotate them by"),
    ({"cache": None}, 1, b"null"),
    ({"slots": None}, 1, b"null"),
    ({"block_size": 70000}, 2, b"block_size 70000"),
    ({"latent": 3}, 1, b"multiple of the element's size"),
])
def test_latent_write_arguments_are_refused_without_a_launch(changes, code, message) -> None:
    args = dict(latent=16, latent_row=576, k_rope=16, k_row=576, q=16, q_row=64, q_head=64, q_out=16, q_out_row=64,
                q_out_head=64, cache=16, positions=16, slots=16, turns=16, pairs=32, interleaved=1, magnitude=1.0, n_rows=2,
                heads=1, latent_dim=512, rope_dim=64, num_blocks=4, block_size=16, dtype=1, stream=None)
    args.update(changes)
    lib = _lib.lib()
    assert lib.ayk_store_latent(*args.values()) == code
    assert message in lib.ayk_last_error()


@pytest.mark.parametrize("changes,code,message", [
    ({"n_rows": -1}, 1, b"n_rows -1"),
    ({"latent_dim": 384}, 2, b"latent_dim 384"),
    ({"rope_dim": 32}, 2, b"rope_dim 32"),
    ({"dtype": 3}, 2, b"dtype 3"),
    ({"heads": 0}, 1, b"num_heads 0"),
    ({"block_size": 0}, 2, b"block_size 0"),
    ({"max_blocks": 8, "stride": 4}, 1, b"table_stride 4"),
    ({"max_blocks": 1 << 24, "stride": 1 << 24}, 1, b"below 2^24"),
    ({"q": None}, 1, b"null"),
    ({"q": 8}, 1, b"16-byte aligned"),
    ({"workspace_bytes": 100}, 4, b"workspace"),
    ({"workspace": None}, 4, b"workspace"),
    ({"n_rows": 1 << 20, "heads": 1 << 12}, 2, b"exceed one launch"),
])
def test_latent_attention_arguments_are_refused_without_a_launch(changes, code, message) -> None:
    args = dict(out=16, q=16, cache=16, table=16, stride=4, lengths=16, rows=16, n_requests=2, n_rows=2, heads=8,
                latent_dim=512, rope_dim=64, num_blocks=4, block_size=16, max_blocks=4, dtype=1, scale=1.0, workspace=16,
                workspace_bytes=1 << 40, stream=None)
    args.update(changes)
    lib = _lib.lib()
    assert lib.ayk_latent_attention(*args.values()) == code
    assert message in lib.ayk_last_error()
    assert lib.ayk_latent_attention(*{**args, "n_rows": 0}.values()) in (0, code)


@pytest.mark.parametrize("changes,code,message", [
    ({"latent_dim": 128}, 2, b"latent_dim 128"),
    ({"rope_dim": 0}, 2, b"rope_dim 0"),
    ({"dtype": 2}, 2, b"dtype 2"),
    ({"at_once": 0}, 1, b"heads_at_once 0"),
    ({"ws_rows": 100}, 1, b"ws_rows 100"),
    ({"n_row_tiles": -1}, 1, b"-1 row tiles"),
    ({"row_tiles": None}, 1, b"null"),
    ({"token_tiles": None}, 1, b"null"),
    ({"keys": 24}, 1, b"16-byte aligned"),
    ({"workspace_bytes": 100}, 4, b"workspace"),
    ({"n_row_tiles": 1 << 30, "at_once": 8}, 2, b"exceed one launch"),
])
def test_latent_chunk_arguments_are_refused_without_a_launch(changes, code, message) -> None:
    args = dict(out=16, q=16, cache=16, keys=16, values=16, table=16, stride=4, token_tiles=16, n_token_tiles=1, row_tiles=16,
                n_row_tiles=1, ws_rows=128, at_once=8, heads=8, latent_dim=512, rope_dim=64, num_blocks=4, block_size=16,
                dtype=1, scale=1.0, workspace=16, workspace_bytes=1 << 40, stream=None)
    args.update(changes)
    lib = _lib.lib()
    assert lib.ayk_latent_chunks(*args.values()) == code
    assert message in lib.ayk_last_error()


def test_workspace_sizes() -> None:
    lib = _lib.lib()
    assert lib.ayk_latent_attention_workspace_bytes(0, 1, 8, 512) == 0
    assert lib.ayk_latent_attention_workspace_bytes(4, 4, 16, 384) == 0
    # 16 pairs a tile: a place, and two partials of 16 (m, l) and 16 x 512, a compute unit
    assert lib.ayk_latent_attention_workspace_bytes(4, 4, 16, 512) % (32 + 2 * 16 * (2 + 512) * 4) == 0
    assert lib.ayk_latent_chunks_workspace_bytes(256, 2) == 256 * 128 + 2 * (256 * 512 + 2 * 8)
    assert lib.ayk_latent_chunks_workspace_bytes(100, 2) == 0
    from ayaka_amd.hip import latent

    assert latent.TILE_TOKENS == latent.TILE_ROWS == 128


def test_chunk_tiles_cover_every_row_and_token_once() -> None:
    from ayaka_amd.hip import latent

    rows, lengths = [1, 300, 0, 128, 2, 5], [500, 300, 40, 129, 0, 1000]
    table = torch.arange(1, 1 + 6 * 63).view(6, 63)
    meta = hip_attention.plan(ForwardMode.MIXED, torch.tensor(rows), torch.tensor(lengths), table, 16)
    tokens, tiles, ws_rows = latent._chunk_tiles("op", meta.plan, torch.device("cpu"), False)
    seen, start = {}, {}
    for request, first, length, at in tokens.view(-1, 4).tolist():
        assert length == lengths[request] and first % 128 == 0 and at % 128 == 0
        start[request] = at - first
        for t in range(first, first + 128):
            assert seen.setdefault(at + t - first, (request, t)) == (request, t)
    assert sorted(seen) == list(range(ws_rows))
    assert sorted(start) == [b for b in range(6) if rows[b] and lengths[b]]
    covered, weight = set(), []
    for first, count, at, position in tiles.view(-1, 4).tolist():
        assert 1 <= count <= 128
        weight.append(position + count)
        for i in range(count):
            covered.add(first + i)
            request = int(meta.request_of_row[first + i])
            if lengths[request]:
                assert int(meta.positions[first + i]) == position + i and at == start[request]
            else:
                assert position == -count
    assert covered == set(range(sum(rows))) and weight == sorted(weight, reverse=True)


def test_weights_record() -> None:
    w = LatentWeights(torch.zeros(2, 128, 512), torch.zeros(2, 128, 512))
    assert w.keys.shape == w.values.shape
    assert isinstance(rotary(8, device="cpu"), Rotary)


def test_tile_pairs_for_known_lengths() -> None:
    """Small tiles while there is little to share, larger ones for many pairs over long contexts, never more
    than the requests hold."""
    import numpy as np

    lib = _lib.lib()

    def pairs(rows, lengths, heads):
        rows, lengths = np.array(rows, dtype=np.int32), np.array(lengths, dtype=np.int32)
        return lib.ayk_latent_tile_pairs(rows.ctypes.data, lengths.ctypes.data, len(rows), heads)

    assert pairs([1] * 64, [4096] * 64, 16) == 16
    assert pairs([4] * 32, [4096] * 32, 32) == 64
    assert pairs([1] * 256, [2048] * 256, 128) == 64
    assert pairs([8, 8], [26, 321], 16) == 16
    assert pairs([1], [0], 1) == pairs([0, 0], [5, 5], 128) == 16
    assert lib.ayk_latent_tile_pairs(None, None, 3, 16) == lib.ayk_latent_tile_pairs(16, 16, 0, 16) == 16
    for tile in (16, 32, 64):  # a place, and two partials of (m, l) and the sums, a compute unit
        assert lib.ayk_latent_tiles_workspace_bytes(512, tile) % (32 + 2 * tile * (2 + 512) * 4) == 0
    assert lib.ayk_latent_tiles_workspace_bytes(512, 48) == lib.ayk_latent_tiles_workspace_bytes(500, 16) == 0
    args = dict(out=16, q=16, cache=16, table=16, stride=4, lengths=16, rows=16, n_requests=2, n_rows=2, heads=8,
                latent_dim=512, rope_dim=64, num_blocks=4, block_size=16, max_blocks=4, dtype=1, scale=1.0, tile_pairs=48,
                workspace=16, workspace_bytes=1 << 40, stream=None)
    assert lib.ayk_latent_attention_tiles(*args.values()) == 1 and b"tile_pairs 48" in lib.ayk_last_error()
    args.update(tile_pairs=64, workspace_bytes=lib.ayk_latent_tiles_workspace_bytes(512, 64) - 1)
    assert lib.ayk_latent_attention_tiles(*args.values()) == 4 and b"workspace" in lib.ayk_last_error()


def test_parts_of_chunk_contexts() -> None:
    """Cut while workgroups are fewer than the compute units and contexts long; room for the parts."""
    from ayaka_amd.hip import latent

    def splits(rows, lengths, heads):
        table = torch.arange(1, 1 + len(rows) * 300).view(len(rows), 300)
        meta = hip_attention.plan(ForwardMode.MIXED, torch.tensor(rows), torch.tensor(lengths), table, 16)
        return latent._chunk_splits(meta.plan, sum(-(-r // 128) for r in rows), heads)

    assert splits([512] * 4, [4096] * 4, 16) == 1
    assert splits([300], [300], 16) == 1
    assert 2 <= splits([600], [4096], 4) <= 16
    assert splits([5, 0], [0, 7], 4) == 1
    lib = _lib.lib()
    assert lib.ayk_latent_chunks_parts_bytes(3, 4, 1) == lib.ayk_latent_chunks_parts_bytes(0, 4, 2) == 0
    assert lib.ayk_latent_chunks_parts_bytes(3, 4, 5) == 3 * 4 * 5 * 128 * 130 * 4
    args = dict(out=16, q=16, cache=16, keys=16, values=16, table=16, stride=4, token_tiles=16, n_token_tiles=1, row_tiles=16,
                n_row_tiles=1, ws_rows=128, at_once=8, heads=8, latent_dim=512, rope_dim=64, num_blocks=4, block_size=16,
                dtype=1, scale=1.0, splits=65, workspace=16, workspace_bytes=1 << 40, stream=None)
    assert lib.ayk_latent_chunks_split(*args.values()) == 1 and b"splits 65" in lib.ayk_last_error()
    room = -(-lib.ayk_latent_chunks_workspace_bytes(128, 8) // 16) * 16 + lib.ayk_latent_chunks_parts_bytes(1, 8, 3)
    args.update(splits=3, workspace_bytes=room - 1)
    assert lib.ayk_latent_chunks_split(*args.values()) == 4 and b"workspace" in lib.ayk_last_error()
