"""Attention over latent caches through the C entries themselves, and what lies beside its buffers."""

from __future__ import annotations

import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType
from ayaka_amd.hip import _lib
from ayaka_amd.hip import latent as hip_latent
from tests.test_gpu_latent import DEV, TYPES, Scene

pytestmark = pytest.mark.gpu

GUARD = 4096  # bytes


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


def guarded(shape, dtype, fill: float) -> tuple[torch.Tensor, torch.Tensor]:
    """A tensor, and the one it is the middle of."""
    n, guard = torch.Size(shape).numel(), GUARD // dtype.itemsize
    whole = torch.full((n + 2 * guard,), fill, dtype=dtype, device=DEV)
    return whole[guard:guard + n].view(shape), whole


def untouched(whole: torch.Tensor, fill: float) -> bool:
    guard = GUARD // whole.dtype.itemsize
    return bool((whole[:guard] == fill).all()) and bool((whole[-guard:] == fill).all())


@pytest.mark.parametrize("rows", [[2, 1], [2, 900], [1, 3], [0, 5], [2, 0]])
def test_device_rows_other_than_the_plans(ops, rows) -> None:
    """Rows on the device that are not the plan's: requests have theirs as far as there are rows of queries, the
    others stay as they were, and nothing beside queries and outputs is touched."""
    s = Scene(ops, [(2, 100), (3, 40)], heads=4, seed=14)
    q, _ = guarded(s.q.shape, s.dtype, float("nan"))
    s.q = q.copy_(s.q)
    out, whole = guarded(s.out().shape, s.dtype, 7.0)
    s.meta.rows_per_request.copy_(torch.tensor(rows, dtype=torch.int32))
    s.run(out)
    torch.cuda.synchronize()
    assert untouched(whole, 7.0)
    if rows == [2, 900]:  # the first of 900 rows lie before the context's first position
        assert not bool(out[2:].any())
        rows = [2, 0]
    else:
        assert bool((out[sum(rows):] == 7.0).all())
    # (not the planned call's bits: where contexts are cut among workgroups goes by all rows)
    s.rows, s.q = rows, s.q[:sum(rows)]
    s.check(out[:sum(rows)].contiguous())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("latent,heads", [(512, 3), (256, 40)])
def test_attention_in_exactly_its_workspace(ops, dtype, latent, heads) -> None:
    lib = _lib.lib()
    s = Scene(ops, [(1, 700), (4, 130), (1, 0), (30, 64)], dtype=dtype, latent=latent, heads=heads, seed=61)
    n, m = len(s.q), s.meta
    size = lib.ayk_latent_attention_workspace_bytes(n, len(s.rows), heads, latent)
    workspace, whole = guarded((size,), torch.uint8, 0xA5)
    out, out_whole = guarded(s.out().shape, s.dtype, 7.0)
    args = (out.data_ptr(), s.q.data_ptr(), s.cache.data_ptr(), m.block_table.data_ptr(), m.block_table.stride(0),
            m.kv_lengths.data_ptr(), m.rows_per_request.data_ptr(), len(s.rows), n, heads, latent, 64, s.blocks, s.block,
            m.block_table.shape[1], int(dtype == "bf16"), s.scale, workspace.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.ayk_latent_attention(*args, size - 1, stream) == 4
    assert lib.ayk_latent_attention(*args, size, stream) == 0, lib.ayk_last_error()
    s.check(out)
    assert untouched(whole, 0xA5) and untouched(out_whole, 7.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,at_once", [(3, 3), (5, 3), (8, 1)])
def test_chunks_in_exactly_their_workspace(ops, monkeypatch, dtype, heads, at_once) -> None:
    """Sizes of 8 past a multiple of 16 among them, and heads that come some at a time."""
    monkeypatch.setattr(hip_latent, "_chunk_splits", lambda *_: 1)
    lib = _lib.lib()
    s = Scene(ops, [(40, 300), (1, 0), (130, 200)], form="chunks", dtype=dtype, latent=256, heads=heads, seed=62)
    m = s.meta
    tokens, tiles, ws_rows = hip_latent._chunk_tiles("op", m.plan, DEV, False)
    size = lib.ayk_latent_chunks_workspace_bytes(ws_rows, at_once)
    workspace, whole = guarded((size,), torch.uint8, 0xA5)
    out, out_whole = guarded(s.out().shape, s.dtype, 7.0)
    args = (out.data_ptr(), s.q.data_ptr(), s.cache.data_ptr(), s.weights.keys.data_ptr(), s.weights.values.data_ptr(),
            m.block_table.data_ptr(), m.block_table.stride(0), tokens.data_ptr(), tokens.numel() // 4, tiles.data_ptr(),
            tiles.numel() // 4, ws_rows, at_once, heads, 256, 64, s.blocks, s.block, int(dtype == "bf16"), s.scale,
            workspace.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.ayk_latent_chunks(*args, size - 1, stream) == 4
    assert lib.ayk_latent_chunks(*args, size, stream) == 0, lib.ayk_last_error()
    torch.cuda.synchronize()
    assert untouched(whole, 0xA5) and untouched(out_whole, 7.0)
    assert torch.equal(out, s.run())
    s.check(out)
