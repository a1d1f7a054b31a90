"""Latent caches on the CPU: what the C entries accept at the ends of their ranges, and what steps they refuse."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from ayaka_amd.enums import ForwardMode
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import _lib
from ayaka_amd.hip import attention as hip_attention
from ayaka_amd.hip import kvcache as hip_kvcache
from ayaka_amd.hip import latent
from ayaka_amd.rotary import rotary


def _chunk_args(**kw) -> dict:
    args = dict(out=16, q=16, cache=16, keys=16, values=16, table=16, stride=4, token_tiles=16, n_token_tiles=1, row_tiles=16,
                n_row_tiles=(1 << 31) - 1, ws_rows=128, at_once=3, heads=3, latent_dim=512, rope_dim=64, num_blocks=4,
                block_size=16, dtype=1, scale=1.0, workspace=16, workspace_bytes=0, stream=None)
    assert not set(kw) - set(args)
    return {**args, **kw}


def test_the_documented_workspace_of_chunks_is_enough() -> None:
    """Sizes that are no multiple of 16 too. (More tiles than one launch takes, which is looked at behind the workspace,
    so that nothing is launched.)"""
    lib = _lib.lib()
    for ws_rows, heads in ((128, 3), (384, 3), (128, 5), (256, 3), (640, 7)):
        size = lib.ayk_latent_chunks_workspace_bytes(ws_rows, heads)
        args = _chunk_args(ws_rows=ws_rows, at_once=heads, heads=heads, workspace_bytes=size)
        assert lib.ayk_latent_chunks(*args.values()) == 2, lib.ayk_last_error()
        assert b"exceed one launch" in lib.ayk_last_error()
        args["workspace_bytes"] -= 1
        assert lib.ayk_latent_chunks(*args.values()) == 4
        assert f"{size} are needed".encode() in lib.ayk_last_error()


def _attention_args(**kw) -> dict:
    args = dict(out=16, q=16, cache=16, table=16, stride=0, lengths=16, rows=16, n_requests=0, n_rows=0, heads=1,
                latent_dim=512, rope_dim=64, num_blocks=4, block_size=7, max_blocks=0, dtype=1, scale=1.0, tile_pairs=64,
                workspace=16, workspace_bytes=1 << 40, stream=None)
    assert not set(kw) - set(args)
    return {**args, **kw}


def test_the_units_of_a_launch_stay_below_2_to_31() -> None:
    """What the kernel counts in 32 bits: every tile's chunks of 32 positions, the last one begun, and the tile's own
    cost (8 chunks with 64 pairs, 5 with fewer), for as many tiles as rows and requests can make."""
    lib = _lib.lib()
    for pairs, cost in ((16, 5), (32, 5), (64, 8)):
        for blocks in (1, 9, 147):  # 7, 63, 1029 positions: 1, 2, 33 chunks, of which the last holds 7, 31, 5
            chunks = -(-blocks * 7 // 32) + cost
            tiles = (1 << 31) // chunks  # the first number of tiles whose units may reach 2^31
            while tiles * chunks < 1 << 31:
                tiles += 1
            requests = tiles - tiles // 2
            rows = (tiles - requests) * pairs  # of one head: that many tiles, and one begun for every request
            args = _attention_args(n_requests=requests, n_rows=rows, max_blocks=blocks, stride=blocks, tile_pairs=pairs)
            if rows > (1 << 31) - 1:
                continue
            assert lib.ayk_latent_attention_tiles(*args.values()) == 2, (pairs, blocks)
            assert b"exceed one launch" in lib.ayk_last_error()


def test_steps_with_fewer_positions_than_rows_are_refused() -> None:
    """Metadata whose positions were replaced by others: a row without one would read past them."""
    meta = hip_attention.plan(ForwardMode.DECODE, torch.ones(4, dtype=torch.int32), torch.full((4,), 3, dtype=torch.int32),
                              torch.arange(1, 5, dtype=torch.int32)[:, None], 16)
    turn, cpu = rotary(64, device="cpu"), torch.device("cpu")
    assert hip_kvcache._rotation("op", meta, turn, cpu, 64, 4)[1][1:] == (32, 0, 1.0)
    assert hip_kvcache._rotation("op", meta, None, cpu, 64, 4) == (0, (0, 0, 0, 1.0))
    for positions in (meta.positions[:3], meta.positions[:0], torch.zeros(5, dtype=torch.int32), torch.zeros(4, 1, dtype=torch.int32)):
        other = dataclasses.replace(meta, positions=positions)
        with pytest.raises(BackendError, match=r"meta.positions must be a contiguous int32 \[4\]"):
            hip_kvcache._rotation("op", other, turn, cpu, 64, 4)


def test_chunks_refuse_a_plan_of_another_step() -> None:
    """Tile lists come from the plan's lengths: a table, or rows, that they do not describe would be read past."""
    rows, lengths = torch.tensor([3, 1, 0], dtype=torch.int32), torch.tensor([40, 17, 90], dtype=torch.int32)
    table = torch.arange(1, 19, dtype=torch.int32).view(3, 6)
    meta = hip_attention.plan(ForwardMode.MIXED, rows, lengths, table, 16)
    latent._require_described("op", meta.plan, meta.block_table, 16, 4)
    latent._require_described("op", meta.plan, meta.block_table[:, :3], 16, 4)  # no row attends to the third request
    for block_table, block_size, n_rows in (
        (meta.block_table[:, :2], 16, 4), (meta.block_table[:2], 16, 4), (meta.block_table, 6, 4), (meta.block_table, 16, 3),
        (meta.block_table, 16, 5),
    ):
        with pytest.raises(BackendError, match="planned for 3 requests of 4 rows in all and up to 40 positions"):
            latent._require_described("op", meta.plan, block_table, block_size, n_rows)
