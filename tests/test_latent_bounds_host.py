"""Latent caches on the CPU: what the C entries accept at the ends of their ranges, and what steps they refuse."""

from __future__ import annotations

from ayaka_amd.hip import _lib


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
