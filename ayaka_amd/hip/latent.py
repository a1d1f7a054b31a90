"""Attention over latent caches: the host side of ``attention.attend_latent`` and
``attention.attend_latent_chunks`` (``include/ayaka_hip_latent.h``).

The first's launch reads lengths, rows and tables on the device and splits the step's contexts there,
so an eagerly planned step, a verify window and a captured bucket are the same call. The second's takes
tile lists of a planned step, made on its first call and kept in the plan, as the multi-row launch's.
The workspace of both is the one the device's split launches share.
"""

from __future__ import annotations

import numpy as np
import torch

from ayaka_amd.attention import AttentionMetadata
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import _fastpath, _lib
from ayaka_amd.hip._checks import capturing, dtype_name, require_device, require_latent_buffers, require_like, stream_handle
from ayaka_amd.kvcache import LatentBuffers, LatentWeights

__all__ = ["LATENT_DIMS", "ROPE_DIM", "attend_latent", "attend_latent_chunks"]

#: Widths of the latent, and of the rotary part, the kernels are built for.
LATENT_DIMS = frozenset({256, 512})
ROPE_DIM = 64
#: Widths of the expanded keys (without their rotary part) and values.
NOPE_DIM = VALUE_DIM = 128
#: Tokens of an expanded tile and rows of an attending one (the C library's).
TILE_TOKENS = TILE_ROWS = 128
#: Most bytes of expanded keys and values; a step that needs more expands some heads at a time.
EXPANDED_BYTES = 512 << 20
_DTYPE_CODES = {torch.float16: 0, torch.bfloat16: 1}


def _require_latent_step(op: str, q: torch.Tensor, buffers: LatentBuffers, meta: AttentionMetadata, out: torch.Tensor,
                         width: int, out_width: int) -> int:
    """The heads of a call of this backend's kernels: cache, step, q [N, heads, width] and out
    [N, heads, out_width] checked."""
    require_latent_buffers(op, buffers)
    cache, table = buffers.cache, meta.block_table
    if buffers.latent_dim not in LATENT_DIMS or buffers.rope_dim != ROPE_DIM:
        raise BackendError(
            f"{op}: the hip kernels are built for latents of {sorted(LATENT_DIMS)} elements and rotary parts of "
            f"{ROPE_DIM}, not {buffers.latent_dim} and {buffers.rope_dim}",
            context={"op": op, "argument": "buffers"},
        )
    if cache.dtype not in _DTYPE_CODES:
        raise BackendError(f"{op}: buffers.cache is {dtype_name(cache.dtype)}; over a latent cache the hip backend "
                           "computes in float16, bfloat16", context={"op": op, "argument": "buffers"})
    if not isinstance(meta.plan, (_attention.HipAttentionPlan, _attention.HipGraphPlan)) or not isinstance(table, torch.Tensor):
        raise BackendError(
            f"{op}: this step was planned by another backend; plan it with the same ops",
            context={"op": op, "argument": "meta"},
        )
    if meta.block_size != buffers.block_size:
        raise BackendError(
            f"{op}: the step was planned for blocks of {meta.block_size} positions "
            f"but the cache has blocks of {buffers.block_size}",
            context={"op": op, "argument": "meta"},
        )
    heads = q.shape[1] if q.ndim == 3 else 0
    if heads == 0:
        raise BackendError(f"{op}: q must be [N, heads, {width}], got {list(q.shape)}", context={"op": op, "argument": "q"})
    n_rows = meta.request_of_row.shape[0]
    require_like(op, "q", q, (n_rows, heads, width), cache.dtype)
    require_like(op, "out", out, (n_rows, heads, out_width), cache.dtype)
    for name, tensor in (("q", q), ("out", out), ("meta.kv_lengths", meta.kv_lengths), ("meta.block_table", table),
                         ("meta.rows_per_request", meta.rows_per_request)):
        require_device(op, name, tensor, cache.device)
    if table.dtype != torch.int32 or not table.is_contiguous() or table.ndim != 2:
        raise BackendError(f"{op}: meta.block_table must be a contiguous int32 [B, max_blocks] tensor")
    for name, tensor in (("meta.kv_lengths", meta.kv_lengths), ("meta.rows_per_request", meta.rows_per_request)):
        require_like(op, name, tensor, (table.shape[0],), torch.int32)
    return heads


def _require_described(op: str, step: "_attention.HipAttentionPlan", table: torch.Tensor, block_size: int, n_rows: int) -> None:
    """Refuse a plan whose lists, which the tiles are made of, are not of this table and these rows."""
    longest = max((length for count, length in zip(step.rows, step.kv_lengths) if count), default=0)
    if len(step.rows) != table.shape[0] or sum(step.rows) != n_rows or longest > table.shape[1] * block_size:
        raise BackendError(
            f"{op}: the step was planned for {len(step.rows)} requests of {sum(step.rows)} rows in all and up to {longest} "
            f"positions, its metadata has {n_rows} rows and a table of {list(table.shape)} blocks of {block_size}",
            context={"op": op, "argument": "meta"},
        )


def _replayed(meta: AttentionMetadata, key: tuple, keep: tuple, q: torch.Tensor, call) -> None:
    cache = getattr(meta.plan, "launches", None)
    if cache is None:
        call(None)
        return
    found = _fastpath.lookup(cache, key)
    if found is not None:
        stream = stream_handle(found.device)
        if found.scratch:
            _attention._order_scratch(found.device, stream, capturing(q))
        _fastpath.run(found, stream)
        return
    record = _fastpath.Recorder()
    call(record)
    _fastpath.remember(cache, key, keep, record)


def attend_latent(q: torch.Tensor, buffers: LatentBuffers, meta: AttentionMetadata, out: torch.Tensor, *,
                  scale: float) -> None:
    """Attention of every row over its request's latent context, keys and values absorbed.

    ``q`` [N, heads, latent_dim + 64] holds each head's query taken through the keys' matrix, and behind
    it its rotated part (what ``store_latent`` rotates); the score of a cached row is their product
    times ``scale``, and ``out`` [N, heads, latent_dim] receives the weighted sum of the latents, for the
    values' matrix to be applied to. Rows see positions up to their own; padding rows get zeros. ``out``
    overlaps no input.
    Any step serves: decode, verify windows, chunks (``attend_latent_chunks`` does those of many rows
    with a third of the work per score), graph metadata. Captured after one eager call. Caches are float16, with
    weights in float16 (within 2^-11 of themselves, or 2^-32 of a row's largest), or bfloat16, with weights of 16 bits
    or more; ``store_latent`` writes float32 ones too, which this backend does not attend to.
    """
    op = "attention.attend_latent"
    key = ("attend_latent", id(buffers), id(meta), scale, _fastpath.signature((q, out, buffers.k)))
    _replayed(meta, key, (buffers, meta), q, lambda record: _attend_latent(op, q, buffers, meta, out, scale, record))


def _attend_latent(op: str, q: torch.Tensor, buffers: LatentBuffers, meta: AttentionMetadata, out: torch.Tensor,
                   scale: float, record: "_fastpath.Recorder | None") -> None:
    require_latent_buffers(op, buffers)
    heads = _require_latent_step(op, q, buffers, meta, out, buffers.latent_dim + buffers.rope_dim, buffers.latent_dim)
    cache, table, n_rows = buffers.cache, meta.block_table, q.shape[0]
    if n_rows == 0:
        return
    device, lib = cache.device, _lib.lib()
    stream, requests = stream_handle(device), table.shape[0]
    pairs = _tile_pairs(meta.plan, n_rows, requests, heads)
    nbytes = lib.ayk_latent_tiles_workspace_bytes(buffers.latent_dim, pairs)
    scratch = _attention._workspace(op, device, nbytes, capturing(q), stream)
    _attention._call(op, lib.ayk_latent_attention_tiles, (
        out.data_ptr(), q.data_ptr(), cache.data_ptr(), table.data_ptr(), table.stride(0), meta.kv_lengths.data_ptr(),
        meta.rows_per_request.data_ptr(), requests, n_rows, heads, buffers.latent_dim, buffers.rope_dim,
        buffers.num_blocks, buffers.block_size, table.shape[1], _DTYPE_CODES[cache.dtype], float(scale), pairs,
        scratch.data_ptr(), scratch.numel(),
    ), stream, device, True, record)


def _tile_pairs(plan: "_attention.HipAttentionPlan | _attention.HipGraphPlan", n_rows: int, requests: int, heads: int) -> int:
    """(Row, head) pairs of a tile: for the step's lengths, or for a bucket's 2048 positions a request."""
    known = isinstance(plan, _attention.HipAttentionPlan)
    found = plan.splits.get(("latent", heads)) if known else None
    if found is None:
        rows, lengths = (plan.rows, plan.kv_lengths) if known else ((-(-n_rows // requests),) * requests, (2048,) * requests)
        rows, lengths = np.array(rows, dtype=np.int32), np.array(lengths, dtype=np.int32)
        found = _lib.lib().ayk_latent_tile_pairs(rows.ctypes.data, lengths.ctypes.data, len(rows), heads)
        if known:
            plan.splits["latent", heads] = found
    return found


def _chunk_tiles(op: str, step: "_attention.HipAttentionPlan", device: torch.device,
                 capture: bool) -> tuple[torch.Tensor, torch.Tensor, int]:
    """The step's token tiles and row tiles (heaviest first) on the device, and its workspace rows."""
    found = step.work.get("latent-chunks")
    if found is not None:
        return found
    if capture:
        raise BackendError(f"{op}: the tile lists of this step are built on its first call; run the step once "
                           "eagerly before capturing it", context={"op": op})
    tokens, rows, ws_rows, first_row = [], [], 0, 0
    for request, (count, length) in enumerate(zip(step.rows, step.kv_lengths)):
        base = first_row + np.arange(0, count, TILE_ROWS)
        size = np.minimum(TILE_ROWS, first_row + count - base)
        if count and length:
            at = np.arange(0, length, TILE_TOKENS)
            tokens.append(np.stack((np.full_like(at, request), at, np.full_like(at, length), ws_rows + at), axis=1))
            rows.append(np.stack((base, size, np.full_like(base, ws_rows), length - count + base - first_row), axis=1))
            ws_rows += at.size * TILE_TOKENS
        elif count:
            rows.append(np.stack((base, size, np.zeros_like(base), -size), axis=1))
        first_row += count
    if ws_rows > np.iinfo(np.int32).max:
        raise BackendError(f"{op}: contexts of {ws_rows} positions in all exceed one launch", context={"op": op})
    row_list = np.concatenate(rows)
    row_list = row_list[np.argsort(-(row_list[:, 1] + row_list[:, 3]), kind="stable")]
    token_list = np.concatenate(tokens) if tokens else np.zeros((0, 4), dtype=np.int64)
    found = (*(torch.from_numpy(x.astype(np.int32).reshape(-1)).to(device) for x in (token_list, row_list)), ws_rows)
    step.work["latent-chunks"] = found
    return found


def _chunk_splits(step: "_attention.HipAttentionPlan", n_tiles: int, heads: int) -> int:
    """Parts to cut each row tile's context into. A workgroup takes about 1.55 us a round of 64 positions and 8 us
    to start and end, and parts cost about 6 us for their joining; the rounds of all are dealt to the compute
    units, none of which is done before the longest tile. Cut where that saves 15% (of the whole call: chunks of 600
    rows of 4 and 8 heads over 3.6K positions 85 and 96 us whole, 42 and 49 cut; of 20 heads over 1.6K, where the
    model saves 7%, 70 whole and 85 cut)."""
    found = step.splits.get(("latent-chunks", n_tiles, heads))
    if found is None:
        longest, total = 0, 0
        for count, length in zip(step.rows, step.kv_lengths):
            if count and length:
                ends = np.minimum(length, length - count + np.arange(TILE_ROWS, count + TILE_ROWS, TILE_ROWS))
                rounds = -(-ends // 64)
                longest, total = max(longest, int(rounds.max())), total + int(rounds.sum())

        def us(parts: int) -> float:
            waves = -(-n_tiles * heads * parts // _attention.COMPUTE_UNITS)
            return (max(-(-longest // parts), total * heads / _attention.COMPUTE_UNITS) * 1.55 + 8 * waves
                    + (6 if parts > 1 else 0))

        found = min((p for p in (1, 2, 3, 4, 6, 8, 12, 16) if p == 1 or 2 * p <= longest), key=us)
        if us(found) > 0.85 * us(1):
            found = 1
        step.splits["latent-chunks", n_tiles, heads] = found
    return found


def attend_latent_chunks(q: torch.Tensor, weights: LatentWeights, buffers: LatentBuffers, meta: AttentionMetadata,
                         out: torch.Tensor, *, scale: float) -> None:
    """Attention of chunks of rows over their requests' latent contexts, keys and values expanded.

    Head h's key of a position is ``weights.keys[h] @ latent`` with the position's rotary part behind it,
    its value ``weights.values[h] @ latent``; ``q`` [N, heads, 128 + 64] are the queries as projected, with
    their rotary part rotated, and ``out`` [N, heads, 128], which overlaps no input, are the heads' outputs. The context's keys and
    values are expanded once for all rows, into scratch, so this is for steps of many rows per request
    (some hundred; ``attend_latent`` serves the others without expanding). For steps made by ``plan``;
    captured after one eager call. Expanded keys and values are held in fp16 with a scale for every 128
    positions of a head: each element is within 2^-11 of itself, whatever its magnitude, or within 2^-38 of
    the largest finite one of those positions (for rows before that one too). Weights are fp16 as well: each weight
    times value is within 2^-11 of itself, or within 2^-32 of the largest weight times largest value of its 128
    positions that the row's sum has met; the sum of weights sees no value. Of queries the first 128 elements are fp16
    under a scale of each row's own.
    """
    op = "attention.attend_latent_chunks"
    key = ("attend_latent_chunks", id(buffers), id(meta), scale,
           _fastpath.signature((q, out, buffers.k, weights.keys, weights.values)))
    _replayed(meta, key, (buffers, meta), q,
              lambda record: _attend_latent_chunks(op, q, weights, buffers, meta, out, scale, record))


def _attend_latent_chunks(op: str, q: torch.Tensor, weights: LatentWeights, buffers: LatentBuffers,
                          meta: AttentionMetadata, out: torch.Tensor, scale: float,
                          record: "_fastpath.Recorder | None") -> None:
    heads = _require_latent_step(op, q, buffers, meta, out, NOPE_DIM + ROPE_DIM, VALUE_DIM)
    cache, table, step = buffers.cache, meta.block_table, meta.plan
    for name, tensor, width in (("weights.keys", weights.keys, NOPE_DIM), ("weights.values", weights.values, VALUE_DIM)):
        require_like(op, name, tensor, (heads, width, buffers.latent_dim), cache.dtype)
        require_device(op, name, tensor, cache.device)
    if not isinstance(step, _attention.HipAttentionPlan):
        raise BackendError(f"{op}: needs a step made by plan; a decode bucket's rows take attend_latent",
                           context={"op": op, "argument": "meta"})
    _require_described(op, step, table, meta.block_size, q.shape[0])
    if q.shape[0] == 0:
        return
    device, lib, capture = cache.device, _lib.lib(), capturing(q)
    tokens, rows, ws_rows = _chunk_tiles(op, step, device, capture)
    at_once = heads if ws_rows == 0 else max(1, min(heads, EXPANDED_BYTES // (ws_rows * 512)))
    if at_once >= 8:
        at_once -= at_once % 8 if at_once < heads else 0  # (a head's workgroups then share an XCD)
    stream, n_tiles = stream_handle(device), rows.numel() // 4
    splits = _chunk_splits(step, n_tiles, at_once)
    nbytes = (-(-lib.ayk_latent_chunks_workspace_bytes(ws_rows, at_once) // 16) * 16
              + lib.ayk_latent_chunks_parts_bytes(n_tiles, at_once, splits))
    scratch = _attention._workspace(op, device, nbytes, capture, stream)
    _attention._call(op, lib.ayk_latent_chunks_split, (
        out.data_ptr(), q.data_ptr(), cache.data_ptr(), weights.keys.data_ptr(), weights.values.data_ptr(),
        table.data_ptr(), table.stride(0), tokens.data_ptr(), tokens.numel() // 4, rows.data_ptr(), n_tiles,
        ws_rows, at_once, heads, buffers.latent_dim, buffers.rope_dim, buffers.num_blocks, buffers.block_size,
        _DTYPE_CODES[cache.dtype], float(scale), splits, scratch.data_ptr(), scratch.numel(),
    ), stream, device, True, record)


# last: attention takes this module's ops into its family, and this module its plans and scratch
from ayaka_amd.hip import attention as _attention  # noqa: E402
