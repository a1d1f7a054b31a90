"""KV-cache ops with the MI355X kernels; implements the ``KVCacheOps`` contract.

``store`` is the KV write (``ayk_reshape_and_cache``): row ``i`` of ``k``/``v``
lands bit for bit in slot ``meta.slot_mapping[i]`` (reference
``python/ayaka/ops/backends/torch/kvcache.py:65-80``); into a ``"fp8_e4m3"``
cache it lands encoded (``ayk_reshape_and_cache_e4m3``), into a
``"fp8_e4m3_block"`` cache encoded with its block's scales, which the write
raises where it has to (``ayk_store_block_scaled``). ``gather``,
``copy_blocks`` and ``zero_blocks`` move whole blocks (same file, ``:83-115``),
of a block-scaled cache with their scales. ``build_tables`` gives a step's
requests the blocks they lack and derives its slots on the device
(``ayk_build_tables``). ``rotate``, ``store_rotated`` and ``store_latent`` apply a step's
rotary positions, the last two together with the cache write
(``include/ayaka_hip_latent.h``).
Both layouts are served; NHD is preferred, as the reference's ``layout()``
returns (``:30-31``).
"""

from __future__ import annotations

import torch

from ayaka_amd.attention import AttentionMetadata
from ayaka_amd.enums import KVLayoutKind
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import _fastpath, _lib
from ayaka_amd.hip._checks import (
    block_scales,
    compute_dtype,
    dtype_name,
    require_buffers,
    require_device,
    require_index_tensor,
    require_latent_buffers,
    require_like,
    require_pool,
    require_rotary,
    require_rows,
    stream_handle,
)
from ayaka_amd.kvcache import FP8_E4M3_CODEC, RAW_CODEC, BlockPool, KVBuffers, LatentBuffers, StepTables, codec_scales
from ayaka_amd.rotary import Rotary

__all__ = ["build_tables", "copy_blocks", "gather", "layout", "rotate", "store", "store_latent", "store_rotated",
           "zero_blocks"]

_LAYOUT_CODES = {KVLayoutKind.NHD: 0, KVLayoutKind.HND: 1}
_DTYPE_CODES = {torch.float16: 0, torch.bfloat16: 1}
_ROW_DTYPE_CODES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 3}
_I32 = torch.int32


def layout() -> KVLayoutKind:
    return KVLayoutKind.NHD


def _stream(device: torch.device) -> int:
    return stream_handle(device)


def _block_bytes(buffers: KVBuffers) -> int:
    return buffers.k[0].numel() * buffers.k.element_size()


def _ids(op: str, name: str, ids: torch.Tensor, device: torch.device) -> None:
    require_index_tensor(op, name, ids, ndim=1)
    require_device(op, name, ids, device)
    if not ids.is_contiguous():
        raise BackendError(f"{op}: {name} must be contiguous", context={"op": op, "argument": name})


def store(k: torch.Tensor, v: torch.Tensor, buffers: KVBuffers, meta: AttentionMetadata) -> None:
    """Write each row's k and v into its slot (reference ``torch/kvcache.py:65-80``).

    As ``attend``: the first call with a combination of k, v, buffers and step metadata is
    checked in full and recorded in the step's plan; later calls with the same buffers and
    metadata, and k and v at the same addresses, shapes, strides and dtype, replay the library
    call on the current stream.
    """
    cache = getattr(meta.plan, "launches", None)
    if cache is None:
        _store(k, v, buffers, meta, None)
        return
    scales = block_scales(buffers)
    key = ("store", id(buffers), id(meta), _fastpath.signature((k, v, buffers.k, buffers.v)),
           0 if scales is None else scales.data_ptr())
    found = _fastpath.lookup(cache, key)
    if found is not None:
        _fastpath.run(found, _stream(found.device))
        return
    record = _fastpath.Recorder()
    _store(k, v, buffers, meta, record)
    _fastpath.remember(cache, key, (buffers, meta), record)


def _store(k: torch.Tensor, v: torch.Tensor, buffers: KVBuffers, meta: AttentionMetadata,
           record: "_fastpath.Recorder | None") -> None:
    op = "kvcache.store"
    require_buffers(op, buffers)
    if meta.block_size != buffers.block_size:
        raise BackendError(
            f"{op}: the step was planned for blocks of {meta.block_size} positions "
            f"but the cache has blocks of {buffers.block_size}",
            context={"op": op, "argument": "meta"},
        )
    rows = meta.slot_mapping.shape[0]
    shape = (rows, buffers.num_kv_heads, buffers.head_dim)
    dtype = compute_dtype(op, "k", k, buffers)
    require_like(op, "k", k, shape, dtype)
    require_like(op, "v", v, shape, dtype)
    device = buffers.k.device
    for name, tensor in (("k", k), ("v", v), ("meta.slot_mapping", meta.slot_mapping)):
        require_device(op, name, tensor, device)
    slots = meta.slot_mapping
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        raise BackendError(f"{op}: meta.slot_mapping must be a contiguous int64 tensor")
    if rows == 0:
        return
    scales = block_scales(buffers)
    if scales is not None:
        fn = _lib.lib().ayk_store_block_scaled
        args = (k.data_ptr(), v.data_ptr(), buffers.k.data_ptr(), buffers.v.data_ptr(), scales.data_ptr(),
                slots.data_ptr(), rows, buffers.num_kv_heads, buffers.head_dim, buffers.num_blocks,
                buffers.block_size, _LAYOUT_CODES[KVLayoutKind(buffers.layout)], _DTYPE_CODES[dtype])
    elif buffers.codec == FP8_E4M3_CODEC:
        fn = _lib.lib().ayk_reshape_and_cache_e4m3
        args = (k.data_ptr(), v.data_ptr(), buffers.k.data_ptr(), buffers.v.data_ptr(), slots.data_ptr(), rows,
                buffers.num_kv_heads, buffers.head_dim, buffers.num_blocks, buffers.block_size,
                _LAYOUT_CODES[KVLayoutKind(buffers.layout)], _DTYPE_CODES[dtype], *codec_scales(buffers.codec))
    else:
        fn = _lib.lib().ayk_reshape_and_cache
        args = (k.data_ptr(), v.data_ptr(), buffers.k.data_ptr(), buffers.v.data_ptr(), slots.data_ptr(), rows,
                buffers.num_kv_heads, buffers.head_dim, buffers.num_blocks, buffers.block_size,
                _LAYOUT_CODES[KVLayoutKind(buffers.layout)], buffers.k.element_size())
    if record is not None:
        record(op, fn, args, device, False)
    _lib.check(op, fn(*args, _stream(device)))


def _rotation(op: str, meta: AttentionMetadata, rotary: Rotary | None, device: torch.device,
              width: int, n_rows: int) -> tuple:
    """The entry points' positions, and turns, pairs, order and magnitude of a rotation of rows of
    ``width`` elements (``None``: nothing turns)."""
    if rotary is None:
        return 0, (0, 0, 0, 1.0)
    pairs = require_rotary(op, rotary, device)
    if 2 * pairs > width:
        raise BackendError(f"{op}: the rotation turns {2 * pairs} elements of heads of {width}",
                           context={"op": op, "argument": "rotary"})
    positions = meta.positions
    if positions.dtype != _I32 or not positions.is_contiguous() or tuple(positions.shape) != (n_rows,):
        raise BackendError(f"{op}: meta.positions must be a contiguous int32 [{n_rows}] tensor, got "
                           f"{dtype_name(positions.dtype)} {list(positions.shape)}", context={"op": op, "argument": "meta"})
    require_device(op, "meta.positions", positions, device)
    return positions.data_ptr(), (rotary.turns.data_ptr(), pairs, int(rotary.interleaved), float(rotary.magnitude))


def _slots(op: str, meta: AttentionMetadata, buffers: "KVBuffers | LatentBuffers") -> torch.Tensor:
    if meta.block_size != buffers.block_size:
        raise BackendError(
            f"{op}: the step was planned for blocks of {meta.block_size} positions "
            f"but the cache has blocks of {buffers.block_size}",
            context={"op": op, "argument": "meta"},
        )
    slots = meta.slot_mapping
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        raise BackendError(f"{op}: meta.slot_mapping must be a contiguous int64 tensor")
    require_device(op, "meta.slot_mapping", slots, buffers.k.device)
    return slots


def _turned(op: str, name: str, rows: torch.Tensor, out: torch.Tensor | None, n_rows: int, width: int,
            dtype: torch.dtype, device: torch.device) -> tuple[int, tuple]:
    """Rows [N, heads, width] to rotate, into ``out`` or in place: the heads, and the entry points'
    addresses and strides."""
    out = rows if out is None else out
    heads = rows.shape[1] if rows.ndim == 3 else 0
    shape = (n_rows, heads, width)
    require_rows(op, name, rows, shape, dtype, device, written=out is rows)
    if out is not rows:
        require_rows(op, f"{name}_out", out, shape, dtype, device, written=True)
        if out.data_ptr() == rows.data_ptr() and out.stride() != rows.stride() and rows.numel():
            raise BackendError(f"{op}: {name}_out shares memory with {name} at other strides",
                               context={"op": op, "argument": f"{name}_out"})
    return heads, (rows.data_ptr(), *rows.stride()[:2], out.data_ptr(), *out.stride()[:2])


_NO_ROWS = (0, 0, 0, 0, 0, 0)


def _given(*tensors: torch.Tensor | None) -> tuple[tuple, int]:
    """Those of a call's tensors that are not ``None``, and which are, as bits. (A rotation's own tensor
    is not among them: it goes by the rotation's identity, which is frozen and kept.)"""
    absent = 0
    for i, t in enumerate(tensors):
        if t is None:
            absent |= 1 << i
    return tuple([t for t in tensors if t is not None]) if absent else tensors, absent


def _replayed(meta: AttentionMetadata, key: tuple, keep: tuple, call) -> None:
    """``call(record)``, or the launch it recorded in the step's plan when it ran with this ``key``."""
    cache = getattr(meta.plan, "launches", None)
    if cache is None:
        call(None)
        return
    found = _fastpath.lookup(cache, key)
    if found is not None:
        _fastpath.run(found, _stream(found.device))
        return
    record = _fastpath.Recorder()
    call(record)
    _fastpath.remember(cache, key, keep, record)


def rotate(q: torch.Tensor | None, k: torch.Tensor | None, meta: AttentionMetadata, rotary: Rotary,
           q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> None:
    """Rotate a step's queries and keys by their positions, in place or into ``q_out`` and ``k_out``.

    ``q`` [N, heads, head_dim] and ``k`` [N, kv_heads, head_dim] may be views of a larger tensor (the
    parts of one projection's output) whose heads are contiguous; either may be ``None``. Row i turns by
    ``meta.positions[i]``; of each head the first ``2 * len(rotary.turns)`` elements turn and the others
    are copied. Angles are reduced in 64 bits, products are fp32, each result is rounded once. An
    output is its input or overlaps neither input. For caches that ``store_rotated`` does not
    write: ``store`` takes the rotated keys.
    """
    op = "kvcache.rotate"
    if q is None and k is None:
        raise BackendError(f"{op}: neither q nor k is given", context={"op": op})
    tensors, absent = _given(q, k, q_out, k_out)
    key = ("rotate", id(meta), id(rotary), absent, _fastpath.signature(tensors))
    _replayed(meta, key, (meta, rotary), lambda record: _rotate(op, q, k, meta, rotary, q_out, k_out, record))


def _rotate(op: str, q, k, meta: AttentionMetadata, rotary: Rotary, q_out, k_out, record) -> None:
    first = q if q is not None else k
    if first.ndim != 3 or first.dtype not in _ROW_DTYPE_CODES or not first.is_cuda:
        raise BackendError(
            f"{op}: rows must be float16, bfloat16 or float32 [N, heads, head_dim] on a HIP device, got "
            f"{first.dtype} {list(first.shape)} on {first.device}", context={"op": op})
    n_rows, width, dtype, device = meta.positions.shape[0], first.shape[2], first.dtype, first.device
    heads, q_args = _turned(op, "q", q, q_out, n_rows, width, dtype, device) if q is not None else (0, _NO_ROWS)
    kv_heads, k_args = _turned(op, "k", k, k_out, n_rows, width, dtype, device) if k is not None else (0, _NO_ROWS)
    positions, turn = _rotation(op, meta, rotary, device, width, n_rows)
    if n_rows == 0:
        return
    _launch(op, _lib.lib().ayk_rotate_and_cache, (
        *q_args, *k_args, 0, 0, 0, 0, 0, positions, 0, *turn, n_rows, heads, kv_heads, width, 0, 0, 0,
        _ROW_DTYPE_CODES[dtype]), device, record)


def _launch(op: str, fn, args: tuple, device: torch.device, record: "_fastpath.Recorder | None") -> None:
    if record is not None:
        record(op, fn, args, device, False)
    _lib.check(op, fn(*args, _stream(device)))


def store_rotated(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, buffers: KVBuffers,
                  meta: AttentionMetadata, rotary: Rotary, q_out: torch.Tensor | None = None) -> None:
    """Rotate a step's queries and keys by their positions and write the keys and values into the cache.

    What ``rotate`` and then ``store`` would do, in one launch: ``q`` is rotated in place or into
    ``q_out`` (see :func:`rotate`), the rotated ``k`` and ``v`` go to the slots of ``meta`` and are left
    as they are themselves. Both may be views, as ``q``. The cache is of the ``"raw"`` codec in the dtype
    of the rows. Rows of padding requests are not stored.
    """
    op = "kvcache.store_rotated"
    tensors, absent = _given(k, v, buffers.k, buffers.v, q, q_out)
    key = ("store_rotated", id(buffers), id(meta), id(rotary), absent, _fastpath.signature(tensors))
    _replayed(meta, key, (buffers, meta, rotary),
              lambda record: _store_rotated(op, q, k, v, buffers, meta, rotary, q_out, record))


def _store_rotated(op: str, q, k, v, buffers: KVBuffers, meta: AttentionMetadata, rotary: Rotary, q_out, record) -> None:
    require_buffers(op, buffers)
    if buffers.codec != RAW_CODEC:
        raise BackendError(
            f"{op}: writes the {RAW_CODEC!r} codec, not {str(buffers.codec)!r}: kvcache.rotate and kvcache.store do",
            context={"op": op, "argument": "buffers"},
        )
    device, dtype, width, kv_heads = buffers.k.device, buffers.k.dtype, buffers.head_dim, buffers.num_kv_heads
    slots = _slots(op, meta, buffers)
    n_rows = slots.shape[0]
    for name, rows in (("k", k), ("v", v)):
        require_rows(op, name, rows, (n_rows, kv_heads, width), dtype, device)
    heads, q_args = _turned(op, "q", q, q_out, n_rows, width, dtype, device) if q is not None else (0, _NO_ROWS)
    positions, turn = _rotation(op, meta, rotary, device, width, n_rows)
    if n_rows == 0:
        return
    _launch(op, _lib.lib().ayk_rotate_and_cache, (
        *q_args, k.data_ptr(), *k.stride()[:2], 0, 0, 0, v.data_ptr(), *v.stride()[:2], buffers.k.data_ptr(),
        buffers.v.data_ptr(), positions, slots.data_ptr(), *turn, n_rows, heads, kv_heads, width, buffers.num_blocks,
        buffers.block_size, _LAYOUT_CODES[KVLayoutKind(buffers.layout)], _ROW_DTYPE_CODES[dtype]), device, record)


def store_latent(latent: torch.Tensor, k_rope: torch.Tensor, buffers: LatentBuffers, meta: AttentionMetadata,
                 rotary: Rotary | None = None, q: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> None:
    """Write a step's latents and key parts into a latent cache, rotating the key parts and the queries'.

    Row i of ``latent`` [N, latent_dim] and, rotated by ``meta.positions[i]``, of ``k_rope`` [N, rope_dim]
    goes to its slot; ``q`` [N, heads, rope_dim], the queries' rotary parts, is rotated in place or
    into ``q_out`` (the tail of the absorbed queries, say) in the same launch. All may be views whose
    rows are contiguous. Without ``rotary`` the key parts are stored as they are, and there is no ``q``.
    Rows of padding requests are not stored. The cache is float16, bfloat16 or float32; this backend's attention is
    over float16 and bfloat16 ones (a float32 cache can be written and its blocks moved, for attention elsewhere).
    """
    op = "kvcache.store_latent"
    tensors, absent = _given(latent, k_rope, buffers.k, q, q_out)
    key = ("store_latent", id(buffers), id(meta), id(rotary), absent, _fastpath.signature(tensors))
    _replayed(meta, key, (buffers, meta, rotary),
              lambda record: _store_latent(op, latent, k_rope, buffers, meta, rotary, q, q_out, record))


def _store_latent(op: str, latent, k_rope, buffers: LatentBuffers, meta: AttentionMetadata, rotary, q, q_out,
                  record) -> None:
    require_latent_buffers(op, buffers)
    cache, latent_dim, rope_dim = buffers.cache, buffers.latent_dim, buffers.rope_dim
    device, dtype = cache.device, cache.dtype
    slots = _slots(op, meta, buffers)
    n_rows = slots.shape[0]
    require_rows(op, "latent", latent, (n_rows, latent_dim), dtype, device)
    require_rows(op, "k_rope", k_rope, (n_rows, rope_dim), dtype, device)
    if rotary is not None and 2 * rotary.turns.numel() != rope_dim:
        raise BackendError(f"{op}: the rotation turns {2 * rotary.turns.numel()} elements, key parts have {rope_dim}",
                           context={"op": op, "argument": "rotary"})
    if rotary is None and q is not None:
        raise BackendError(f"{op}: q is given and nothing to rotate it by", context={"op": op, "argument": "q"})
    heads, q_args = _turned(op, "q", q, q_out, n_rows, rope_dim, dtype, device) if q is not None else (0, _NO_ROWS)
    positions, turn = _rotation(op, meta, rotary, device, rope_dim, n_rows)
    if n_rows == 0:
        return
    _launch(op, _lib.lib().ayk_store_latent, (
        latent.data_ptr(), latent.stride(0), k_rope.data_ptr(), k_rope.stride(0), *q_args, cache.data_ptr(), positions,
        slots.data_ptr(), *turn, n_rows, heads, latent_dim, rope_dim, buffers.num_blocks, buffers.block_size,
        _ROW_DTYPE_CODES[dtype]), device, record)


def _require_any(op: str, buffers: "KVBuffers | LatentBuffers") -> None:
    if isinstance(buffers, LatentBuffers):
        require_latent_buffers(op, buffers)
    else:
        require_buffers(op, buffers)


def _planes(buffers: "KVBuffers | LatentBuffers") -> tuple[torch.Tensor, torch.Tensor]:
    """The two caches a block op moves; a latent cache is one, given twice (and moved once)."""
    return (buffers.cache, buffers.cache) if isinstance(buffers, LatentBuffers) else (buffers.k, buffers.v)


def gather(
    buffers: KVBuffers | LatentBuffers, block_ids: torch.Tensor, out_k: torch.Tensor, out_v: torch.Tensor | None = None,
    out_scales: torch.Tensor | None = None,
) -> None:
    """Copy whole blocks out (reference ``torch/kvcache.py:83-93``); a block-scaled cache's codes
    mean nothing without their scales, which go to ``out_scales`` float32 [n, kv_heads, 2]. A latent
    cache's blocks go to ``out_k``; it has no ``out_v``."""
    op = "kvcache.gather"
    _require_any(op, buffers)
    one = isinstance(buffers, LatentBuffers)
    if one != (out_v is None):
        raise BackendError(f"{op}: out_v goes with a cache of keys and values, and a latent cache has none",
                           context={"op": op, "argument": "out_v"})
    if one:
        out_v = out_k
    device = buffers.k.device
    _ids(op, "block_ids", block_ids, device)
    shape = (block_ids.shape[0], *buffers.k.shape[1:])
    require_like(op, "out_k", out_k, shape, buffers.k.dtype)
    require_like(op, "out_v", out_v, shape, buffers.k.dtype)
    require_device(op, "out_k", out_k, device)
    require_device(op, "out_v", out_v, device)
    scales = block_scales(buffers)
    if (scales is None) != (out_scales is None):
        raise BackendError(
            f"{op}: out_scales goes with a block-scaled cache: the cache is {str(buffers.codec)!r} and out_scales "
            f"is {'not given' if out_scales is None else 'given'}",
            context={"op": op, "argument": "out_scales"},
        )
    if scales is not None:
        require_like(op, "out_scales", out_scales, (block_ids.shape[0], *scales.shape[1:]), scales.dtype)
        require_device(op, "out_scales", out_scales, device)
    if block_ids.shape[0] == 0:
        return
    _lib.check(
        op,
        _lib.lib().ayk_gather_blocks(
            *(t.data_ptr() for t in _planes(buffers)),
            out_k.data_ptr(),
            out_v.data_ptr(),
            block_ids.data_ptr(),
            int(block_ids.dtype == torch.int64),
            block_ids.shape[0],
            buffers.num_blocks,
            _block_bytes(buffers),
            _stream(device),
        ),
    )
    if scales is not None:
        _move_scales(op, "ayk_gather_blocks", (scales, scales, out_scales, out_scales), (block_ids,), scales, device)


def _move_scales(op: str, name: str, tensors: tuple[torch.Tensor, ...], ids: tuple[torch.Tensor, ...],
                 scales: torch.Tensor, device: torch.device) -> None:
    """The block op ``name`` on a block-scaled cache's scales, one block of them a row (the op
    takes two caches of one shape: both are the scales, moved once)."""
    _lib.check(
        op,
        getattr(_lib.lib(), name)(
            *(t.data_ptr() for t in tensors),
            *(i.data_ptr() for i in ids),
            int(ids[0].dtype == torch.int64),
            ids[0].shape[0],
            scales.shape[0],
            scales.shape[1] * 8,
            _stream(device),
        ),
    )


def copy_blocks(buffers: KVBuffers | LatentBuffers, src: torch.Tensor, dst: torch.Tensor) -> None:
    op = "kvcache.copy_blocks"
    _require_any(op, buffers)
    device = buffers.k.device
    _ids(op, "src", src, device)
    _ids(op, "dst", dst, device)
    if src.shape != dst.shape:
        raise BackendError(
            f"{op}: src has {src.shape[0]} blocks but dst has {dst.shape[0]}",
            context={"op": op, "argument": "dst"},
        )
    if src.shape[0] == 0:
        return
    if src.dtype != dst.dtype:
        src, dst = src.to(torch.int64), dst.to(torch.int64)
    _lib.check(
        op,
        _lib.lib().ayk_copy_blocks(
            *(t.data_ptr() for t in _planes(buffers)),
            src.data_ptr(),
            dst.data_ptr(),
            int(src.dtype == torch.int64),
            src.shape[0],
            buffers.num_blocks,
            _block_bytes(buffers),
            _stream(device),
        ),
    )
    scales = block_scales(buffers)
    if scales is not None:
        _move_scales(op, "ayk_copy_blocks", (scales, scales), (src, dst), scales, device)


def zero_blocks(buffers: KVBuffers | LatentBuffers, block_ids: torch.Tensor) -> None:
    op = "kvcache.zero_blocks"
    _require_any(op, buffers)
    device = buffers.k.device
    _ids(op, "block_ids", block_ids, device)
    if block_ids.shape[0] == 0:
        return
    _lib.check(
        op,
        _lib.lib().ayk_zero_blocks(
            *(t.data_ptr() for t in _planes(buffers)),
            block_ids.data_ptr(),
            int(block_ids.dtype == torch.int64),
            block_ids.shape[0],
            buffers.num_blocks,
            _block_bytes(buffers),
            _stream(device),
        ),
    )
    scales = block_scales(buffers)
    if scales is not None:
        _move_scales(op, "ayk_zero_blocks", (scales, scales), (block_ids,), scales, device)


def build_tables(
    rows_per_request: torch.Tensor,
    kv_lengths: torch.Tensor,
    block_table: torch.Tensor,
    pool: BlockPool,
    tables: StepTables,
    block_size: int,
) -> None:
    """Give every request of a step the blocks it lacks, and derive its rows' positions and slots.

    All on the device, from int32 device tensors: request ``b`` brings ``rows_per_request[b]`` rows,
    the last of the ``kv_lengths[b]`` tokens it has after the step, and its row of ``block_table``
    [B, W] already holds the blocks of the tokens before them. The blocks it lacks come from
    ``pool`` in request order and are written into ``block_table``; ``tables`` receives what
    ``attention.plan`` derives on the host (reference ``torch/attention.py:64-164``).

    A request that cannot be served -- negative rows, more rows than tokens, more blocks than W,
    rows past the tables' N, the padding block 0 where its last held block should be, or a pool that
    runs out at it or before it while it needs a block -- gets no block, slots and positions of 0 and
    a length of 0 in ``tables.kv_lengths``, and counts into ``pool.after[1]``; a request of length 0
    is padding and does not. Rows of the tables behind the last request's get request, position and
    slot 0. ``tables.kv_lengths`` may be ``kv_lengths`` itself. Nothing waits for the device, and the
    call can be captured.

    The slots serve ``store`` at once. To attend to the step, plan it from ``tables.kv_lengths`` and
    ``block_table`` (``attention.plan``, which reads them on the host); only a decode bucket is served
    without the host (``attention.advance_graph_metadata``).
    """
    op = "kvcache.build_tables"
    free, taken, after = pool
    request_of_row, positions, slots, lengths = tables
    requests, rows, width = kv_lengths.numel(), positions.numel(), block_table.shape[-1] if block_table.ndim else 0
    index = block_table.get_device()
    if not (index >= 0 and block_table.ndim == 2 and block_table.shape[0] == requests and block_table.dtype is _I32
            and block_table.is_contiguous() and _vector(rows_per_request, requests, _I32, index)
            and _vector(kv_lengths, requests, _I32, index) and _vector(lengths, requests, _I32, index)
            and _vector(request_of_row, rows, _I32, index) and _vector(positions, rows, _I32, index)
            and _vector(slots, rows, torch.int64, index) and _vector(free, free.numel(), _I32, index)
            and _vector(taken, 1, _I32, index) and _vector(after, 4, _I32, index)):
        _refuse_tables(op, rows_per_request, kv_lengths, block_table, pool, tables)
    _lib.check(op, _lib.lib().ayk_build_tables(
        rows_per_request.data_ptr(), kv_lengths.data_ptr(), requests, block_table.data_ptr(), width, width,
        free.data_ptr(), free.numel(), taken.data_ptr(), after.data_ptr(), block_size, request_of_row.data_ptr(),
        positions.data_ptr(), slots.data_ptr(), rows, lengths.data_ptr(), _stream(block_table.device),
    ))


def _vector(tensor: torch.Tensor, count: int, dtype: torch.dtype, index: int) -> bool:
    """Whether ``tensor`` is a contiguous vector of ``count`` elements on device ``index`` (the quick
    form of the checks below: ten tensors a call, on a kernel of a few microseconds)."""
    return (tensor.numel() == count and tensor.ndim == 1 and tensor.dtype is dtype and tensor.is_contiguous()
            and tensor.get_device() == index)


def _refuse_tables(op: str, rows_per_request: torch.Tensor, kv_lengths: torch.Tensor, block_table: torch.Tensor,
                   pool: BlockPool, tables: StepTables) -> None:
    """Say what is wrong with a call of :func:`build_tables`."""
    device = block_table.device
    if not block_table.is_cuda:
        raise BackendError(f"{op}: the hip backend runs on a HIP device; block_table is on {device}",
                           context={"op": op, "argument": "block_table"})
    requests, rows = kv_lengths.numel(), tables.positions.numel()
    width = block_table.shape[1] if block_table.ndim == 2 else 0
    require_pool(op, pool, device)
    for name, tensor, shape, dtype in (
        ("rows_per_request", rows_per_request, (requests,), torch.int32),
        ("kv_lengths", kv_lengths, (requests,), torch.int32),
        ("block_table", block_table, (requests, width), torch.int32),
        ("tables.request_of_row", tables.request_of_row, (rows,), torch.int32),
        ("tables.positions", tables.positions, (rows,), torch.int32),
        ("tables.slot_mapping", tables.slot_mapping, (rows,), torch.int64),
        ("tables.kv_lengths", tables.kv_lengths, (requests,), torch.int32),
    ):
        require_like(op, name, tensor, shape, dtype)
        if tensor.device != device:
            raise BackendError(f"{op}: {name} is on {tensor.device}, the table is on {device}",
                               context={"op": op, "argument": name})
