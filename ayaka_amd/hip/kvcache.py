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
(``ayk_build_tables``).
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
    require_buffers,
    require_device,
    require_index_tensor,
    require_like,
    require_pool,
    stream_handle,
)
from ayaka_amd.kvcache import FP8_E4M3_CODEC, BlockPool, KVBuffers, StepTables, codec_scales

__all__ = ["build_tables", "copy_blocks", "gather", "layout", "store", "zero_blocks"]

_LAYOUT_CODES = {KVLayoutKind.NHD: 0, KVLayoutKind.HND: 1}
_DTYPE_CODES = {torch.float16: 0, torch.bfloat16: 1}
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


def gather(
    buffers: KVBuffers, block_ids: torch.Tensor, out_k: torch.Tensor, out_v: torch.Tensor,
    out_scales: torch.Tensor | None = None,
) -> None:
    """Copy whole blocks out (reference ``torch/kvcache.py:83-93``); a block-scaled cache's codes
    mean nothing without their scales, which go to ``out_scales`` float32 [n, kv_heads, 2]."""
    op = "kvcache.gather"
    require_buffers(op, buffers)
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
            buffers.k.data_ptr(),
            buffers.v.data_ptr(),
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
    takes two caches of one shape: both are the scales, so each word is written twice alike)."""
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


def copy_blocks(buffers: KVBuffers, src: torch.Tensor, dst: torch.Tensor) -> None:
    op = "kvcache.copy_blocks"
    require_buffers(op, buffers)
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
            buffers.k.data_ptr(),
            buffers.v.data_ptr(),
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


def zero_blocks(buffers: KVBuffers, block_ids: torch.Tensor) -> None:
    op = "kvcache.zero_blocks"
    require_buffers(op, buffers)
    device = buffers.k.device
    _ids(op, "block_ids", block_ids, device)
    if block_ids.shape[0] == 0:
        return
    _lib.check(
        op,
        _lib.lib().ayk_zero_blocks(
            buffers.k.data_ptr(),
            buffers.v.data_ptr(),
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
