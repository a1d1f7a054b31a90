"""The paged KV-cache layout and the contract a backend implements to write it.

Restates the reference's layout definition (``python/ayaka/ops/kvcache.py:1-38``):

* ``k`` and ``v`` are separate contiguous tensors of one dtype, shaped
  ``[num_blocks, block_size, kv_heads, head_dim]`` (NHD) or
  ``[num_blocks, kv_heads, block_size, head_dim]`` (HND).
* Position ``pos`` of a request lives in ``slot = table[pos // block_size] *
  block_size + pos % block_size``. A request of ``length`` tokens uses the first
  ``ceil(length / block_size)`` entries of its table.
* Block 0 is the padding block: never assigned to a request; padding rows are
  stored into slot 0 and its contents are never read as context.
* ``codec`` names how values are stored. The reference defines ``"raw"`` only
  (values in the compute dtype). This package adds ``"fp8_e4m3"``: the
  tensors are ``torch.float8_e4m3fn``, one byte per element, holding what
  torch's cast to that type gives (round to nearest even; a magnitude that
  rounds above 448 becomes NaN); readers decode it exactly to the compute dtype.
  A layer may carry a key and a value scale (:func:`fp8_e4m3_codec`): the codes
  are then those of ``x / scale`` and readers multiply by the scale. It also adds
  ``"fp8_e4m3_block"`` (:func:`fp8_e4m3_block_codec`): the same codes under a key
  scale and a value scale for every block and key/value head, which the KV write
  settles from the values themselves, so nothing is calibrated and no finite value
  becomes NaN.
* A latent cache (:class:`LatentBuffers`, layout ``NLD``) is one tensor ``[num_blocks, block_size,
  latent_dim + rope_dim]`` in the compute dtype: a token's latent vector and, behind it, its rotated
  key part, shared by all heads. Slots, tables and the padding block are the same.

Importing this module does not import torch.
"""

from __future__ import annotations

from typing import TYPE_CHECKING, NamedTuple, Protocol

from ayaka_amd.enums import KVLayoutKind

if TYPE_CHECKING:
    from torch import Tensor

    from ayaka_amd.attention import AttentionMetadata
    from ayaka_amd.rotary import Rotary

__all__ = [
    "FP8_E4M3_BLOCK_CODEC",
    "FP8_E4M3_CODEC",
    "RAW_CODEC",
    "BlockPool",
    "BlockScaledFp8Codec",
    "KVBuffers",
    "KVCacheOps",
    "LatentBuffers",
    "LatentWeights",
    "ScaledFp8Codec",
    "StepTables",
    "codec_scales",
    "fp8_e4m3_block_codec",
    "fp8_e4m3_codec",
]

RAW_CODEC = "raw"
#: Keys and values as OCP fp8 e4m3 codes (``torch.float8_e4m3fn``), no scale.
FP8_E4M3_CODEC = "fp8_e4m3"
#: The same codes with a key and a value scale for every block and key/value head.
FP8_E4M3_BLOCK_CODEC = "fp8_e4m3_block"


class ScaledFp8Codec(str):
    """The ``"fp8_e4m3"`` codec of one layer with a key scale and a value scale.

    It is the string ``"fp8_e4m3"`` (equal to :data:`FP8_E4M3_CODEC`, so code that compares
    codecs keeps working) carrying ``k_scale`` and ``v_scale``: the cache holds the codes of
    ``k * (1 / k_scale)`` and ``v * (1 / v_scale)`` (the inverse rounded once to float32, the
    product once to float32, then encoded), and readers decode ``code * scale``. A layer whose
    keys reach 4,000 stores them finite with ``k_scale = 4000 / 448``. Scales of 1 are the
    unscaled codec, bit for bit. Make one with :func:`fp8_e4m3_codec`.
    """

    k_scale: float
    v_scale: float

    def __new__(cls, k_scale: float = 1.0, v_scale: float = 1.0) -> "ScaledFp8Codec":
        import math
        import struct

        scales = []
        for name, value in (("k_scale", k_scale), ("v_scale", v_scale)):
            value = struct.unpack("f", struct.pack("f", float(value)))[0]  # as the library reads it
            if not (math.isfinite(value) and value > 0.0):
                raise ValueError(f"{name} must be a positive finite float32, got {value!r}")
            scales.append(value)
        codec = super().__new__(cls, FP8_E4M3_CODEC)
        codec.k_scale, codec.v_scale = scales
        return codec

    def __repr__(self) -> str:
        return f"fp8_e4m3_codec(k_scale={self.k_scale!r}, v_scale={self.v_scale!r})"

    def __reduce__(self):
        return (ScaledFp8Codec, (self.k_scale, self.v_scale))


def fp8_e4m3_codec(k_scale: float = 1.0, v_scale: float = 1.0) -> ScaledFp8Codec:
    """The ``"fp8_e4m3"`` codec with a layer's key and value scales (see :class:`ScaledFp8Codec`)."""
    return ScaledFp8Codec(k_scale, v_scale)


class BlockScaledFp8Codec(str):
    """The ``"fp8_e4m3_block"`` codec of one layer, carrying the scales of its cache.

    It is the string ``"fp8_e4m3_block"`` (equal to :data:`FP8_E4M3_BLOCK_CODEC`) with
    ``scales``, a contiguous float32 ``[num_blocks, kv_heads, 2]`` tensor on the cache's device:
    the key scale and the value scale of every block and key/value head. An element is worth
    ``code * scale``. Scales are powers of two 2^e with -40 <= e <= 80, or 0 for a block of nothing
    but zeros; a fresh cache starts with zeros. ``store`` settles them as it writes: the first call
    that writes a block from its first token on takes the least scale that keeps its largest finite
    magnitude there within 448 codes, and a later call the larger of what it needs in the same way
    and the block's scale. Growth re-encodes the block's tokens (a power of two apart, so exactly,
    down to the codes' subnormals). A scale never falls while tokens are added, also where the loud
    one was a rejected draft that the next call overwrites.

    Attention resolves what blocks far quieter than the loudest add to an output element to 2^-25 of
    the largest scaled weight (the C header has the rule).

    Storing infinities and NaN gives the NaN code and leaves the scale to the finite values.
    A layer's copy, swap and clear move the scales with the blocks (``copy_blocks``,
    ``gather(..., out_scales=)``, ``zero_blocks``).
    """

    __slots__ = ("_scales",)

    def __new__(cls, scales: "Tensor") -> "BlockScaledFp8Codec":
        import torch

        if scales.dtype != torch.float32 or scales.ndim != 3 or scales.shape[2] != 2 or not scales.is_contiguous():
            raise ValueError(
                "scales must be a contiguous float32 [num_blocks, kv_heads, 2] tensor, got "
                f"{str(scales.dtype).removeprefix('torch.')} {list(scales.shape)}"
            )
        codec = super().__new__(cls, FP8_E4M3_BLOCK_CODEC)
        codec._scales = scales
        return codec

    @property
    def scales(self) -> "Tensor":
        return self._scales

    def __repr__(self) -> str:
        return f"fp8_e4m3_block_codec(scales={list(self._scales.shape)} on {self._scales.device})"

    def __reduce__(self):
        return (BlockScaledFp8Codec, (self._scales,))


def fp8_e4m3_block_codec(scales: "Tensor") -> BlockScaledFp8Codec:
    """The ``"fp8_e4m3_block"`` codec of a layer whose blocks have these scales (see
    :class:`BlockScaledFp8Codec`); ``torch.zeros(num_blocks, kv_heads, 2)`` on the cache's device
    for a fresh cache."""
    return BlockScaledFp8Codec(scales)


def codec_scales(codec: str) -> tuple[float, float]:
    """``(k_scale, v_scale)`` of a codec: its own for a :class:`ScaledFp8Codec`, else (1, 1) (a
    :class:`BlockScaledFp8Codec` has none for the whole layer)."""
    return (getattr(codec, "k_scale", 1.0), getattr(codec, "v_scale", 1.0))


class _KVBuffers(NamedTuple):
    """The key and value tensors of one layer (reference ``ops/kvcache.py:58-91``)."""

    k: Tensor
    v: Tensor
    layout: KVLayoutKind
    codec: str

    @property
    def num_blocks(self) -> int:
        return int(self.k.shape[0])

    @property
    def block_size(self) -> int:
        return int(self.k.shape[1 if self.layout == KVLayoutKind.NHD else 2])

    @property
    def num_kv_heads(self) -> int:
        return int(self.k.shape[2 if self.layout == KVLayoutKind.NHD else 1])

    @property
    def head_dim(self) -> int:
        return int(self.k.shape[3])


try:  # pragma: no cover - only where the engine is installed
    from ayaka.ops.kvcache import KVBuffers  # type: ignore[import-not-found]
except ImportError:
    KVBuffers = _KVBuffers  # type: ignore[misc]


class LatentBuffers(NamedTuple):
    """The latent cache of one layer: ``cache`` contiguous ``[num_blocks, block_size, latent_dim +
    rope_dim]`` in the compute dtype, the latent first. (The hip backend attends to float16 and bfloat16 ones; it writes
    and moves float32 ones too.)"""

    cache: Tensor
    latent_dim: int

    @property
    def k(self) -> Tensor:
        """What scores are taken with: the whole rows."""
        return self.cache

    @property
    def v(self) -> Tensor:
        """What outputs are sums of: the latents, a view."""
        return self.cache[..., : self.latent_dim]

    @property
    def layout(self) -> KVLayoutKind:
        return KVLayoutKind.NLD

    @property
    def codec(self) -> str:
        return RAW_CODEC

    @property
    def num_blocks(self) -> int:
        return int(self.cache.shape[0])

    @property
    def block_size(self) -> int:
        return int(self.cache.shape[1])

    @property
    def rope_dim(self) -> int:
        return int(self.cache.shape[2]) - self.latent_dim


class LatentWeights(NamedTuple):
    """What expands a layer's latents into keys and values: head ``h``'s key (without its rotary part)
    is ``keys[h] @ latent``, its value ``values[h] @ latent``; ``keys`` contiguous ``[heads, nope_dim,
    latent_dim]``, ``values`` ``[heads, value_dim, latent_dim]``, in the compute dtype."""

    keys: Tensor
    values: Tensor


class BlockPool(NamedTuple):
    """The free blocks a step's requests draw from, in device memory.

    ``free`` int32 [F] lists block ids in the order they are handed out, ``taken`` int32 [1] how
    many of them are. A step that draws blocks writes ``after`` int32 [4]: how many are taken after
    it, and how many requests it could not serve; the other two words are the ops' own. ``after`` is
    zeros before its first use. :meth:`in_place` makes a pool that advances itself (``taken`` is
    ``after``'s first word), as a decode loop on the device needs; with a ``taken`` of its own the
    caller moves the count on. The host returns blocks by rewriting ``free`` and ``taken`` between
    steps. Steps that overlap in time need an ``after`` each.
    """

    free: Tensor
    taken: Tensor
    after: Tensor

    @classmethod
    def in_place(cls, free: Tensor) -> "BlockPool":
        """A pool of which nothing is taken yet and whose count advances with every step."""
        after = free.new_zeros(4)
        return cls(free, after[:1], after)


class StepTables(NamedTuple):
    """What a step's cache writes and attention read of its requests, at fixed addresses in device
    memory: ``request_of_row``, ``positions`` (int32) and ``slot_mapping`` (int64), each [N], and
    ``kv_lengths`` int32 [B] (see :class:`~ayaka_amd.attention.AttentionMetadata`).

    ``store`` writes by the slots as they are. ``attend`` takes its launch and tile lists from a plan:
    ``attention.plan`` on ``kv_lengths`` and the block table, which reads both on the host."""

    request_of_row: Tensor
    positions: Tensor
    slot_mapping: Tensor
    kv_lengths: Tensor


class KVCacheOps(Protocol):
    """Writing, reading and clearing the paged cache (reference ``ops/kvcache.py:94-144``)."""

    def layout(self) -> KVLayoutKind: ...

    def store(self, k: Tensor, v: Tensor, buffers: KVBuffers, meta: AttentionMetadata) -> None: ...

    def rotate(
        self, q: Tensor | None, k: Tensor | None, meta: AttentionMetadata, rotary: Rotary,
        q_out: Tensor | None = None, k_out: Tensor | None = None,
    ) -> None: ...

    def store_rotated(
        self, q: Tensor | None, k: Tensor, v: Tensor, buffers: KVBuffers, meta: AttentionMetadata,
        rotary: Rotary, q_out: Tensor | None = None,
    ) -> None: ...

    def store_latent(
        self, latent: Tensor, k_rope: Tensor, buffers: LatentBuffers, meta: AttentionMetadata,
        rotary: Rotary | None = None, q: Tensor | None = None, q_out: Tensor | None = None,
    ) -> None: ...

    def gather(
        self, buffers: KVBuffers | LatentBuffers, block_ids: Tensor, out_k: Tensor, out_v: Tensor | None = None,
        out_scales: Tensor | None = None,
    ) -> None: ...

    def copy_blocks(self, buffers: KVBuffers | LatentBuffers, src: Tensor, dst: Tensor) -> None: ...

    def zero_blocks(self, buffers: KVBuffers | LatentBuffers, block_ids: Tensor) -> None: ...

    def build_tables(
        self, rows_per_request: Tensor, kv_lengths: Tensor, block_table: Tensor, pool: BlockPool,
        tables: StepTables, block_size: int,
    ) -> None: ...
