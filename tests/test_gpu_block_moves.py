"""Block moves over caches, outputs and scales at any address their elements may have."""

from __future__ import annotations

import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, KVLayoutKind
from ayaka_amd.kvcache import KVBuffers, fp8_e4m3_block_codec

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


def moved(t: torch.Tensor, bytes_in: int) -> tuple[torch.Tensor, torch.Tensor]:
    """``t`` again, ``bytes_in`` bytes into a storage of its own, and that storage as bytes."""
    size = t.numel() * t.element_size()
    flat = torch.full((size + 64,), 0x55, dtype=torch.uint8, device=t.device)
    part = flat[bytes_in:bytes_in + size]
    part.copy_(t.contiguous().view(torch.uint8).flatten())
    return part.view(t.dtype).view(t.shape), flat


@pytest.mark.parametrize("kv_heads", [1, 2, 4])
def test_block_moves_at_any_address(ops, kv_heads) -> None:
    # caches, scales and outputs that begin where their elements may, not where the widest vector may;
    # what lies around them stays
    g = torch.Generator(device="cuda").manual_seed(kv_heads)
    blocks, block, dim = 9, 4, 64
    k, v = (torch.randint(0, 256, (blocks, block, kv_heads, dim), generator=g, device="cuda", dtype=torch.uint8)
            for _ in range(2))
    scales = torch.exp2(torch.randint(-9, 9, (blocks, kv_heads, 2), generator=g, device="cuda").float())
    ids = torch.tensor([7, 3, 5], device="cuda")
    src, dst = torch.tensor([2, 5], device="cuda"), torch.tensor([8, 1], device="cuda")
    for cache_at, scales_at, out_at in ((0, 8, 4), (8, 24, 8), (4, 8, 12), (2, 16, 20), (1, 8, 4)):
        (k2, _), (v2, _) = moved(k, cache_at), moved(v, cache_at)
        s2, s_flat = moved(scales, scales_at)
        buffers = KVBuffers(k2.view(torch.float8_e4m3fn), v2.view(torch.float8_e4m3fn), KVLayoutKind.NHD,
                            fp8_e4m3_block_codec(s2))
        (ok, ok_flat), (ov, _) = (moved(torch.zeros_like(k[:3]), cache_at + 16) for _ in range(2))
        os, os_flat = moved(torch.zeros_like(scales[:3]), out_at)
        ops.kvcache.gather(buffers, ids, ok.view(torch.float8_e4m3fn), ov.view(torch.float8_e4m3fn), os)
        assert torch.equal(ok, k[ids]) and torch.equal(ov, v[ids]) and torch.equal(os, scales[ids])
        for flat, at, size in ((os_flat, out_at, os.numel() * 4), (ok_flat, cache_at + 16, ok.numel())):
            assert (flat[:at] == 0x55).all() and (flat[at + size:] == 0x55).all()
        ops.kvcache.copy_blocks(buffers, src, dst)
        ops.kvcache.zero_blocks(buffers, ids[:1])
        for got, was in ((k2, k), (v2, v), (s2, scales)):
            want = was.clone()
            want[dst] = was[src]
            want[ids[:1]] = 0
            assert torch.equal(got, want)
        assert (s_flat[:scales_at] == 0x55).all() and (s_flat[scales_at + scales.numel() * 4:] == 0x55).all()
