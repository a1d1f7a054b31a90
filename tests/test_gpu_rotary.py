"""Rotary positions and the cache writes joined to them, against the definition in 64 bits.

Bounds. The angle of a pair is exact but for the rounding of its remainder (half a step of at most pi/4)
and of its cosine and sine (series cut below 2^-25, a few half steps of 2^-24, one more for the
magnitude): 2^-21 of 1 covers them. The products and their sum add two half steps. So a result is within
(|x| + |y|) * magnitude * 2^-21, and half a step of its own type, of the true one.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, ForwardMode, KVLayoutKind
from ayaka_amd.errors import BackendError
from ayaka_amd.kvcache import RAW_CODEC, KVBuffers, LatentBuffers, fp8_e4m3_codec
from ayaka_amd.rotary import LinearScaling, Rotary, YarnScaling, rotary
from oracle import latent as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


class Step:
    """Requests of ``(rows, length)``, their table and plan."""

    def __init__(self, ops, steps, block, seed=0) -> None:
        rng = np.random.default_rng(seed)
        self.rows, self.lengths, self.block = [r for r, _ in steps], [n for _, n in steps], block
        need = [-(-n // block) for n in self.lengths]
        ids = rng.permutation(np.arange(1, 1 + sum(need)))
        self.table = np.zeros((len(steps), max(1, max(need))), dtype=np.int64)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.blocks = 2 + sum(need)
        self.positions, self.slots = oracle.positions_and_slots(self.rows, self.lengths, self.table, block)
        mode = ForwardMode.DECODE if all(r == 1 for r in self.rows) else ForwardMode.MIXED
        self.meta = ops.attention.plan(mode, torch.tensor(self.rows, device=DEV), torch.tensor(self.lengths, device=DEV),
                                       torch.tensor(self.table, device=DEV), block)


def rows_of(n, heads, width, dtype, seed, pad=0):
    """Rows whose heads may be a slice of a wider row."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, heads * width + pad, generator=g, device="cuda").to(dtype)
    return x[:, pad // 2: pad // 2 + heads * width].unflatten(1, (heads, width))


def check(got, x, positions, turn: Rotary) -> None:
    x = x.double().cpu().numpy()
    turns = turn.turns.cpu().numpy()
    want = oracle.rotate(x, positions, turns, turn.interleaved, turn.magnitude)
    pairs = len(turns)
    first = np.arange(pairs) * (2 if turn.interleaved else 1)
    second = first + (1 if turn.interleaved else pairs)
    reach = np.zeros_like(x)
    reach[..., first] = reach[..., second] = (np.abs(x[..., first]) + np.abs(x[..., second])) * abs(turn.magnitude)
    dtype = got.dtype
    bound = reach * 2.0 ** -21 + torch.finfo(dtype).eps / 2 * np.abs(want) + float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    bound[..., 2 * pairs:] = 0.0
    got = got.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) - bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,dim", [(64, 64), (128, 64), (80, 40), (96, 12), (256, 256), (6, 2), (34, 34)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotate(ops, dtype, width, dim, interleaved) -> None:
    step = Step(ops, [(1, 1), (3, 700), (1, 0), (5, 40)], 16)
    n = len(step.positions)
    q, k = rows_of(n, 5, width, TYPES[dtype], 1), rows_of(n, 2, width, TYPES[dtype], 2)
    turn = rotary(dim, interleaved=interleaved, device=DEV, scaling=YarnScaling(4.0, 512))
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    ops.kvcache.rotate(q, k, step.meta, turn, q_out, k_out)
    check(q_out, q, step.positions, turn)
    check(k_out, k, step.positions, turn)
    before = q.clone()
    ops.kvcache.rotate(q, None, step.meta, turn)  # in place
    assert torch.equal(q, q_out)
    ops.kvcache.rotate(None, before, step.meta, turn)
    assert torch.equal(before, q_out)


@pytest.mark.parametrize("pad", [16, 6, 2])
@pytest.mark.parametrize("interleaved", [False, True])
def test_views_of_wider_rows(ops, pad, interleaved) -> None:
    """Strides and addresses that take 16-, 4- and 2-byte accesses; what lies between the rows stays."""
    step = Step(ops, [(1, 9)] * 7, 4)
    whole = torch.randn(7, 4 * 64 + pad, device="cuda").to(torch.bfloat16)
    q = whole[:, pad // 2: pad // 2 + 256].unflatten(1, (4, 64))
    turn = rotary(48, interleaved=interleaved, device=DEV)
    before, x = whole.clone(), q.clone()
    out = torch.zeros(4, 7, 66 + pad, device="cuda", dtype=torch.bfloat16)  # heads outermost
    ops.kvcache.rotate(q, None, step.meta, turn, out.transpose(0, 1)[:, :, 2:66])
    assert torch.equal(whole, before)
    check(out.transpose(0, 1)[:, :, 2:66].contiguous(), x, step.positions, turn)
    assert not out[:, :, :2].any() and not out[:, :, 66:].any()
    ops.kvcache.rotate(q, None, step.meta, turn)
    check(q.contiguous(), x, step.positions, turn)
    assert torch.equal(whole[:, : pad // 2], before[:, : pad // 2]) and torch.equal(whole[:, pad // 2 + 256:], before[:, pad // 2 + 256:])


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_far_positions_keep_their_angle(ops, dtype) -> None:
    """At position 2^24 and beyond an angle in 32 bits would be off by radians."""
    far = (1 << 30) + 12345
    step = Step(ops, [(1, 5)] * 4, 8)
    step.meta.positions.copy_(torch.tensor([far, 1 << 24, 2_000_000_011, 0]))
    x = rows_of(4, 3, 128, TYPES[dtype], 3)
    turn = rotary(128, device=DEV, scaling=LinearScaling(3.0))
    out = torch.empty_like(x)
    ops.kvcache.rotate(x, None, step.meta, turn, out)
    # (the angle itself, in 64 bits, is off by 2^-53 of position * turns: 2^-24 turns at 2^30)
    check(out, x, step.meta.positions.cpu().numpy(), turn)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("heads,kv_heads,width,dim,block", [(9, 3, 64, 64, 16), (8, 8, 128, 64, 7), (4, 1, 80, 80, 1), (64, 8, 128, 128, 32)])
def test_store_rotated(ops, dtype, layout, heads, kv_heads, width, dim, block) -> None:
    """What rotate and store do, bit for bit; every other slot and the padding block as they were."""
    step = Step(ops, [(1, 1), (40, 90), (1, 0), (1, 33), (7, 7), (2, 0)], block)
    n, kind = len(step.positions), KVLayoutKind.NHD if layout == "nhd" else KVLayoutKind.HND
    whole = rows_of(n, heads + 2 * kv_heads, width, TYPES[dtype], 4)
    q, k, v = whole.split((heads, kv_heads, kv_heads), dim=1)
    turn = rotary(dim, interleaved=width == 80, device=DEV)
    shape = (step.blocks, block, kv_heads, width) if layout == "nhd" else (step.blocks, kv_heads, block, width)
    k_cache, v_cache = (torch.randn(shape, device="cuda").to(TYPES[dtype]) for _ in range(2))
    buffers = KVBuffers(k_cache, v_cache, kind, RAW_CODEC)
    want = KVBuffers(k_cache.clone(), v_cache.clone(), kind, RAW_CODEC)
    saved, k_turned, q_want, q_out = whole.clone(), torch.empty_like(k), torch.empty_like(q), torch.empty_like(q)
    ops.kvcache.rotate(q, k, step.meta, turn, q_want, k_turned)
    check(k_turned, k, step.positions, turn)
    ops.kvcache.store_rotated(q, k, v, buffers, step.meta, turn, q_out=q_out)
    assert torch.equal(q_out, q_want) and torch.equal(whole, saved)
    ops.kvcache.store(k_turned.contiguous(), v.contiguous(), want, step.meta)
    for got, ref, name in ((k_cache, want.k, "k"), (v_cache, want.v, "v")):
        assert torch.equal(got[1:].view(torch.uint8), ref[1:].view(torch.uint8)), name
    # the padding block: left alone (store writes padding rows there)
    fresh = torch.zeros_like(k_cache), torch.zeros_like(v_cache)
    ops.kvcache.store_rotated(None, k, v, KVBuffers(*fresh, kind, RAW_CODEC), step.meta, turn)
    assert not fresh[0][0].any() and not fresh[1][0].any()
    ops.kvcache.store_rotated(q, k, v, buffers, step.meta, turn)  # queries in place
    assert torch.equal(q, q_want)


def test_rows_outside_the_pool_are_dropped(ops) -> None:
    step = Step(ops, [(1, 3)] * 4, 4)
    step.meta.slot_mapping.copy_(torch.tensor([-1, 3, step.blocks * 4, 1 << 40]))  # 3: the padding block
    k, v = rows_of(4, 2, 64, torch.bfloat16, 5), rows_of(4, 2, 64, torch.bfloat16, 6)
    caches = tuple(torch.zeros(step.blocks, 4, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.kvcache.store_rotated(None, k, v, KVBuffers(*caches, KVLayoutKind.NHD, RAW_CODEC), step.meta, rotary(64, device=DEV))
    assert not caches[0].any() and not caches[1].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("latent,rope,heads,block", [(512, 64, 16, 16), (256, 64, 1, 7), (96, 32, 5, 1), (10, 6, 3, 24)])
def test_store_latent(ops, dtype, latent, rope, heads, block) -> None:
    step = Step(ops, [(1, 1), (50, 61), (1, 0), (1, 700), (3, 3)], block)
    n, t = len(step.positions), TYPES[dtype]
    down = rows_of(n, 1, latent + rope, t, 7)[:, 0]
    q = rows_of(n, heads, 128 + rope, t, 8)[:, :, 128:]
    cache = torch.randn(step.blocks, block, latent + rope, device="cuda").to(t)
    want = cache.clone()
    turn = rotary(rope, interleaved=True, device=DEV, base=500.0)
    q_out = torch.zeros(n, heads, latent + rope, device="cuda", dtype=t)
    buffers = LatentBuffers(cache, latent)
    ops.kvcache.store_latent(down[:, :latent], down[:, latent:], buffers, step.meta, turn, q, q_out[:, :, latent:])
    assert not q_out[:, :, :latent].any()
    check(q_out[:, :, latent:].contiguous(), q, step.positions, turn)
    key = torch.empty(n, 1, rope, device="cuda", dtype=t)
    ops.kvcache.rotate(None, down[:, None, latent:], step.meta, turn, k_out=key)
    check(key, down[:, None, latent:], step.positions, turn)
    live = torch.as_tensor(step.slots >= block)
    flat = want.view(-1, latent + rope)
    flat[torch.as_tensor(step.slots)[live].to(DEV)] = torch.cat((down[:, :latent], key[:, 0]), dim=1)[live.to(DEV)]
    assert torch.equal(cache, want)
    # without a rotation the key parts go in as they are
    cache.zero_()
    ops.kvcache.store_latent(down[:, :latent], down[:, latent:], buffers, step.meta)
    assert torch.equal(cache.view(-1, latent + rope)[torch.as_tensor(step.slots)[live].to(DEV)], down[live.to(DEV)])


def test_no_rows(ops) -> None:
    meta = ops.attention.plan(ForwardMode.IDLE, torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV),
                              torch.zeros(2, 1, dtype=torch.int32, device=DEV), 16)
    q = torch.zeros(0, 4, 64, device="cuda")
    ops.kvcache.rotate(q, q, meta, rotary(64, device=DEV))
    ops.kvcache.store_latent(torch.zeros(0, 512, device="cuda"), torch.zeros(0, 64, device="cuda"),
                             LatentBuffers(torch.zeros(2, 16, 576, device="cuda"), 512), meta, rotary(64, device=DEV))


def test_many_rows_one_launch(ops) -> None:
    """Enough rows that several share a workgroup, and a last workgroup that is not full."""
    step = Step(ops, [(9001, 9001)], 128)
    x = rows_of(9001, 2, 64, torch.float16, 9)
    turn = rotary(64, device=DEV)
    out = torch.empty_like(x)
    ops.kvcache.rotate(x, None, step.meta, turn, out)
    check(out, x, step.positions, turn)


def test_repeated_calls_and_replaced_tensors(ops) -> None:
    """The recorded launch serves the same tensors only."""
    step = Step(ops, [(1, 50)] * 3, 16)
    turn, other = rotary(64, device=DEV), rotary(64, device=DEV, base=77.0)
    x = rows_of(3, 2, 64, torch.bfloat16, 10)
    out = torch.empty_like(x)
    for t in (turn, turn, other, turn):
        ops.kvcache.rotate(x, None, step.meta, t, out)
        check(out, x, step.positions, t)
    x.copy_(rows_of(3, 2, 64, torch.bfloat16, 11))
    ops.kvcache.rotate(x, None, step.meta, turn, out)
    check(out, x, step.positions, turn)
    again = torch.empty_like(x)
    ops.kvcache.rotate(x, None, step.meta, turn, again)
    assert torch.equal(again, out)


def test_captured(ops) -> None:
    """Replayed on other positions and rows, with eager calls between."""
    step = Step(ops, [(1, 30), (1, 50)], 16)
    turn = rotary(64, device=DEV)
    down, q = rows_of(2, 1, 576, torch.bfloat16, 12)[:, 0], rows_of(2, 4, 64, torch.bfloat16, 13)
    q_out = torch.empty_like(q)
    buffers = LatentBuffers(torch.zeros(step.blocks, 16, 576, dtype=torch.bfloat16, device="cuda"), 512)

    def call():
        ops.kvcache.store_latent(down[:, :512], down[:, 512:], buffers, step.meta, turn, q, q_out)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        step.meta.positions.copy_(torch.tensor([3 + i, 40 * i], device=DEV))
        q.copy_(rows_of(2, 4, 64, torch.bfloat16, 20 + i))
        q_out.zero_()
        buffers.cache.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = q_out.clone(), buffers.cache.clone()
        check(q_out, q, step.meta.positions.cpu().numpy(), turn)
        call()
        assert torch.equal(got[0], q_out) and torch.equal(got[1], buffers.cache)


def test_refusals(ops) -> None:
    step = Step(ops, [(1, 5)] * 2, 16)
    turn = rotary(64, device=DEV)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    caches = tuple(torch.zeros(step.blocks, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv = KVBuffers(*caches, KVLayoutKind.NHD, RAW_CODEC)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    rot, put = ops.kvcache.rotate, ops.kvcache.store_rotated
    fp8 = KVBuffers(*(c.to(torch.float8_e4m3fn) for c in caches), KVLayoutKind.NHD, fp8_e4m3_codec())
    cases = [
        (lambda: rot(q[:1], None, step.meta, turn), "q must be bfloat16"),
        (lambda: rot(q, k.half(), step.meta, turn), "k must be bfloat16"),
        (lambda: rot(q, None, step.meta, rotary(66, device=DEV)), "turns 66 elements of heads of 64"),
        (lambda: rot(q, None, step.meta, rotary(64, device="cpu")), "rotary.turns is on cpu"),
        (lambda: rot(q, None, step.meta, turn._replace(turns=turn.turns.float())), "float64"),
        (lambda: rot(q, None, step.meta, turn, q[:, :, :32]), "q_out must be"),
        (lambda: rot(q, None, step.meta, turn, torch.zeros(2, 1, 64, dtype=q.dtype, device="cuda").expand(2, 4, 64)), "share memory"),
        (lambda: rot(q, None, step.meta, turn, q.view(-1).as_strided((2, 4, 64), (64, 128, 1))), "at other strides"),
        (lambda: rot(torch.zeros(2, 4, 63, device="cuda"), None, step.meta, rotary(62, device=DEV)), "not even"),
        (lambda: put(q, k, k, fp8, step.meta, turn), "kvcache.rotate and kvcache.store do"),
        (lambda: put(q, k[:, :1], k, kv, step.meta, turn), "k must be bfloat16"),
        (lambda: put(q.float(), k, k, kv, step.meta, turn), "q must be bfloat16"),
        (lambda: put(q, k, k, KVBuffers(*(c.view(step.blocks * 2, 8, 2, 64) for c in caches), KVLayoutKind.NHD, RAW_CODEC), step.meta, turn), "planned for blocks of 16"),
    ]
    latent = LatentBuffers(torch.zeros(step.blocks, 16, 576, dtype=torch.bfloat16, device="cuda"), 512)
    x = torch.zeros(2, 576, dtype=torch.bfloat16, device="cuda")
    cases += [
        (lambda: ops.kvcache.store_latent(x[:, :512], x[:, 512:], latent, step.meta, rotary(32, device=DEV)), "turns 32 elements, key parts have 64"),
        (lambda: ops.kvcache.store_latent(x[:, :512], x[:, 512:], latent, step.meta, None, q), "nothing to rotate it by"),
        (lambda: ops.kvcache.store_latent(x[:, :500], x[:, 512:], latent, step.meta), "latent must be"),
        (lambda: ops.kvcache.store_latent(x[:, :512], x[:, 512:], latent._replace(latent_dim=576), step.meta), "rope_dim above 0"),
        (lambda: ops.kvcache.gather(latent, torch.zeros(1, dtype=torch.int64, device=DEV), latent.cache[:1].clone(), latent.cache[:1].clone()), "a latent cache has none"),
        (lambda: ops.kvcache.gather(kv, torch.zeros(1, dtype=torch.int64, device=DEV), caches[0][:1].clone()), "out_v goes with"),
    ]
    for call, message in cases:
        with pytest.raises(BackendError, match=message):
            call()


def test_block_moves_of_latent_caches(ops) -> None:
    g = torch.Generator(device="cuda").manual_seed(1)
    for dtype, width in ((torch.bfloat16, 576), (torch.float16, 102), (torch.float32, 33)):
        cache = torch.randn(9, 7, width, generator=g, device="cuda").to(dtype)
        buffers, want = LatentBuffers(cache, width - 2), cache.clone()
        ids = torch.tensor([4, 0, 8], device=DEV)
        out = torch.empty(3, 7, width, dtype=dtype, device="cuda")
        ops.kvcache.gather(buffers, ids, out)
        assert torch.equal(out, want[ids])
        ops.kvcache.copy_blocks(buffers, ids.int(), torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV))
        want[1:4] = want[ids]
        assert torch.equal(cache, want)
        ops.kvcache.zero_blocks(buffers, torch.tensor([5, 7], device=DEV))
        want[5] = want[7] = 0
        assert torch.equal(cache, want)
