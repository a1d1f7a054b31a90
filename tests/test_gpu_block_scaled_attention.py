"""Attention over block-scaled caches against float64, at tolerances derived from the arithmetic.

A row and head with true weights w_t over its visible positions and values v_t (decoded) has the
output y = sum w_t v_t. What the kernels compute is off by at most

    A * (2^-11 + 2 d) + Z + |y| * eps / 2,      A = sum w_t |v_t|

elementwise. Each weight, times its value scale and in units of the largest of them, enters P.V
rounded to fp16: half a step, 2^-11 of itself, or below 2^-14, where fp16 holds subnormals, by at
most 2^-25 and at most itself (Z, the sum of those times |code|). It carries the relative error d
of its exponential, in the numerator and in the sum. The output is rounded once to its type (half a
step, eps / 2, and half the smallest subnormal). d: the score is a sum of head_dim products in
fp32, whatever the order within (D + 8) 2^-24 of S = max_t scale sum |q||k|, in units of e; the
exponent's shift by its value scale and the maximum's subtraction round values of up to S + 128
once each; exp2, the value and weight sums over L positions and the merges add (L + 16) 2^-24.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, ForwardMode, KVLayoutKind
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import attention as hip_attention
from ayaka_amd.kvcache import KVBuffers, fp8_e4m3_block_codec
from oracle import block_scaled
from oracle.numerics import bits_to_f32, e4m3_to_f32, f32_to_bits, f32_to_e4m3

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}
LAYOUTS = {"nhd": KVLayoutKind.NHD, "hnd": KVLayoutKind.HND}
NAN = 0x7F


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


class Step:
    """A planned step over a block-scaled cache of random codes and scales.

    Every slot that no context holds is a NaN code and every other block's scales are NaN, so a
    read outside the contexts shows. ``steps`` is ``[(rows, length), ...]``; blocks of one request
    have key scales within 2^3 of each other and value scales within 2^``spread``.
    """

    def __init__(self, steps, *, dtype="bf16", layout="nhd", heads=4, kv_heads=2, head_dim=64, block=16, mode="mixed",
                 spread=12, seed=0) -> None:
        rng = np.random.default_rng(seed)
        self.dtype, self.layout, self.kv_heads, self.block = dtype, layout, kv_heads, block
        self.rows, self.lengths = [r for r, _ in steps], [n for _, n in steps]
        need = [-(-n // block) for n in self.lengths]
        blocks = 1 + sum(need) + 2
        free = list(1 + rng.permutation(blocks - 2))
        self.table = np.zeros((len(steps), max(max(need), 1) + 1), dtype=np.int64)
        # codes of magnitude up to 448 with most of their weight well below
        codes = [f32_to_e4m3(np.clip(rng.standard_normal((blocks, block, kv_heads, head_dim)) * 90, -448, 448)
                             .astype(np.float32)) for _ in range(2)]
        scales = np.full((blocks, kv_heads, 2), np.nan)
        held = np.zeros((blocks, block), bool)
        for b, n in enumerate(need):
            ids = [int(free.pop()) for _ in range(n)]
            self.table[b, :n] = ids
            scales[ids, :, 0] = np.exp2(rng.integers(-8, -5, (n, kv_heads)))
            scales[ids, :, 1] = np.exp2(rng.integers(-spread, spread + 1, (n, kv_heads)))
            for i, block_id in enumerate(ids):
                held[block_id, : min(block, self.lengths[b] - i * block)] = True
        for c in codes:
            c[~held] = NAN
        self.codes, self.scales = codes, scales
        self.q_bits = f32_to_bits(rng.standard_normal((sum(self.rows), heads, head_dim)).astype(np.float32), dtype)
        self.scale = head_dim ** -0.5
        self.mode = ForwardMode.DECODE if mode == "decode" else ForwardMode.MIXED

    def device(self, ops):
        """(q, buffers, metadata, out) on the device; out poisoned."""
        def cache(codes):
            x = codes if self.layout == "nhd" else np.ascontiguousarray(codes.transpose(0, 2, 1, 3))
            return torch.from_numpy(x).to(DEV).view(torch.float8_e4m3fn)

        scales = torch.from_numpy(self.scales.astype(np.float32)).to(DEV)
        buffers = KVBuffers(cache(self.codes[0]), cache(self.codes[1]), LAYOUTS[self.layout],
                            fp8_e4m3_block_codec(scales))
        meta = ops.attention.plan(self.mode, torch.tensor(self.rows, device=DEV), torch.tensor(self.lengths, device=DEV),
                                  torch.from_numpy(self.table).to(DEV), self.block)
        q = torch.from_numpy(self.q_bits.view(np.int16)).view(TORCH[self.dtype]).to(DEV)
        return q, buffers, meta, torch.full_like(q, float("nan"))

    def reference(self) -> tuple[np.ndarray, np.ndarray]:
        """(y, tolerance) of every row and head, float64."""
        q = bits_to_f32(self.q_bits, self.dtype).astype(np.float64)
        n, heads, dim = q.shape
        group = heads // self.kv_heads
        y, tol = np.zeros_like(q), np.zeros_like(q)
        k_all, v_all = (e4m3_to_f32(c).astype(np.float64) * self.scales[:, None, :, which, None]
                        for which, c in enumerate(self.codes))
        at = 0
        for b, (count, length) in enumerate(zip(self.rows, self.lengths)):
            ids = self.table[b, : -(-length // self.block)]
            k, v = (x[ids].reshape(-1, self.kv_heads, dim)[:length] for x in (k_all, v_all))
            for j in range(count):
                end = length - count + j + 1 if length else 0
                if end:
                    for h in range(heads):
                        kk, vv = k[:end, h // group], v[:end, h // group]
                        s = self.scale * (kk @ q[at + j, h])
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        size = abs(self.scale) * (np.abs(kk) @ np.abs(q[at + j, h])).max()
                        d = ((dim + 8) * size + 2 * (size + 128) + end + 16) * 2.0 ** -24
                        y[at + j, h] = w @ vv
                        vs = self.scales[ids, h // group, 1].repeat(self.block)[:end]
                        unit = (w * vs).max()
                        u = w * vs / unit
                        small = np.where(u < 2.0 ** -14, np.minimum(u, 2.0 ** -25), 0.0) * unit / vs
                        tol[at + j, h] = np.abs(vv).T @ (w * (2.0 ** -11 + 2 * d) + small)
            at += count
        eps, tiny = {"bf16": (2.0 ** -7, 2.0 ** -133), "fp16": (2.0 ** -10, 2.0 ** -24)}[self.dtype]
        return y, tol + np.abs(y) * eps / 2 + tiny / 2

    def check(self, out: torch.Tensor, label: str = "") -> None:
        y, tol = self.reference()
        got = out.float().cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(y)), f"{label}: NaN where the oracle has none, or the reverse"
        # a value whose magnitude is past the type's largest by half a step rounds to infinity
        most = {"bf16": np.inf, "fp16": 65520.0}[self.dtype]
        past = ~np.isnan(y) & np.isinf(got)
        assert (np.abs(y)[past] + tol[past] >= most).all() and (np.sign(got) == np.sign(y))[past].all(), label
        assert not (np.abs(y)[~past] - tol[~past] > most).any(), f"{label}: finite where the type holds no such value"
        fine = ~np.isnan(y) & ~past
        over = np.abs(got - y)[fine] - tol[fine]
        worst = over.max(initial=-np.inf)
        assert worst <= 0.0, (
            f"{label}: {np.abs(got - y)[fine].max()} off, {(over > 0).sum()} of {over.size} past their tolerance, "
            f"the worst by {worst} at tolerance {tol[fine][over.argmax()]}")


def run(ops, step: Step, label: str = "", **launch) -> torch.Tensor:
    q, buffers, meta, out = step.device(ops)
    if launch:
        hip_attention.attend_with(q, buffers, meta, out, scale=step.scale, **{"partitions": None, **launch})
    else:
        ops.attention.attend(q, buffers, meta, out, scale=step.scale)
    torch.cuda.synchronize()
    step.check(out, f"{label} {launch}")
    return out


DECODE = [(1, 1), (1, 16), (1, 17), (1, 0), (1, 250), (1, 700)]
HEADS = [(1, 1), (6, 2), (5, 1), (12, 3), (16, 2), (32, 2)]  # groups of 1, 3, 5, 4, 8 and 16


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_decode(ops, heads, kv_heads, head_dim, dtype, layout) -> None:
    step = Step(DECODE, dtype=dtype, layout=layout, heads=heads, kv_heads=kv_heads, head_dim=head_dim, mode="decode",
                seed=heads + head_dim)
    run(ops, step)
    for waves in (1, 2, 4, 8):
        run(ops, step, partitions=0, waves=waves)
    for size, merge in ((64, "in-kernel"), (64, "reduce-kernel"), (320, None)):
        run(ops, step, partitions=-(-701 // size), partition_size=size, merge=merge)


@pytest.mark.parametrize("block", [1, 3, 7, 16, 24, 64, 100])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_block_sizes(ops, block, head_dim) -> None:
    for layout in ("nhd", "hnd"):
        run(ops, Step([(1, 613), (1, 40), (1, 0), (1, 99)], layout=layout, head_dim=head_dim, block=block, heads=8,
                      mode="decode", seed=block), label=layout)
        run(ops, Step([(3, 613), (2, 40), (1, 0), (4, 99)], layout=layout, head_dim=head_dim, block=block, heads=8,
                      seed=block), label=layout)
        run(ops, Step([(70, 613), (1, 40), (2, 0), (99, 99)], layout=layout, head_dim=head_dim, block=block, heads=8,
                      seed=block), label=layout)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_windows(ops, heads, kv_heads, head_dim, dtype) -> None:
    most = max(1, 16 // (heads // kv_heads))
    steps = [(min(4, most), 300), (1, 1), (min(2, most), 2), (min(3, most), 0), (most, 517), (1, 64)]
    step = Step(steps, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim, seed=head_dim + heads)
    for size in (0, 64, 256):
        run(ops, step, prefill=True, window=True, partitions=0 if size == 0 else None, partition_size=size or None)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_multi_row(ops, heads, kv_heads, head_dim, dtype) -> None:
    step = Step([(65, 200), (1, 33), (7, 7), (3, 0), (40, 129)], dtype=dtype, layout="hnd", heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, seed=head_dim + heads)
    run(ops, step)
    full = hip_attention.PREFILL_PAIRS[head_dim]
    for pairs in ((2 * full,) if head_dim != 64 else ()) + (full, full // 2, full // 4):
        if heads // kv_heads <= pairs:
            run(ops, step, prefill=True, window=False, tile_pairs=pairs, partitions=0)
            run(ops, step, prefill=True, window=False, tile_pairs=pairs, partition_size=64)


@pytest.mark.parametrize("steps,mode", [([(1, 9000), (1, 2)], "decode"), ([(3, 9000), (2, 2)], "mixed"),
                                        ([(40, 9000)], "mixed")])
def test_contexts_of_many_table_segments(ops, steps, mode) -> None:
    # blocks of one position: a table segment holds 512 of them
    run(ops, Step(steps, block=1, heads=8, head_dim=128, mode=mode, seed=3))


@pytest.mark.parametrize("mode,steps", [("decode", [(1, 300)]), ("mixed", [(4, 300)]), ("mixed", [(33, 300)])])
def test_value_scales_far_apart(ops, mode, steps) -> None:
    # values from 2^-40 to 2^80 times their codes side by side: the sum of the weights neither
    # overflows nor loses the positions whose values are small (bf16 holds all of it)
    step = Step(steps, heads=8, head_dim=128, mode=mode, seed=11)
    rng = np.random.default_rng(0)
    for ids, exponents in ((step.table[0, :19], rng.integers(-40, 81, (19, 2))), (step.table[0, :19], None)):
        if exponents is None:
            exponents = np.full((19, 2), -40)
            exponents[-1] = 80
        step.scales[ids, :, 1] = np.exp2(exponents)
        run(ops, step)
    # a last block whose scores are the lowest holds the largest values
    step.scales[step.table[0, :19], :, 1] = 2.0 ** 80
    step.scales[step.table[0, 0], :, 1] = 2.0 ** -40
    step.codes[0][step.table[0, 0]] = f32_to_e4m3(np.full((16, 2, 128), 448.0, np.float32))
    step.q_bits = f32_to_bits(np.abs(bits_to_f32(step.q_bits, "bf16")), "bf16")
    run(ops, step)


def test_one_visible_key_returns_its_value_exactly(ops) -> None:
    step = Step([(1, 1), (1, 1)], heads=4, head_dim=64, mode="decode", spread=6)
    out = run(ops, step).float().cpu().numpy()
    for b in range(2):
        value = e4m3_to_f32(step.codes[1][step.table[b, 0], 0]) * step.scales[step.table[b, 0], :, 1][:, None]
        assert np.array_equal(out[b], np.repeat(value, 2, axis=0))


# --- values that are not finite -----------------------------------------------------------------------


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("launch", ["decode", "windows", "windows split", "tiles", "tiles split", "half", "quarter",
                                    "double"])
def test_nan_reaches_the_rows_that_attend_to_it_alone(ops, launch, head_dim) -> None:
    if launch == "double" and head_dim == 64:
        pytest.skip("no double tile at this head width")
    full = hip_attention.PREFILL_PAIRS[head_dim]
    forced = {"decode": {}, "windows": dict(prefill=True, window=True, partitions=0),
              "windows split": dict(prefill=True, window=True, partition_size=64),
              "tiles": dict(prefill=True, window=False, tile_pairs=full, partitions=0),
              "tiles split": dict(prefill=True, window=False, tile_pairs=full, partition_size=64),
              "half": dict(prefill=True, window=False, tile_pairs=full // 2, partitions=0),
              "quarter": dict(prefill=True, window=False, tile_pairs=full // 4, partitions=0),
              "double": dict(prefill=True, window=False, tile_pairs=2 * full, partitions=0)}[launch]
    count = 1 if launch == "decode" else 4 if launch.startswith("windows") else 37
    step = Step([(count, 140), (count, 131)], heads=8, head_dim=head_dim, mode="decode" if count == 1 else "mixed",
                block=8, seed=2)

    def put(which, request, position, head, element, code=NAN):
        step.codes[which][step.table[request, position // 8], position % 8, head, element] = code

    # values: one that only the last row sees, one in the middle of the window, two of one piece, a
    # negative NaN, one that every row sees; the second request has none
    put(1, 0, 139, 0, 5)
    put(1, 0, 138, 1, head_dim - 1, 0xFF)
    put(1, 0, 137, 1, slice(8, 10))
    if count > 4:
        put(1, 0, 110, 0, 17)
    run(ops, step, label="values late", **forced)
    put(1, 0, 3, 0, 33)
    run(ops, step, label="values early", **forced)
    # a key: every element of the rows that attend to it
    put(0, 1, 130, 1, 7)
    run(ops, step, label="a key", **forced)


# --- the write and the attention that reads it ----------------------------------------------------------


def test_prompts_then_tokens_then_a_window(ops) -> None:
    # store and attend as an engine calls them, each step's attention over what the writes left,
    # against the oracle's own cache
    rng = np.random.default_rng(9)
    heads, kv_heads, dim, block = 8, 2, 128, 16
    lengths = [0, 0, 0]
    width = 8
    table = (1 + rng.permutation(3 * width)).reshape(3, width)
    step = Step([(1, 1)], heads=heads, kv_heads=kv_heads, head_dim=dim, block=block)
    step.codes = [block_scaled.empty(1 + 3 * width, block, kv_heads, dim)[0] for _ in range(2)]
    scales = [block_scaled.empty(1 + 3 * width, block, kv_heads, dim)[1] for _ in range(2)]
    step.table = table
    buffers = KVBuffers(*(torch.from_numpy(c.copy()).to(DEV).view(torch.float8_e4m3fn) for c in step.codes),
                        KVLayoutKind.NHD, fp8_e4m3_block_codec(torch.zeros(1 + 3 * width, kv_heads, 2, device=DEV)))
    for rows in ([40, 1, 17], [1, 1, 1], [1, 1, 1], [4, 2, 4], [1, 1, 1], [30, 1, 5]):
        lengths = [n + r for n, r in zip(lengths, rows)]
        n = sum(rows)
        size = np.exp2(rng.integers(-3, 3, (n, 1, 1)))
        k, v = ((rng.standard_normal((n, kv_heads, dim)) * size).astype(np.float32) for _ in range(2))
        bits = [f32_to_bits(x, "bf16") for x in (k, v)]
        step.rows, step.lengths = rows, lengths
        step.q_bits = f32_to_bits(rng.standard_normal((n, heads, dim)).astype(np.float32), "bf16")
        mode = ForwardMode.DECODE if max(rows) == 1 else ForwardMode.MIXED
        meta = ops.attention.plan(mode, torch.tensor(rows, device=DEV), torch.tensor(lengths, device=DEV),
                                  torch.from_numpy(table).to(DEV), block)
        dk, dv, q = (torch.from_numpy(b.view(np.int16)).view(torch.bfloat16).to(DEV) for b in (*bits, step.q_bits))
        out = torch.full_like(q, float("nan"))
        ops.kvcache.store(dk, dv, buffers, meta)
        ops.attention.attend(q, buffers, meta, out, scale=step.scale)
        for which in range(2):
            block_scaled.store(bits_to_f32(bits[which], "bf16"), meta.slot_mapping.cpu().numpy(), step.codes[which],
                               scales[which])
        step.scales = np.stack(scales, axis=2)
        step.check(out, f"rows {rows}")


def test_a_captured_decode_bucket(ops) -> None:
    # the write and the attention of two layers captured once on graph metadata and replayed over
    # steps whose scales grow, against the same steps run eagerly on caches of their own
    rng = np.random.default_rng(4)
    heads, kv_heads, dim, block, bucket, width = 8, 2, 64, 16, 4, 12
    lengths = np.array([30, 1, 0, 100])
    table = (1 + rng.permutation(bucket * width)).reshape(bucket, width).astype(np.int32)

    def caches():
        made = []
        for layer in range(2):
            g = torch.Generator(device=DEV).manual_seed(layer)
            codes = [torch.randint(0, 0x78, (1 + bucket * width, block, kv_heads, dim), generator=g, device=DEV,
                                   dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
            scales = torch.full((1 + bucket * width, kv_heads, 2), 2.0 ** -8, device=DEV)
            made.append(KVBuffers(*codes, KVLayoutKind.NHD, fp8_e4m3_block_codec(scales)))
        return made

    ours, theirs = caches(), caches()
    k, v = (torch.zeros(bucket, kv_heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(bucket, heads, dim, dtype=torch.bfloat16, device=DEV)
    outs = [torch.empty_like(q) for _ in range(2)]
    meta = ops.attention.graph_metadata(bucket, width, block, DEV)

    def layers(metadata, pools, results):
        for buffers, out in zip(pools, results):
            ops.kvcache.store(k, v, buffers, metadata)
            ops.attention.attend(q, buffers, metadata, out, scale=0.125)

    ops.attention.update_graph_metadata(meta, torch.zeros(bucket, dtype=torch.int32), torch.from_numpy(table))
    layers(meta, ours, outs)  # padding rows alone: the scratch exists, nothing is stored
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        layers(meta, ours, outs)
    for at in range(6):
        lengths = np.where(lengths > 0, lengths + 1, 0)
        if at == 3:
            lengths[2] = 1
        for x in (k, v, q):
            x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32) * (1.0 if x is q else 2.0 ** at)))
        ops.attention.update_graph_metadata(meta, torch.from_numpy(lengths.astype(np.int32)), torch.from_numpy(table))
        graph.replay()
        planned = ops.attention.plan(ForwardMode.DECODE, torch.ones(bucket, dtype=torch.int32, device=DEV),
                                     torch.from_numpy(lengths).to(DEV), torch.from_numpy(table).to(DEV), block)
        eager = [torch.empty_like(q) for _ in range(2)]
        layers(planned, theirs, eager)
        torch.cuda.synchronize()
        for a, b, x, y in zip(ours, theirs, outs, eager):
            assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)), at
            assert torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8)), at
            assert torch.equal(a.codec.scales, b.codec.scales), at
            # another split of the context: each of the two within the rounding of its weights
            # and its output, half a step of bf16 and of fp16 each
            size = y.float().abs().max()
            assert (x.float() - y.float()).abs().max() <= 2 * size * (2.0 ** -8 + 2.0 ** -10), at
            assert not x[lengths == 0].any()


@pytest.mark.parametrize("scale", [0.0, -0.1])
@pytest.mark.parametrize("mode,steps", [("decode", [(1, 300), (1, 0)]), ("mixed", [(4, 300)]), ("mixed", [(50, 300)])])
def test_softmax_scales_of_zero_and_below(ops, mode, steps, scale) -> None:
    for block in (16, 12, 7):
        step = Step(steps, heads=8, head_dim=128, mode=mode, block=block, seed=4)
        step.scale = scale
        # (S is of the scores' magnitudes; a scale of 0 averages the values)
        run(ops, step)


def test_queries_and_outputs_inside_other_tensors(ops) -> None:
    # rows that begin 16 bytes into their storage, caches 8 bytes; a step's first rows of larger outputs,
    # whose other rows stay as they were
    step = Step([(1, 40), (1, 77)], heads=4, mode="decode", head_dim=64)
    q, buffers, meta, out = step.device(ops)

    def moved(t, bytes_in, rows=None):
        flat = torch.full((t.numel() * t.element_size() + bytes_in + 512,), 0x55, dtype=torch.uint8, device=DEV)
        view = flat[bytes_in:bytes_in + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
        view.view(torch.uint8).copy_(t.view(torch.uint8))
        return view, flat

    q2, _ = moved(q, 16)
    out2, whole = moved(out, 16)
    k2, _ = moved(buffers.k, 8)
    v2, _ = moved(buffers.v, 8)
    ops.attention.attend(q2, buffers._replace(k=k2, v=v2), meta, out2, scale=step.scale)
    step.check(out2)
    size = out.numel() * out.element_size()
    assert (whole[:16] == 0x55).all() and (whole[16 + size:] == 0x55).all()
    odd, _ = moved(q, 2)
    with pytest.raises(BackendError, match="not 16-byte aligned"):
        ops.attention.attend(odd, buffers, meta, out, scale=step.scale)


@pytest.mark.parametrize("rows", [3, 40])
def test_a_captured_multi_row_step(ops, rows) -> None:
    step = Step([(rows, 900), (2, 60)], heads=8, head_dim=128, block=16, seed=6)
    q, buffers, meta, out = step.device(ops)
    ops.attention.attend(q, buffers, meta, out, scale=step.scale)  # its tiles and scratch
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.attention.attend(q, buffers, meta, out, scale=step.scale)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        ops.attention.attend(q, buffers, meta, torch.empty_like(out), scale=step.scale)
    step.check(out)


def test_repeated_calls_follow_scales_that_moved(ops) -> None:
    # a call is replayed from its record only while the scales lie where they did
    step = Step([(1, 40), (1, 70)], heads=4, mode="decode")
    q, buffers, meta, out = step.device(ops)
    for _ in range(3):
        ops.attention.attend(q, buffers, meta, out, scale=step.scale)
    step.check(out)
    moved = buffers._replace(codec=fp8_e4m3_block_codec(buffers.codec.scales * 2.0))
    ops.attention.attend(q, moved, meta, out, scale=step.scale)
    step.scales = step.scales * 2.0
    step.check(out)


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_a_pool_just_under_the_largest(ops, layout) -> None:
    # blocks whose byte offsets pass 2^31, up to the pool's last, beside its first: the write, the moves and
    # every kind of step give bit for bit what they give over a small pool
    block, kv_heads, dim = 16, 8, 128
    blocks = 2 ** 32 // (block * kv_heads * dim) - 1
    shape = (blocks, block, kv_heads, dim) if layout == "nhd" else (blocks, kv_heads, block, dim)
    big = KVBuffers(*(torch.empty(shape, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2)), LAYOUTS[layout],
                    fp8_e4m3_block_codec(torch.zeros(blocks, kv_heads, 2, device=DEV)))
    codes = lambda t: t.view(torch.uint8)
    for mode, steps in (("decode", [(1, 700), (1, 33)]), ("mixed", [(3, 500), (2, 40)]), ("mixed", [(50, 300), (70, 90)])):
        step = Step(steps, layout=layout, heads=16, kv_heads=kv_heads, head_dim=dim, block=block, mode=mode, seed=8)
        q, small, meta, out = step.device(ops)
        n = small.k.shape[0]
        ids = torch.arange(n, device=DEV)
        ids[n // 2:] += blocks - n  # the upper half at the pool's end
        assert int(ids[-1]) == blocks - 1
        for a, b in ((big.k, small.k), (big.v, small.v)):
            codes(a)[ids] = codes(b)
        big.codec.scales[ids] = small.codec.scales
        table = ids[torch.from_numpy(step.table).to(DEV)]
        far = ops.attention.plan(step.mode, torch.tensor(step.rows, device=DEV), torch.tensor(step.lengths, device=DEV),
                                 table, block)
        rows = [torch.randn(len(q), kv_heads, dim, device=DEV).to(q.dtype) for _ in range(2)]
        again = torch.full_like(out, float("nan"))
        for buffers, metadata, to in ((small, meta, out), (big, far, again)):
            ops.kvcache.store(*rows, buffers, metadata)
            ops.attention.attend(q, buffers, metadata, to, scale=step.scale)
        assert torch.equal(out, again)
        got = [torch.empty_like(small.k), torch.empty_like(small.v)]
        scales = torch.empty_like(small.codec.scales)
        ops.kvcache.gather(big, ids, *got, out_scales=scales)
        assert torch.equal(codes(got[0]), codes(small.k)) and torch.equal(codes(got[1]), codes(small.v))
        assert torch.equal(scales.nan_to_num(-1.0), small.codec.scales.nan_to_num(-1.0))


def test_another_stream(ops) -> None:
    step = Step([(1, 900), (1, 2000), (1, 50)], heads=8, head_dim=128, mode="decode")
    q, buffers, meta, out = step.device(ops)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        ops.attention.attend(q, buffers, meta, out, scale=step.scale)
        with torch.cuda.stream(other):
            again = torch.empty_like(out)
            ops.attention.attend(q, buffers, meta, again, scale=step.scale)
    torch.cuda.synchronize()
    step.check(out)
    assert torch.equal(out, again)


def test_refusals(ops) -> None:
    step = Step([(1, 40)], heads=4, mode="decode")
    q, buffers, meta, out = step.device(ops)
    with pytest.raises(BackendError, match="16-bit caches only"):
        hip_attention.attend_with(q, buffers, meta, out, scale=1.0, partitions=0, qk="dpp")
    with pytest.raises(BackendError, match="computes in float16, bfloat16"):
        ops.attention.attend(q.float(), buffers, meta, out.float(), scale=1.0)
    with pytest.raises(BackendError, match=r"scales must be float32 \[6, 2, 2\]"):
        wrong = buffers._replace(codec=fp8_e4m3_block_codec(torch.zeros(3, 2, 2, device=DEV)))
        ops.attention.attend(q, wrong, meta, out, scale=1.0)
