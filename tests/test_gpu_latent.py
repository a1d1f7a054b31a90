"""Attention over latent caches, both forms, against the definitions in 64 bits.

Bounds, per output element, with A the element's sum of weighted magnitudes (sum p |v|), R the largest
sum of |q| |k| over a visible position times the scale, and e the type's half step (eps / 2):

* the output's own rounding, e |out|;
* a score is a sum of products in fp32, at most 64 roundings deep (18 products of 32 in two chains, or 12,
  and their ends), each 2^-24 of R; a relative change d of every weight moves the output by at most
  2 d A (numerator and denominator), and so do the exponential's and the split's errors:
  2 (64 R 2^-24 + 2^-20) A;
* weights: bf16 in two parts lose 2^-14 of themselves, fp16 half a step, 2^-11, below 2^-14 of the running
  maximum (up to 2^8 under the true one) an absolute 2^-25, of up to n positions:
  A 2^-11 + n 2^-25 max |v|;
* expanded keys and values are fp16: 2^-11 R more on scores, 2^-11 A more on values (and 2^-38 of a tile's
  largest, which the factor of 2 of the first bound covers here);
* sums of n weighted values in fp32: (n / 32 + 40) 2^-24 A.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, ForwardMode
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import latent as hip_latent
from ayaka_amd.kvcache import BlockPool, LatentBuffers, LatentWeights
from ayaka_amd.rotary import rotary
from oracle import latent as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


class Scene:
    """A latent cache with every unheld slot NaN, a step of ``(rows, length)``, and its queries."""

    def __init__(self, ops, steps, *, dtype="bf16", heads=4, latent=512, block=16, seed=0, loud=1.0, form="absorbed",
                 q_scale=1.0) -> None:
        rng = np.random.default_rng(seed)
        self.ops, self.form, self.dtype, self.latent, self.heads, self.block = ops, form, TYPES[dtype], latent, heads, block
        self.rows, self.lengths = [r for r, _ in steps], [n for _, n in steps]
        need = [-(-n // block) for n in self.lengths]
        self.blocks = 1 + sum(need) + 2
        ids = list(rng.permutation(np.arange(1, self.blocks)))
        self.table = np.zeros((len(steps), max(1, max(need))), dtype=np.int64)
        cache = np.full((self.blocks, block, latent + 64), np.nan, dtype=np.float32)
        for b, (n, length) in enumerate(zip(need, self.lengths)):
            self.table[b, :n] = [ids.pop() for _ in range(n)]
            t = np.arange(length)
            cache[self.table[b, t // block], t % block] = rng.standard_normal((length, latent + 64)) * loud
        self.cache = torch.tensor(cache).to(self.dtype).to(DEV)
        n = sum(self.rows)
        if form == "absorbed":
            q = rng.standard_normal((n, heads, latent + 64)) * (128 / latent) ** 0.5
        else:
            q = rng.standard_normal((n, heads, 192))
            self.weights = LatentWeights(*(torch.tensor(rng.standard_normal((heads, 128, latent)) * latent ** -0.5)
                                           .to(self.dtype).to(DEV) for _ in range(2)))
        self.q = torch.tensor(q * q_scale / loud).to(self.dtype).to(DEV)
        self.scale = 192 ** -0.5
        mode = ForwardMode.DECODE if all(r == 1 for r in self.rows) else ForwardMode.MIXED
        self.meta = ops.attention.plan(mode, torch.tensor(self.rows, device=DEV), torch.tensor(self.lengths, device=DEV),
                                       torch.tensor(self.table, device=DEV), block)

    @property
    def buffers(self) -> LatentBuffers:
        return LatentBuffers(self.cache, self.latent)

    def out(self) -> torch.Tensor:
        return torch.full((len(self.q), self.heads, self.latent if self.form == "absorbed" else 128), 7.0, dtype=self.dtype, device=DEV)

    def run(self, out=None, meta=None) -> torch.Tensor:
        out = self.out() if out is None else out
        meta = self.meta if meta is None else meta
        if self.form == "absorbed":
            self.ops.attention.attend_latent(self.q, self.buffers, meta, out, scale=self.scale)
        else:
            self.ops.attention.attend_latent_chunks(self.q, self.weights, self.buffers, meta, out, scale=self.scale)
        return out

    def want(self):
        host = self.cache.double().cpu().numpy(), self.table, self.rows, self.lengths, self.scale
        q = self.q.double().cpu().numpy()
        if self.form == "absorbed":
            return oracle.attention(q, *host, self.latent)
        return oracle.chunk_attention(q, *(w.double().cpu().numpy() for w in self.weights), *host)

    def check(self, got=None) -> None:
        got = self.run() if got is None else got
        out, size, reach = self.want()
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(out))
        e, n = torch.finfo(self.dtype).eps / 2, max(self.lengths)
        expanded = self.form != "absorbed"
        fine = np.isfinite(size)
        half = 2.0 ** -11
        d = 2 * (64 * reach * 2.0 ** -24 + 2.0 ** -20) + (n / 32 + 40) * 2.0 ** -24 + 2.0 ** -14
        if expanded or self.dtype is torch.float16:
            d = d + half
        if expanded:
            d = d + 2 * reach * half + half
        most = np.max(size[fine], initial=0.0)
        bound = e * np.abs(out) + size * d + n * 2.0 ** -25 * most * 2 + float(torch.finfo(self.dtype).smallest_normal) * e * 2
        off = np.abs(got - out)[fine]
        assert np.all(off <= bound[fine]), (float((off - bound[fine]).max()), float(off.max()))
        # and on average: the roundings are independent, so the whole is off by a root mean square of them
        norm = np.sqrt((out[fine] ** 2).sum())
        if norm:
            reach = min(4.0, float(np.max(reach)))
            rms = np.sqrt(3 + (reach if expanded else 0) ** 2) if expanded or self.dtype is torch.float16 else 1.5
            assert np.sqrt((off ** 2).sum()) / norm <= max(e, half if expanded else 0) * rms + 1e-6


LENGTHS = [(1, 1), (1, 31), (1, 32), (1, 33), (1, 0), (1, 64), (1, 500), (1, 129), (1, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("latent", [256, 512])
@pytest.mark.parametrize("heads", [1, 5, 16, 20, 32, 128])
def test_decode(ops, dtype, latent, heads) -> None:
    Scene(ops, LENGTHS, dtype=dtype, latent=latent, heads=heads, block=16).check()


@pytest.mark.parametrize("block", [1, 7, 24, 128, 1024])
def test_block_sizes(ops, block) -> None:
    Scene(ops, [(1, 1100), (2, 1030), (1, 5)], heads=3, block=block, seed=block).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [1, 7, 16, 48])
@pytest.mark.parametrize("steps", [
    [(4, 200), (4, 33), (1, 0), (4, 4)],          # verify windows
    [(1, 90), (0, 50), (70, 70), (3, 0), (33, 300)],  # decode beside prompts, a request without rows
    [(130, 130)],
])
def test_several_rows(ops, dtype, heads, steps) -> None:
    Scene(ops, steps, dtype=dtype, heads=heads, block=24, seed=heads).check()


def test_one_long_context_is_cut_among_workgroups(ops) -> None:
    Scene(ops, [(1, 20000)], heads=2, block=64).check()
    Scene(ops, [(2, 9000)], heads=64, block=64, dtype="fp16").check()


def test_more_requests_than_workgroups_threads(ops) -> None:
    """The sums over requests run through several of them a thread."""
    rng = np.random.default_rng(5)
    steps = [(int(r), int(n)) if n >= r else (1, 0) for r, n in zip(rng.integers(0, 3, 1300), rng.integers(0, 40, 1300))]
    Scene(ops, steps, heads=2, latent=256, block=8).check()


def test_wide_tables_are_read_in_windows(ops) -> None:
    """More blocks than the table's window in LDS holds, whose ends fall inside chunks."""
    Scene(ops, [(1, 2500), (3, 1999)], heads=2, latent=256, block=1).check()
    Scene(ops, [(1, 5000)], heads=2, latent=256, block=3).check()
    Scene(ops, [(2, 2500), (1, 30), (3, 1700)], heads=40, latent=256, block=1).check()


@pytest.mark.parametrize("form", ["absorbed", "chunks"])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(ops, form, dtype) -> None:
    """Scores of hundreds, where one position takes nearly all weight, and all equal ones."""
    Scene(ops, [(1, 300), (6, 150)], form=form, dtype=dtype, heads=3, q_scale=200.0, seed=3).check()
    Scene(ops, [(1, 300), (6, 150)], form=form, dtype=dtype, heads=3, q_scale=0.0, seed=3).check()


@pytest.mark.parametrize("form", ["absorbed", "chunks"])
@pytest.mark.parametrize("scale", [-0.05, 0.0, 1e-30])
def test_scales_of_any_sign(ops, form, scale) -> None:
    s = Scene(ops, [(1, 300), (6, 150), (70, 70)], form=form, heads=3, seed=31)
    s.scale = scale
    s.check()


@pytest.mark.parametrize("form", ["absorbed", "chunks"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
@pytest.mark.parametrize("size", [16.0, 2.0 ** 14])
def test_scores_far_apart(ops, form, dtype, order, size) -> None:
    """Scores thousands apart, up to 2^30: each row is the value of one position it sees. Every number that the
    scores are made of is exact, so the position that wins is, and its weight is 1."""
    length, rows, heads = 250, 130, 3
    s = Scene(ops, [(1, 40), (rows, length)], form=form, dtype=dtype, heads=heads, seed=32)
    key = {"up": np.arange(length), "down": -np.arange(length), "mixed": (np.arange(length) * 89) % 251 - 125}[order]
    t = np.arange(length)
    at = torch.as_tensor(s.table[1, t // 16]), torch.as_tensor(t % 16)
    s.cache[(*at, 0)] = torch.tensor(key).to(s.dtype).to(DEV)
    s.q.zero_()
    s.q[..., 0] = size
    if form == "chunks":  # the key's first element is the latent's
        s.weights.keys.zero_()
        s.weights.keys[:, 0, 0] = 1
    s.scale = 1024.0
    got, want = s.run().double().cpu().numpy()[1:], s.want()[0][1:]
    winner = np.array([np.argmax(key[:length - rows + i + 1]) for i in range(rows)])
    values = s.cache[at].double().cpu().numpy()[winner][:, None, :s.latent].repeat(heads, 1)
    if form == "chunks":
        values = np.einsum("rhc,hvc->rhv", values, s.weights.values.double().cpu().numpy())
    assert np.allclose(want, values, rtol=1e-12, atol=1e-12)
    bound = torch.finfo(s.dtype).eps / 2 * np.abs(values) + (2.0 ** -11 + 2.0 ** -20) * (np.abs(values) + 2.0 ** -26)
    if form == "chunks":  # three half steps of fp16, and a value's sum: 18 roundings of 2^-24 of up to 40
        bound = bound * 2 + 2.0 ** -14
    assert np.all(np.abs(got - values) <= bound)


def test_a_maximum_that_grows_all_the_way(ops) -> None:
    """Every chunk moves the running maximum; and scores that all lie far below zero."""
    s = Scene(ops, [(1, 400), (2, 390)], heads=4, seed=8)
    for sign in (1, -1):
        direction = s.q[:1, 0].float().mean(0).sign()
        for b, length in enumerate(s.lengths):
            t = np.arange(length)
            at = torch.as_tensor(s.table[b, t // 16]), torch.as_tensor(t % 16)
            grow = torch.linspace(0, 3, length)[:, None].to(DEV) + (2.0 if sign < 0 else 0.0)
            s.cache[at] = (sign * direction * grow).to(s.dtype)
        s.q.copy_(direction.expand_as(s.q).to(s.dtype) * 0.5)
        s.check()


@pytest.mark.parametrize("form", ["absorbed", "chunks"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["latent", "rope"])
def test_rows_do_not_notice_what_they_do_not_see(ops, form, dtype, value, where) -> None:
    """A non-finite element at a position some rows of the request see and others do not."""
    s = Scene(ops, [(5, 300), (1, 64), (40, 40)], form=form, dtype=dtype, heads=5, seed=4)
    for b, t in ((0, 298), (2, 20)):
        s.cache[int(s.table[b, t // 16]), t % 16, 3 if where == "latent" else s.latent + 3] = value
    clean = Scene(ops, [(5, 300), (1, 64), (40, 40)], form=form, dtype=dtype, heads=5, seed=4)
    got, ref = s.run(), clean.run()
    blind = [0, 1, 2, 5, *range(6, 26)]  # rows before the position, and another request's
    assert torch.equal(got[blind], ref[blind])
    seeing = [3, 4, *range(26, 46)]
    want = s.want()[0]
    if value != value:
        assert got[seeing].isnan().all()
    # an infinity makes a row NaN where its score is +inf or NaN, and where that is -inf only its own element
    # (0 times infinity): what the definition gives, element by element
    if form == "absorbed":
        assert np.array_equal(got[seeing].isnan().cpu().numpy(), np.isnan(want[seeing]))
    for row in seeing:
        for h in range(s.heads):
            assert np.isnan(want[row, h]).all() == bool(got[row, h].isnan().all())


def test_types_lowest_and_highest_values(ops) -> None:
    s = Scene(ops, [(2, 70)], heads=2, seed=6)
    s.cache[int(s.table[0, 4]), 5] = torch.finfo(torch.bfloat16).min  # position 69: every product with it overflows
    got = s.run()
    assert torch.equal(got[0], Scene(ops, [(2, 70)], heads=2, seed=6).run()[0])  # the row before it
    # scores that overflowed make NaN or, at -inf, no weight: what is a number is the definition's
    got, want = got.double().cpu().numpy(), s.want()[0]
    assert np.all(np.isnan(got) | (np.abs(got - want) <= 2 ** -6 * (1 + np.abs(want))))


@pytest.mark.parametrize("form", ["absorbed", "chunks"])
def test_values_of_all_that_the_type_holds(ops, form) -> None:
    s = Scene(ops, [(2, 70)], form=form, heads=2, seed=6, q_scale=0.0)
    s.cache[int(s.table[0, 1]), 3] = torch.where(s.cache[int(s.table[0, 1]), 3] > 0, 1e30, -1e30)
    s.check()


@pytest.mark.parametrize("loud", [1e-6, 1e4, 1e12])
def test_chunks_of_any_magnitude(ops, loud) -> None:
    """Expanded keys and values past what fp16 holds, or all far below 1."""
    Scene(ops, [(5, 300), (40, 140)], form="chunks", heads=3, loud=loud, seed=7).check()


def test_chunks_beside_louder_and_quieter_ones(ops) -> None:
    """Tiles of 128 tokens of very different size, in every order."""
    s = Scene(ops, [(3, 900)], form="chunks", heads=2, seed=9, q_scale=0.05)
    t = np.arange(900)
    sizes = torch.tensor([1.0, 64.0, 2.0 ** -8, 2.0 ** 9, 1.0, 2.0 ** -20, 32.0, 0.0])[t // 128].to(DEV)
    at = torch.as_tensor(s.table[0, t // 16]), torch.as_tensor(t % 16)
    s.cache[at] = (s.cache[at].float() * sizes[:, None]).to(s.dtype)
    s.check()


def test_chunks_over_a_long_context(ops) -> None:
    """More tiles than the window of their scales holds, each of another magnitude."""
    s = Scene(ops, [(3, 33100), (130, 140)], form="chunks", heads=1, block=64, seed=33, q_scale=0.3)
    t = np.arange(33100)
    sizes = torch.tensor(2.0 ** ((t // 128 * 5) % 7 - 3), dtype=torch.float32).to(DEV)
    at = torch.as_tensor(s.table[0, t // 64]), torch.as_tensor(t % 64)
    s.cache[at] = (s.cache[at].float() * sizes[:, None]).to(s.dtype)
    s.check()


CHUNKS = [(1, 1), (127, 127), (128, 128), (129, 300), (1, 0), (0, 30), (33, 65), (200, 257)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("latent", [256, 512])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_chunks(ops, dtype, latent, heads) -> None:
    Scene(ops, CHUNKS, form="chunks", dtype=dtype, latent=latent, heads=heads, block=24, seed=heads).check()


@pytest.mark.parametrize("block", [1, 7, 128])
def test_chunk_block_sizes(ops, block) -> None:
    Scene(ops, [(60, 500), (300, 333)], form="chunks", heads=2, block=block, seed=block).check()


def test_chunks_some_heads_at_a_time(ops, monkeypatch) -> None:
    s = Scene(ops, CHUNKS, form="chunks", heads=20, latent=256, seed=2)
    whole = s.run()
    ws_rows = sum(-(-n // 128) * 128 for r, n in CHUNKS if r and n)
    for heads in (1, 3, 8, 17):
        again = Scene(ops, CHUNKS, form="chunks", heads=20, latent=256, seed=2)
        monkeypatch.setattr(hip_latent, "EXPANDED_BYTES", ws_rows * 512 * heads)
        assert torch.equal(again.run(), whole), heads


def test_only_rows_without_a_context(ops) -> None:
    for form in ("absorbed", "chunks"):
        s = Scene(ops, [(1, 0), (3, 0)], form=form, heads=4)
        assert not s.run().any()
        none = ops.attention.plan(ForwardMode.IDLE, *(torch.zeros(2, dtype=torch.int32, device=DEV),) * 2,
                                  torch.zeros(2, 1, dtype=torch.int32, device=DEV), 16)
        s.q = s.q[:0]
        s.run(out=torch.empty(0, 4, s.out().shape[2], dtype=s.dtype, device=DEV), meta=none)


def test_both_forms_agree(ops) -> None:
    """Absorbed between the projections is the expanded form, and the expanded one over the same cache."""
    s = Scene(ops, [(3, 400), (100, 150), (1, 9)], form="chunks", heads=6, dtype="fp16", seed=11)
    q = s.q.float()
    absorbed = torch.cat((torch.bmm(q[..., :128].transpose(0, 1).contiguous(), s.weights.keys.float()).transpose(0, 1), q[..., 128:]), dim=-1)
    mid = torch.empty(len(q), 6, 512, dtype=s.dtype, device=DEV)
    ops.attention.attend_latent(absorbed.to(s.dtype).contiguous(), s.buffers, s.meta, mid, scale=s.scale)
    got = torch.bmm(mid.float().transpose(0, 1).contiguous(), s.weights.values.float().transpose(1, 2).contiguous()).transpose(0, 1)
    want = s.run().float()
    # queries and latents sums rounded to fp16 in between: a few half steps of 2^-11, on scores of up to 8
    assert float((got - want).norm() / want.norm()) < 8 * 2 ** -11


@pytest.fixture(params=[16, 32, 64])
def tiles(request, monkeypatch) -> int:
    """The (row, head) pairs of a tile, whatever a step's lengths would have."""
    monkeypatch.setattr(hip_latent, "_tile_pairs", lambda *_: request.param)
    return request.param


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("latent", [256, 512])
@pytest.mark.parametrize("heads", [1, 5, 16, 40, 128])
def test_tiles_of_every_size(ops, tiles, dtype, latent, heads) -> None:
    steps = [(1, 1), (1, 0), (2, 33), (1, 700), (5, 64), (0, 20), (17, 130), (1, 300)]
    Scene(ops, steps, dtype=dtype, latent=latent, heads=heads, seed=tiles).check()


def test_tiles_over_cut_contexts_and_windows(ops, tiles) -> None:
    Scene(ops, [(1, 9000), (3, 4001)], heads=24, block=64, seed=42).check()
    Scene(ops, [(2, 2500), (1, 30), (3, 1700)], heads=40, latent=256, block=1, dtype="fp16", seed=43).check()
    Scene(ops, [(1, 300), (6, 150)], heads=30, q_scale=200.0, seed=44).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_tiles_do_not_show_what_a_row_does_not_see(ops, tiles, dtype, value) -> None:
    steps = [(5, 300), (1, 64), (40, 40)]
    s, clean = (Scene(ops, steps, dtype=dtype, heads=9, seed=45) for _ in range(2))
    for b, t in ((0, 298), (2, 20)):
        s.cache[int(s.table[b, t // 16]), t % 16, 7] = value
    got, ref = s.run(), clean.run()
    blind, seeing = [0, 1, 2, 5, *range(6, 26)], [3, 4, *range(26, 46)]
    assert torch.equal(got[blind], ref[blind])
    assert np.array_equal(got[seeing].isnan().cpu().numpy(), np.isnan(s.want()[0][seeing]))


@pytest.fixture(params=[1, 2, 3, 7])
def parts(request, monkeypatch) -> int:
    """The parts that contexts are cut into, whatever a step's lengths would have."""
    monkeypatch.setattr(hip_latent, "_chunk_splits", lambda *_: request.param)
    return request.param


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [1, 5])
def test_chunks_over_cut_contexts(ops, parts, dtype, heads) -> None:
    """Parts of many rounds and of none, of which a row sees some."""
    Scene(ops, CHUNKS, form="chunks", dtype=dtype, heads=heads, seed=46).check()
    Scene(ops, [(300, 1500), (2, 900)], form="chunks", dtype=dtype, heads=heads, q_scale=20.0, seed=47).check()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_cut_contexts_do_not_show_what_a_row_does_not_see(ops, parts, value) -> None:
    s, clean = (Scene(ops, [(150, 400), (1, 64)], form="chunks", heads=3, seed=48) for _ in range(2))
    s.cache[int(s.table[0, 330 // 16]), 330 % 16, 5] = value
    got, ref = s.run(), clean.run()
    assert torch.equal(got[:80], ref[:80]) and torch.equal(got[150], ref[150])
    want = s.want()[0]
    for row in range(80, 150):
        for h in range(3):
            assert np.isnan(want[row, h]).all() == bool(got[row, h].isnan().all())


def test_long_contexts_cut_inside_their_scales_window(ops, monkeypatch) -> None:
    monkeypatch.setattr(hip_latent, "_chunk_splits", lambda *_: 5)
    s = Scene(ops, [(3, 40100)], form="chunks", heads=1, block=64, seed=49, q_scale=0.3)
    t = np.arange(40100)
    sizes = torch.tensor(2.0 ** ((t // 128 * 5) % 7 - 3), dtype=torch.float32).to(DEV)
    at = torch.as_tensor(s.table[0, t // 64]), torch.as_tensor(t % 64)
    s.cache[at] = (s.cache[at].float() * sizes[:, None]).to(s.dtype)
    s.check()


@pytest.mark.parametrize("form", ["absorbed", "chunks"])
def test_same_bits_every_time(ops, form) -> None:
    s = Scene(ops, [(2, 3000), (1, 77), (30, 600)], form=form, heads=9, seed=12)
    first = s.run()
    for _ in range(5):
        assert torch.equal(s.run(), first)


def test_bad_block_ids_stay_inside_the_pool(ops) -> None:
    """Ids outside the pool read block 0, as the other attention kernels do."""
    for form in ("absorbed", "chunks"):
        s = Scene(ops, [(2, 100), (1, 40)], form=form, heads=2, seed=13)
        s.cache[0] = 0.25
        for bad in (-1, s.blocks, 1 << 30, -(1 << 31)):
            s.meta.block_table[0, 2] = bad
            s.table[0, 2] = 0
            s.check(s.run())


def test_rows_past_the_requests_are_left_alone(ops) -> None:
    """A step whose device rows were lowered behind the plan: the rows no request has stay as they were."""
    s = Scene(ops, [(2, 100), (3, 40)], heads=4, seed=14)
    s.meta.rows_per_request.copy_(torch.tensor([2, 1], dtype=torch.int32))
    out = s.run()
    assert bool((out[3:] == 7.0).all())
    s.meta.rows_per_request.copy_(torch.tensor([2, 900], dtype=torch.int32))  # more than there are
    out = s.run()
    assert out.shape[0] == 5


def test_a_cache_of_more_than_2_to_32_elements(ops) -> None:
    block, blocks = 64, (1 << 32) // (64 * 576) + 200
    cache = torch.empty(blocks, block, 576, dtype=torch.bfloat16, device=DEV)
    s = Scene(ops, [(1, 150), (20, 90)], heads=4, block=block, seed=15)
    c = Scene(ops, [(1, 150), (20, 90)], heads=4, block=block, seed=15, form="chunks")
    for x in (s, c):
        small, want = x.cache, x.run()
        used = x.table > 0
        far = np.where(used, blocks - 1 - x.table, 0)
        cache[torch.as_tensor(far[used])] = small[torch.as_tensor(x.table[used])]
        x.cache, x.table = cache, far
        x.meta = ops.attention.plan(ForwardMode.MIXED, torch.tensor(x.rows, device=DEV), torch.tensor(x.lengths, device=DEV),
                                    torch.tensor(far, device=DEV), block)
        assert torch.equal(x.run(), want)
    turn = rotary(64, device=DEV)
    down = torch.randn(21, 576, device=DEV).to(torch.bfloat16)
    ops.kvcache.store_latent(down[:, :512], down[:, 512:], LatentBuffers(cache, 512), s.meta, turn)
    slots = s.meta.slot_mapping
    assert int(slots.max()) * 576 > 1 << 32
    assert torch.equal(cache.view(-1, 576)[slots][:, :512], down[:, :512])


@pytest.mark.parametrize("heads", [4, 16, 40])
def test_captured_bucket(ops, heads) -> None:
    """A decode bucket captured once and replayed over other lengths, with eager calls between."""
    rng = np.random.default_rng(heads)
    block, width, requests = 16, 40, 6
    s = Scene(ops, [(1, width * block)] * requests, heads=heads, block=block, seed=16)
    meta = ops.attention.graph_metadata(requests, width, block, DEV)
    table = torch.tensor(s.table, dtype=torch.int32)
    ops.attention.update_graph_metadata(meta, torch.full((requests,), 100, dtype=torch.int32), table)
    out = s.out()
    s.run(out, meta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(out, meta)
    for _ in range(4):
        lengths = rng.integers(0, width * block + 1, requests)
        lengths[rng.integers(0, requests)] = 0
        ops.attention.update_graph_metadata(meta, torch.tensor(lengths, dtype=torch.int32), table)
        s.q.copy_(torch.randn_like(s.q, dtype=torch.float32).to(s.dtype) * 0.5)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        s.lengths = lengths.tolist()
        s.check(replayed)
        assert torch.equal(s.run(meta=meta), replayed)


def test_captured_chunks(ops) -> None:
    s = Scene(ops, [(40, 300), (1, 20)], form="chunks", heads=3, seed=17)
    fresh = Scene(ops, [(40, 300), (1, 20)], form="chunks", heads=3, seed=17)
    with pytest.raises(BackendError, match="run the step once eagerly"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.run()
    torch.cuda.synchronize()
    out = s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(out)
    for i in range(3):
        s.q.copy_(torch.randn_like(s.q, dtype=torch.float32).to(s.dtype))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        s.check(out)
        assert torch.equal(s.run(), out)


def test_two_streams_share_the_scratch(ops) -> None:
    a = Scene(ops, [(1, 9000)], heads=3, seed=18)
    b = Scene(ops, [(100, 700)], heads=3, form="chunks", seed=19)
    want = a.run(), b.run()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [(a.out(), b.out()) for _ in range(6)]
    for x, y in outs:
        with torch.cuda.stream(streams[0]):
            a.run(x)
        with torch.cuda.stream(streams[1]):
            b.run(y)
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_refusals(ops) -> None:
    s = Scene(ops, [(1, 30), (2, 20)], heads=4)
    c = Scene(ops, [(1, 30), (2, 20)], heads=4, form="chunks")
    out, attend, chunks = s.out(), ops.attention.attend_latent, ops.attention.attend_latent_chunks
    bucket = ops.attention.graph_metadata(3, 4, 16, DEV)
    odd = torch.zeros(4, 16, 448, dtype=torch.bfloat16, device=DEV)
    cases = [
        (lambda: attend(s.q[:2], s.buffers, s.meta, out, scale=1.0), "q must be bfloat16"),
        (lambda: attend(s.q[..., :512].contiguous(), s.buffers, s.meta, out, scale=1.0), r"\[3, 4, 576\]"),
        (lambda: attend(s.q.half(), s.buffers, s.meta, out, scale=1.0), "q must be bfloat16"),
        (lambda: attend(s.q.transpose(0, 1).contiguous().transpose(0, 1), s.buffers, s.meta, out, scale=1.0), "contiguous"),
        (lambda: attend(s.q, s.buffers, s.meta, out[..., :64], scale=1.0), "out must be"),
        (lambda: attend(s.q, LatentBuffers(odd, 384), s.meta, out, scale=1.0), "not 384 and 64"),
        (lambda: attend(s.q, LatentBuffers(s.cache, 500), s.meta, out, scale=1.0), "not 500 and 76"),
        (lambda: attend(s.q.float(), LatentBuffers(s.cache.float(), 512), s.meta, out.float(), scale=1.0), "computes in float16, bfloat16"),
        (lambda: attend(s.q, LatentBuffers(s.cache.view(-1, 8, 576), 512), s.meta, out, scale=1.0), "planned for blocks of 16"),
        (lambda: attend(s.q[:, 0], s.buffers, s.meta, out, scale=1.0), "q must be"),
        (lambda: chunks(c.q, c.weights._replace(keys=c.weights.keys[:2]), c.buffers, c.meta, c.out(), scale=1.0), "weights.keys must be"),
        (lambda: chunks(c.q, c.weights._replace(values=c.weights.values.float()), c.buffers, c.meta, c.out(), scale=1.0), "weights.values must be"),
        (lambda: chunks(c.q, c.weights, c.buffers, bucket, c.out(), scale=1.0), "made by plan"),
        (lambda: chunks(s.q, c.weights, c.buffers, c.meta, c.out(), scale=1.0), "q must be"),
    ]
    for call, message in cases:
        with pytest.raises(BackendError, match=message):
            call()


def test_a_model_layer_from_prompt_to_decode(ops) -> None:
    """Prompts stored and attended to in chunks, then a decode loop on a captured bucket that stores, and
    attends in absorbed form: each step against the definition over all tokens so far."""
    heads, latent, block, width = 4, 512, 16, 12
    g = torch.Generator(device="cuda").manual_seed(21)
    t = torch.bfloat16

    def rand(*shape, size=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * size).to(t)

    weights = LatentWeights(rand(heads, 128, latent, size=latent ** -0.5), rand(heads, 128, latent, size=latent ** -0.5))
    turn, scale = rotary(64, interleaved=True, device=DEV), 192 ** -0.5
    lengths = [70, 33, 150]
    table = torch.tensor(np.random.default_rng(3).permutation(np.arange(1, 1 + 3 * width)).reshape(3, width), dtype=torch.int32)
    cache = torch.full((2 + 3 * width, block, latent + 64), float("nan"), dtype=t, device=DEV)
    buffers = LatentBuffers(cache, latent)

    def definition(q, rows, lens):
        return oracle.chunk_attention(q.double().cpu().numpy(), *(w.double().cpu().numpy() for w in weights),
                                      cache.double().cpu().numpy(), table.numpy(), rows, lens, scale)[0]

    n = sum(lengths)
    down, q = rand(n, latent + 64), rand(n, heads, 192)
    meta = ops.attention.plan(ForwardMode.PREFILL, torch.tensor(lengths, device=DEV), torch.tensor(lengths, device=DEV), table.to(DEV), block)
    ops.kvcache.store_latent(down[:, :latent], down[:, latent:], buffers, meta, turn, q[:, :, 128:])
    out = torch.empty(n, heads, 128, dtype=t, device=DEV)
    ops.attention.attend_latent_chunks(q, weights, buffers, meta, out, scale=scale)
    want = definition(q, lengths, lengths)
    assert np.linalg.norm(out.double().cpu().numpy() - want) <= 2 ** -8 * np.linalg.norm(want)

    bucket = ops.attention.graph_metadata(3, width, block, DEV)
    new, q1 = rand(3, latent + 64), rand(3, heads, 192)
    absorbed = torch.empty(3, heads, latent + 64, dtype=t, device=DEV)
    mid, final = torch.empty(3, heads, latent, dtype=t, device=DEV), torch.empty(3, heads, 128, dtype=torch.float32, device=DEV)
    keys32, values32 = weights.keys.float(), weights.values.float().transpose(1, 2).contiguous()

    def layer():
        absorbed[:, :, :latent] = torch.bmm(q1[:, :, :128].transpose(0, 1).float().contiguous(), keys32).transpose(0, 1)
        ops.kvcache.store_latent(new[:, :latent], new[:, latent:], buffers, bucket, turn, q1[:, :, 128:], absorbed[:, :, latent:])
        ops.attention.attend_latent(absorbed, buffers, bucket, mid, scale=scale)
        final.copy_(torch.bmm(mid.transpose(0, 1).float().contiguous(), values32).transpose(0, 1))

    graph = None
    for step in range(5):
        lengths = [length + 1 for length in lengths]
        ops.attention.update_graph_metadata(bucket, torch.tensor(lengths, dtype=torch.int32), table)
        new.copy_(rand(3, latent + 64))
        q1.copy_(rand(3, heads, 192))
        if step == 1:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                layer()
        if graph is None:
            layer()
        else:
            graph.replay()
        torch.cuda.synchronize()
        turned = torch.cat((q1[:, :, :128], absorbed[:, :, latent:]), dim=-1)
        want = definition(turned, [1, 1, 1], lengths)
        # queries rounded to bf16 after the keys' matrix (a half step, 2^-9 at most, of scores about 1) and
        # the latents' sums before the values' (another)
        assert np.linalg.norm(final.double().cpu().numpy() - want) <= 3 * 2 ** -8 * np.linalg.norm(want), step


def test_a_decode_loop_that_advances_itself(ops) -> None:
    """One captured graph raises the lengths, hands out blocks, stores and attends: every replay against the
    definition over what the cache then holds, with rows of padding and a request that the pool cannot serve."""
    heads, latent, block, width = 20, 512, 8, 6
    t = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(41)
    start = [5, 0, 8, 30]
    ids = torch.arange(1, 33, dtype=torch.int32)
    table = torch.zeros(4, width, dtype=torch.int32)
    taken = 0
    for b, length in enumerate(start):
        held = -(-length // block)
        table[b, :held] = ids[taken:taken + held]
        taken += held
    pool = BlockPool.in_place(ids[taken:taken + 4].to(DEV))  # 4 more blocks, and then none
    cache = torch.randn(34, block, latent + 64, generator=g, device=DEV).to(t)
    buffers = LatentBuffers(cache, latent)
    turn, scale = rotary(64, device=DEV), 192 ** -0.5
    bucket = ops.attention.graph_metadata(4, width, block, DEV)
    ops.attention.update_graph_metadata(bucket, torch.tensor(start, dtype=torch.int32), table)
    lengths = bucket.kv_lengths
    new = torch.randn(4, latent + 64, generator=g, device=DEV).to(t)
    q = torch.randn(4, heads, latent + 64, generator=g, device=DEV).to(t) * 0.4
    turned, out = q.clone(), torch.empty(4, heads, latent, dtype=t, device=DEV)

    def step():
        lengths.add_(lengths > 0)
        ops.attention.advance_graph_metadata(bucket, lengths, pool)
        ops.kvcache.store_latent(new[:, :latent], new[:, latent:], buffers, bucket, turn, q[:, :, latent:], turned[:, :, latent:])
        ops.attention.attend_latent(turned, buffers, bucket, out, scale=scale)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    served = set()
    for i in range(14):
        new.copy_(torch.randn(4, latent + 64, generator=g, device=DEV).to(t))
        before = lengths.tolist()
        graph.replay()
        torch.cuda.synchronize()
        now, held = lengths.tolist(), bucket.block_table.cpu().numpy()
        for b in range(4):
            assert now[b] in (0, before[b] + 1) and (before[b] or not now[b])
            if now[b]:
                slot = cache[int(held[b, (now[b] - 1) // block]), (now[b] - 1) % block]
                assert torch.equal(slot[:latent], new[b, :latent])
            served.add((b, bool(now[b])))
        want = oracle.attention(turned.double().cpu().numpy(), cache.double().cpu().numpy(), held, [1] * 4, now, scale, latent)[0]
        got = out.double().cpu().numpy()
        assert np.linalg.norm(got - want) <= 1.5 * 2 ** -8 * np.linalg.norm(want)  # a half step of the output, weights 2^-14
        assert not got[[b for b in range(4) if not now[b]]].any()
    assert (1, True) not in served and any((b, False) in served and (b, True) in served for b in (0, 2, 3))
