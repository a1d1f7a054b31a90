"""Step tables built on the device, word for word against the oracle, and decode buckets that advance
themselves."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, ForwardMode, KVLayoutKind
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import attention as hip_attention
from ayaka_amd.kvcache import RAW_CODEC, BlockPool, KVBuffers, StepTables, fp8_e4m3_block_codec
from oracle import step_tables

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


def dev(x, dtype=torch.int32) -> torch.Tensor:
    return torch.as_tensor(np.asarray(x)).to(device=DEV, dtype=dtype)


class Built:
    """One call of build_tables; outputs start poisoned."""

    def __init__(self, ops, rows, lengths, table, free, taken, block, n_rows, in_place=False) -> None:
        self.args = (rows, lengths, np.array(table), np.asarray(free), taken, block, n_rows)
        self.table = dev(table)
        lens = dev(lengths)
        self.tables = StepTables(dev(np.full(n_rows, -7)), dev(np.full(n_rows, -7)), dev(np.full(n_rows, -7), torch.int64),
                                 lens if in_place else dev(np.full(len(lengths), -7)))
        after = torch.zeros(4, dtype=torch.int32, device=DEV)
        if in_place:
            after[0] = taken
        self.pool = BlockPool(dev(free), after[:1] if in_place else dev([taken]), after)
        self.call = lambda: ops.kvcache.build_tables(dev(rows), lens, self.table, self.pool, self.tables, block)
        self.call()

    def check(self, label: str = "") -> None:
        want = step_tables.build(*self.args)
        t = self.tables
        for name, got in (("request_of_row", t.request_of_row), ("positions", t.positions), ("slots", t.slot_mapping),
                          ("lengths", t.kv_lengths), ("table", self.table), ("after", self.pool.after[:2])):
            assert np.array_equal(got.cpu().numpy(), want[name]), f"{label}: {name}"
        assert self.pool.after[2:].tolist() == [0, 0], label


def draw(rng, requests, most_rows, longest, block, lacking=0, spare=0):
    lengths = rng.integers(0, longest + 1, requests)
    rows = np.where(lengths > 0, np.minimum(rng.integers(0, most_rows + 1, requests), lengths), 1)
    width = -(-longest // block) + 1
    had = np.where(lengths > 0, -(-(lengths - rows) // block), 0)
    need = int((np.where(lengths > 0, -(-lengths // block), 0) - had).sum())
    ids = 1 + rng.permutation(int(had.sum()) + need + 50)
    table, at = np.full((requests, width), 777777), 0
    for b, n in enumerate(had):
        table[b, :n] = ids[at:at + n]
        at += n
    taken = int(rng.integers(0, 9))
    free = np.concatenate((np.full(taken, 888888), ids[at:at + max(need - lacking, 0) + (0 if lacking else 5)]))
    return rows, lengths, table, free, taken, block, int(rows.sum()) + spare


@pytest.mark.parametrize("block", [1, 5, 16, 128, 1000])
@pytest.mark.parametrize("requests", [1, 2, 63, 64, 65, 255, 257, 700])
def test_tables_are_the_oracles(ops, requests, block) -> None:
    rng = np.random.default_rng(requests * 1000 + block)
    for most_rows, longest, lacking, spare in ((1, 500, 0, 0), (30, 400, 0, 3), (200, 2000, 7, 300), (3, 90, 1000, 1)):
        case = draw(rng, requests, most_rows, longest, block, lacking, spare)
        for in_place in (False, True):
            Built(ops, *case, in_place=in_place).check(f"rows <= {most_rows}, in place {in_place}")


def test_many_rows_and_the_most_requests(ops) -> None:
    rng = np.random.default_rng(1)
    Built(ops, *draw(rng, 4096, 20, 600, 16)).check("4096 requests")
    Built(ops, *draw(rng, 40, 9000, 20000, 16, 0, 5000), in_place=True).check("long prompts")
    # more rows than one round of workgroups takes at a row per thread
    Built(ops, *draw(rng, 12, 30000, 40000, 64, 11, 1), in_place=True).check("longer ones, a pool that runs out")


def test_requests_that_cannot_be(ops) -> None:
    table = np.arange(1, 41).reshape(8, 5)
    rows = [2, -3, 5, 1, 1, 4, 0, 3]
    lengths = [9, 8, 4, 21, -5, 12, 6, 17]  # 1: rows < 0; 2: more rows than tokens; 3: over the table; 4: < 0
    for n_rows in (16, 13, 12, 3, 1, 20):  # fewer rows than the requests bring: the last do not fit
        Built(ops, rows, lengths, table, [90, 91, 92, 93], 0, 4, n_rows).check(f"{n_rows} rows")
    big = 2 ** 31 - 1
    Built(ops, [big, big, 1], [big, 3, 3], np.ones((3, 2), int), [5, 6], 0, 4, 8).check("rows past 32 bits")
    for taken in (-4, 3, 4, 5, 99):
        Built(ops, [1, 1], [5, 9], np.ones((2, 3), int), [50, 51, 52, 53], taken, 4, 2).check(f"taken {taken}")
    Built(ops, [1, 1], [3, 9], np.ones((2, 3), int), np.zeros(0, int), 0, 4, 2).check("no free list")
    Built(ops, [], [], np.zeros((0, 3), int), [4], 0, 4, 3).check("no requests")
    Built(ops, [1], [1], np.zeros((1, 0), int), [4], 0, 4, 1).check("a table of no columns")


def test_repeated_and_captured_calls(ops) -> None:
    rng = np.random.default_rng(8)
    built = Built(ops, *draw(rng, 300, 40, 900, 16, 3))
    for _ in range(3):
        built.call()
    built.check("repeated")
    graph = torch.cuda.CUDAGraph()
    lens = dev(built.args[1])
    rows = dev(built.args[0])
    with torch.cuda.graph(graph):
        ops.kvcache.build_tables(rows, lens, built.table, built.pool, built.tables, 16)
    for at in range(4):
        for t in built.tables:
            t.fill_(-7)
        built.table.copy_(dev(built.args[2]))
        torch.cuda.synchronize()
        graph.replay()
        built.check(f"replay {at}")


def test_a_pool_that_advances_through_steps(ops) -> None:
    # a pool in place of 7 blocks: steps draw 3, 2 and 2 of them, and the last finds none
    pool = BlockPool.in_place(dev(np.arange(1, 8)))
    table = torch.zeros(2, 8, dtype=torch.int32, device=DEV)
    host, taken = np.zeros((2, 8), np.int64), 0
    for rows, lengths in (([5, 1], [5, 1]), ([4, 4], [9, 5]), ([1, 9], [10, 14]), ([1, 9], [11, 23])):
        n = sum(rows)
        tables = StepTables(*(torch.empty(n, dtype=d, device=DEV) for d in (torch.int32, torch.int32, torch.int64)),
                            torch.empty(2, dtype=torch.int32, device=DEV))
        ops.kvcache.build_tables(dev(rows), dev(lengths), table, pool, tables, 4)
        want = step_tables.build(rows, lengths, host, np.arange(1, 8), taken, 4, n)
        host, taken = want["table"], int(want["after"][0])
        assert np.array_equal(table.cpu().numpy(), host)
        assert np.array_equal(tables.slot_mapping.cpu().numpy(), want["slots"])
        assert pool.after.tolist() == [taken, int(want["after"][1]), 0, 0]
    assert taken == 7 and pool.after[1] == 1


# --- decode buckets ---------------------------------------------------------------------------------


def staged_split(meta) -> tuple[int, list[tuple[int, int]], list[int]]:
    words = meta.plan.staged.cpu().numpy()
    n = meta.kv_lengths.shape[0]
    size, count = int(words[0]), int(words[1])
    items = words[2 + n:2 + n + 2 * count].reshape(-1, 2)
    return size, [tuple(i) for i in items.tolist()], words[2:2 + n].tolist()


def check_split(meta, lengths: np.ndarray) -> None:
    size, items, offsets = staged_split(meta)
    assert size % 64 == 0 and size >= meta.plan.min_size
    assert len(items) <= meta.plan.capacity
    parts = -(-lengths // size)
    assert parts.max(initial=0) <= meta.plan.partitions
    assert sorted(items) == [(r, p) for r, n in enumerate(parts) for p in range(max(int(n), 1))]
    assert offsets == (np.cumsum(parts) - parts).tolist()
    # longest first, to a 256th of the size; rows without context last
    left = [min(size, int(lengths[r]) - p * size) for r, p in items]
    assert all(b <= a + -(-size // 256) for a, b in zip(left, left[1:])), left


@pytest.mark.parametrize("requests,block,longest", [(1, 16, 4000), (3, 5, 100), (64, 16, 4096), (256, 32, 16384),
                                                    (600, 16, 900), (2048, 16, 700), (4096, 128, 300)])
def test_advancing_a_bucket(ops, requests, block, longest) -> None:
    rng = np.random.default_rng(requests)
    width = -(-longest // block) + 1
    meta = ops.attention.graph_metadata(requests, width, block, DEV)
    for shape in ([], [8, 4, 1], [2, 16, 2]):
        meta.plan.head_shape[:] = shape
        lengths = np.exp(rng.uniform(0, np.log(longest), requests)).astype(np.int64)
        lengths[rng.random(requests) < 0.1] = 0
        before = np.maximum(lengths - 1, 0)
        had = -(-before // block)
        ids = 1 + rng.permutation(int(had.sum()) + requests + 1)
        table, at = np.zeros((requests, width), np.int64), 0
        for b, n in enumerate(had):
            table[b, :n] = ids[at:at + n]
            at += n
        free = ids[at:]
        ops.attention.update_graph_metadata(meta, torch.from_numpy(before.astype(np.int32)),
                                            torch.from_numpy(table.astype(np.int32)))
        pool = BlockPool.in_place(dev(free))
        for _ in range(3):  # the call, its record, and the record again: the same inputs, the same outputs
            pool.after.zero_()
            meta.block_table.copy_(dev(table))
            ops.attention.advance_graph_metadata(meta, dev(lengths), pool)
        want = step_tables.build(np.ones(requests, int), lengths, table, free, 0, block, requests)
        for name, got in (("positions", meta.positions), ("slots", meta.slot_mapping), ("lengths", meta.kv_lengths),
                          ("table", meta.block_table), ("after", pool.after[:2])):
            assert np.array_equal(got.cpu().numpy(), want[name]), name
        assert np.array_equal(meta.request_of_row.cpu().numpy(), np.arange(requests))
        check_split(meta, want["lengths"])


def test_the_split_of_uneven_batches(ops) -> None:
    meta = ops.attention.graph_metadata(6, 4000, 16, DEV)
    pool = BlockPool.in_place(dev(np.arange(1, 100)))
    for lengths in ([64000, 1, 0, 64, 63, 65], [0] * 6, [1] * 6, [63999, 64000, 1000, 0, 12345, 320]):
        meta.block_table.fill_(1)
        pool.after.zero_()
        ops.attention.advance_graph_metadata(meta, dev(lengths), pool)
        assert meta.kv_lengths.tolist() == lengths
        check_split(meta, np.array(lengths))


def bucket_caches(codec: str, blocks: int, block: int, kv_heads: int, dim: int) -> KVBuffers:
    g = torch.Generator(device=DEV).manual_seed(3)
    shape = (blocks, block, kv_heads, dim)
    if codec == "block":
        k, v = (torch.randint(0, 0x78, shape, generator=g, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
                for _ in range(2))
        return KVBuffers(k, v, KVLayoutKind.NHD, fp8_e4m3_block_codec(torch.full((blocks, kv_heads, 2), 2.0 ** -8,
                                                                                 device=DEV)))
    return KVBuffers(*(torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)),
                     KVLayoutKind.NHD, RAW_CODEC)


@pytest.mark.parametrize("codec", ["raw", "block"])
def test_a_captured_step_that_advances_itself(ops, codec) -> None:
    # lengths raised, the bucket advanced, two layers written and read, all in one graph that the
    # host replays without a word; against the same steps planned eagerly on the host
    rng = np.random.default_rng(5)
    heads, kv_heads, dim, block, width = 8, 2, 64, 16, 40
    lengths = np.array([15, 300, 0, 64, 1])
    n = len(lengths)
    blocks = 200
    ours, theirs = (bucket_caches(codec, blocks, block, kv_heads, dim) for _ in range(2))
    ids = 1 + rng.permutation(blocks - 1)
    had = -(-lengths // block)
    table, at = np.zeros((n, width), np.int64), 0
    for b, count in enumerate(had):
        table[b, :count] = ids[at:at + count]
        at += count
    free = ids[at:at + 5]  # runs out within the run
    meta = ops.attention.graph_metadata(n, width, block, DEV)
    ops.attention.update_graph_metadata(meta, torch.from_numpy(lengths.astype(np.int32)),
                                        torch.from_numpy(table.astype(np.int32)))
    pool = BlockPool.in_place(dev(free))
    live = dev((lengths > 0).astype(np.int64))
    k, v = (torch.zeros(n, kv_heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(n, heads, dim, dtype=torch.bfloat16, device=DEV)
    out = torch.empty_like(q)
    ops.attention.attend(q, ours, meta, out, scale=0.125)  # the scratch, and the bucket's head shape
    goal = meta.kv_lengths.clone()

    def step():
        goal.add_(live)
        ops.attention.advance_graph_metadata(meta, goal, pool)
        ops.kvcache.store(k, v, ours, meta)
        ops.attention.attend(q, ours, meta, out, scale=0.125)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    goals, taken = lengths.copy(), 0
    for at in range(40):
        for x in (k, v, q):
            x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        goals = goals + (lengths > 0)
        want = step_tables.build(np.ones(n, int), goals, table, free, taken, block, n)
        table, taken = want["table"], int(want["after"][0])
        planned = ops.attention.plan(ForwardMode.DECODE, dev(np.ones(n, int)), dev(want["lengths"]), dev(table), block)
        eager = torch.empty_like(q)
        ops.kvcache.store(k, v, theirs, planned)
        ops.attention.attend(q, theirs, planned, eager, scale=0.125)
        torch.cuda.synchronize()
        assert np.array_equal(meta.block_table.cpu().numpy(), table), at
        assert pool.after.tolist() == [taken, int(want["after"][1]), 0, 0], at
        assert torch.equal(meta.slot_mapping, planned.slot_mapping), at
        for a, b in ((ours.k, theirs.k), (ours.v, theirs.v)):  # block 0 takes a raw cache's padding rows, in any order
            assert torch.equal(a[1:].view(torch.uint8), b[1:].view(torch.uint8)), at
        # the split may be another: each output within its roundings (bf16 half a step, the weights'
        # fp16 half a step or the split bf16's 2^-14)
        size = eager.float().abs().amax(-1, keepdim=True)
        assert ((out.float() - eager.float()).abs() <= 2 * (2.0 ** -8 + 2.0 ** -10) * size + 1e-30).all(), at
        assert not out[torch.from_numpy(want["lengths"] == 0).to(DEV)].any(), at
    assert int(want["after"][1]) > 0  # the pool did run out


def test_a_bucket_that_raises_its_own_lengths(ops) -> None:
    # kv_lengths is the bucket's own: a request that the pool cannot serve stays padding from there on
    block, n = 4, 3
    meta = ops.attention.graph_metadata(n, 6, block, DEV)
    table = np.zeros((n, 6), np.int32)
    table[0, 0], table[1, 0] = 7, 8
    ops.attention.update_graph_metadata(meta, torch.tensor([3, 2, 0], dtype=torch.int32), torch.from_numpy(table))
    pool = BlockPool.in_place(dev([20, 21]))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        meta.kv_lengths.add_(meta.kv_lengths > 0)
        ops.attention.advance_graph_metadata(meta, meta.kv_lengths, pool)
    # request 0 takes block 20 at length 5, request 1 block 21 at length 5, and 0 finds none at 9
    for at in range(9):
        graph.replay()
        lengths = [4 + at if at < 5 else 0, 3 + at if at < 6 else 0, 0]
        assert meta.kv_lengths.tolist() == lengths, at
        assert pool.after.tolist() == [(at >= 1) + (at >= 2), int(at in (5, 6)), 0, 0], at
    assert meta.block_table.tolist() == [[7, 20, 0, 0, 0, 0], [8, 21, 0, 0, 0, 0], [0] * 6]


def test_a_request_left_without_its_block_stays_out(ops) -> None:
    # its length is raised although the step before could not serve it
    Built(ops, [1, 1, 1], [6, 6, 9], np.array([[3, 0, 0], [3, 4, 0], [5, 6, 0]]), [30, 31], 0, 4, 3).check()


def test_a_bucket_of_one_partition_per_row(ops) -> None:
    # a table of one partition runs the single-pass kernel: the staged split is written and not read
    heads, kv_heads, dim, block = 4, 2, 64, 16
    buffers = bucket_caches("block", 20, block, kv_heads, dim)
    meta = ops.attention.graph_metadata(3, 3, block, DEV)
    assert meta.plan.partitions == 1
    table = np.array([[1, 2, 0], [3, 0, 0], [0, 0, 0]])
    ops.attention.update_graph_metadata(meta, torch.tensor([20, 16, 0], dtype=torch.int32),
                                        torch.from_numpy(table.astype(np.int32)))
    lengths = np.array([21, 17, 1])
    ops.attention.advance_graph_metadata(meta, dev(lengths), BlockPool.in_place(dev([9, 10])))
    check_split(meta, lengths)
    q = torch.randn(3, heads, dim, device=DEV).to(torch.bfloat16)
    out, eager = torch.empty_like(q), torch.empty_like(q)
    ops.attention.attend(q, buffers, meta, out, scale=0.125)
    planned = ops.attention.plan(ForwardMode.DECODE, dev([1, 1, 1]), dev(lengths), meta.block_table, block)
    hip_attention.attend_with(q, buffers, planned, eager, scale=0.125, partitions=0)
    assert torch.equal(out, eager)


def test_attend_keeps_the_device_split(ops) -> None:
    # a first attend whose head shape the host had not guessed stages the host's split again, but
    # not over one that the device has made since
    heads, kv_heads, dim, block, width = 32, 2, 64, 16, 100
    buffers = bucket_caches("raw", 300, block, kv_heads, dim)
    meta = ops.attention.graph_metadata(2, width, block, DEV)
    table = np.arange(1, 1 + 2 * width).reshape(2, width)
    ops.attention.update_graph_metadata(meta, torch.tensor([100, 200], dtype=torch.int32),
                                        torch.from_numpy(table.astype(np.int32)))
    lengths = np.array([1500, 1600])
    ops.attention.advance_graph_metadata(meta, dev(lengths), BlockPool.in_place(dev(np.arange(250, 260))))
    q = torch.randn(2, heads, dim, device=DEV).to(torch.bfloat16)
    out = torch.empty_like(q)
    ops.attention.attend(q, buffers, meta, out, scale=0.125)
    torch.cuda.synchronize()
    check_split(meta, lengths)


def test_refusals(ops) -> None:
    i32 = dict(dtype=torch.int32, device=DEV)
    table, pool = torch.zeros(2, 3, **i32), BlockPool.in_place(torch.ones(4, **i32))
    tables = StepTables(torch.zeros(2, **i32), torch.zeros(2, **i32), torch.zeros(2, dtype=torch.int64, device=DEV),
                        torch.zeros(2, **i32))
    ones = torch.ones(2, **i32)
    build = ops.kvcache.build_tables
    with pytest.raises(BackendError, match=r"rows_per_request must be int32 \[2\], got int64"):
        build(ones.long(), ones, table, pool, tables, 4)
    with pytest.raises(BackendError, match=r"block_table must be int32 \[2, 3\], got int32 \[1, 3\]"):
        build(ones, ones, table[:1], pool, tables, 4)
    with pytest.raises(BackendError, match="block_table must be contiguous"):
        build(ones, ones, torch.zeros(2, 6, **i32)[:, ::2], pool, tables, 4)
    with pytest.raises(BackendError, match=r"tables.slot_mapping must be int64 \[2\]"):
        build(ones, ones, table, pool, tables._replace(slot_mapping=ones), 4)
    with pytest.raises(BackendError, match=r"pool.after must be int32 \[4\]"):
        build(ones, ones, table, pool._replace(after=ones), tables, 4)
    with pytest.raises(BackendError, match="pool.free is on cpu, the table is on cuda:0"):
        build(ones, ones, table, pool._replace(free=torch.ones(4, dtype=torch.int32)), tables, 4)
    with pytest.raises(BackendError, match="block_size 0"):
        build(ones, ones, table, pool, tables, 0)
    meta = ops.attention.graph_metadata(2, 3, 4, DEV)
    with pytest.raises(BackendError, match=r"kv_lengths must be int32 \[2\]"):
        ops.attention.advance_graph_metadata(meta, torch.ones(3, **i32), pool)
    with pytest.raises(BackendError, match="kv_lengths is on cpu"):
        ops.attention.advance_graph_metadata(meta, ones.cpu(), pool)
