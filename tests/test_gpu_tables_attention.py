"""From tables built on the device to attention: the blocks and slots of ``build_tables`` written and
read through a plan made of its lengths and block table, against the same steps planned on the host."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ayaka_amd.attention import AttentionMetadata
from ayaka_amd.backend import load_backend
from ayaka_amd.enums import DType, ForwardMode
from ayaka_amd.errors import BackendError
from ayaka_amd.kvcache import BlockPool, StepTables
from oracle import step_tables
from tests.test_gpu_tables import bucket_caches, dev

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops():
    return load_backend(["hip"], device="cuda", dtype=DType.BF16)


@pytest.mark.parametrize("codec", ["raw", "block"])
def test_built_tables_through_store_and_attend(ops, codec) -> None:
    # prompts, chunks, single tokens and a request the pool cannot serve (several rows, then again): the
    # rows go into the cache through the tables' own slots, the attention over a plan of the tables'
    # lengths; every output equals the host-planned step's bit for bit, an unserved request's rows are zeros
    rng = np.random.default_rng(2)
    heads, kv_heads, dim, block, width, n = 8, 2, 64, 16, 30, 4
    blocks = 60
    ours, theirs = (bucket_caches(codec, blocks, block, kv_heads, dim) for _ in range(2))
    free = 1 + rng.permutation(blocks - 1)[:14]
    pool = BlockPool.in_place(dev(free))
    table = torch.zeros(n, width, dtype=torch.int32, device=DEV)
    host, taken = np.zeros((n, width), np.int64), 0
    held = np.zeros(n, np.int64)
    short = 0
    for rows in ([40, 1, 100, 17], [1, 1, 20, 4], [2, 30, 40, 1], [3, 3, 90, 5], [1, 1, 1, 1]):
        rows = np.array(rows)
        lengths = held + rows
        total = int(rows.sum())
        tables = StepTables(*(torch.full((total,), -7, dtype=d, device=DEV)
                              for d in (torch.int32, torch.int32, torch.int64)), dev(np.full(n, -7)))
        ops.kvcache.build_tables(dev(rows), dev(lengths), table, pool, tables, block)
        want = step_tables.build(rows, lengths, host, free, taken, block, total)
        host, taken, short = want["table"], int(want["after"][0]), short + int(want["after"][1])
        held = np.where(want["lengths"] > 0, lengths, held)  # an unserved request stays as it was
        k, v = (torch.from_numpy(rng.standard_normal((total, kv_heads, dim)).astype(np.float32)).to(DEV, torch.bfloat16)
                for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((total, heads, dim)).astype(np.float32)).to(DEV, torch.bfloat16)

        # the write needs the slots alone; attention a plan, which reads the lengths and the table
        step = AttentionMetadata(mode=ForwardMode.MIXED, block_size=block, rows_per_request=dev(rows),
                                 request_of_row=tables.request_of_row, positions=tables.positions,
                                 slot_mapping=tables.slot_mapping, kv_lengths=tables.kv_lengths, block_table=table,
                                 plan=None)
        ops.kvcache.store(k, v, ours, step)
        out = torch.full_like(q, float("nan"))
        with pytest.raises(BackendError, match="plan it with the same ops"):
            ops.attention.attend(q, ours, step, out, scale=0.125)
        planned = ops.attention.plan(ForwardMode.MIXED, dev(rows), tables.kv_lengths, table, block)
        assert torch.equal(planned.positions, tables.positions)
        assert torch.equal(planned.slot_mapping, tables.slot_mapping)
        assert torch.equal(planned.request_of_row, tables.request_of_row)
        ops.attention.attend(q, ours, planned, out, scale=0.125)

        by_host = ops.attention.plan(ForwardMode.MIXED, dev(rows), dev(want["lengths"]), dev(host), block)
        eager = torch.full_like(q, float("nan"))
        ops.kvcache.store(k, v, theirs, by_host)
        ops.attention.attend(q, theirs, by_host, eager, scale=0.125)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        unserved = np.repeat(want["lengths"] == 0, rows)
        assert not out[torch.from_numpy(unserved).to(DEV)].any() and not out.isnan().any()
        for a, b in ((ours.k, theirs.k), (ours.v, theirs.v)):  # (block 0 takes a raw cache's unserved rows)
            assert torch.equal(a[1:].view(torch.uint8), b[1:].view(torch.uint8))
        if codec == "block":
            assert torch.equal(ours.codec.scales, theirs.codec.scales)
    assert short > 1
