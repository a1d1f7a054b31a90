"""The step tables built on the device, as far as the CPU goes: the oracle's rule and the refusals."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np
import pytest
import torch

from ayaka_amd.enums import ForwardMode
from ayaka_amd.errors import BackendError
from ayaka_amd.hip import _lib
from ayaka_amd.hip import attention as hip_attention
from ayaka_amd.hip import kvcache as hip_kvcache
from ayaka_amd.kvcache import BlockPool, StepTables
from oracle import step_tables

HEADER = Path(__file__).resolve().parent.parent / "include" / "ayaka_hip_tables.h"


def test_every_declared_function_is_exported_and_bound() -> None:
    names = re.findall(r"\b(ayk_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S))
    assert sorted(names) == sorted(_lib.TABLES_EXPORTS)


def test_the_oracle_derives_what_plan_derives() -> None:
    rng = np.random.default_rng(0)
    for block in (1, 5, 16):
        rows, lengths = [3, 1, 9, 1], [10, 40, 9, 0]
        before = [n - r if n else 0 for r, n in zip(rows, lengths)]
        ids = iter(1 + rng.permutation(300))
        table = np.zeros((4, 40), np.int64)
        for b, n in enumerate(before):
            for i in range(-(-n // block)):
                table[b, i] = next(ids)
        free = [next(ids) for _ in range(60)]
        got = step_tables.build(rows, lengths, table, free, 0, block, sum(rows))
        meta = hip_attention.plan(ForwardMode.MIXED, torch.tensor(rows), torch.tensor(lengths),
                                  torch.from_numpy(got["table"]), block)
        for name, tensor in (("request_of_row", meta.request_of_row), ("positions", meta.positions),
                             ("slots", meta.slot_mapping), ("lengths", meta.kv_lengths)):
            assert np.array_equal(got[name], tensor.numpy()), name
        assert got["after"].tolist() == [sum(-(-n // block) + -(n and (n - r + block - 1) // block)
                                             for r, n in zip(rows, lengths) if n), 0]


def test_the_oracle_serves_in_order_until_the_pool_runs_out() -> None:
    table = np.zeros((4, 3), np.int64)
    table[3, 0] = 9
    # 2 blocks, 2 blocks (one too many of 3), none needed, 1 block: the third is served, the last is not
    got = step_tables.build([8, 7, 1, 2], [8, 7, 2, 5], np.array([[0, 0, 0], [0, 0, 0], [4, 0, 0], [9, 0, 0]]),
                            [21, 22, 23], 0, 4, 18)
    assert got["table"].tolist() == [[21, 22, 0], [0, 0, 0], [4, 0, 0], [9, 0, 0]]
    assert got["lengths"].tolist() == [8, 0, 2, 0] and got["after"].tolist() == [2, 2]
    assert got["slots"][:8].tolist() == [84, 85, 86, 87, 88, 89, 90, 91] and got["slots"][15] == 17


def _pool(n: int = 4) -> BlockPool:
    return BlockPool.in_place(torch.arange(1, 1 + n, dtype=torch.int32))


def test_a_pool_in_place_counts_in_its_own_state() -> None:
    pool = _pool()
    assert pool.after.tolist() == [0, 0, 0, 0] and pool.taken.data_ptr() == pool.after.data_ptr()


def test_host_tensors_are_refused() -> None:
    i32 = dict(dtype=torch.int32)
    tables = StepTables(torch.zeros(2, **i32), torch.zeros(2, **i32), torch.zeros(2, dtype=torch.int64),
                        torch.zeros(1, **i32))
    with pytest.raises(BackendError, match="runs on a HIP device"):
        hip_kvcache.build_tables(torch.ones(1, **i32), torch.ones(1, **i32), torch.zeros(1, 2, **i32), _pool(), tables, 4)
    meta = hip_attention.graph_metadata(2, 4, 16, torch.device("cpu"))
    with pytest.raises(BackendError, match="runs on a HIP device"):
        hip_attention.advance_graph_metadata(meta, torch.zeros(2, **i32), _pool())
    planned = hip_attention.plan(ForwardMode.DECODE, torch.tensor([1]), torch.tensor([3]), torch.tensor([[1]]), 4)
    with pytest.raises(BackendError, match="not made by this backend's graph_metadata"):
        hip_attention.advance_graph_metadata(planned, torch.zeros(1, **i32), _pool())


def _build(**kw: object) -> int:
    args = dict(rows=1, lengths=1, n_requests=2, table=1, stride=4, max_blocks=4, free=1, n_free=3, taken=1, after=1,
                block_size=16, ror=1, positions=1, slots=1, n_rows=5, kv_lengths=1, stream=None)
    args.update(kw)
    return _lib.lib().ayk_build_tables(*args.values())


@pytest.mark.parametrize("changes,code,message", [
    ({"n_requests": -1}, 1, b"-1 requests"),
    ({"n_requests": 4097}, 2, b"4097 requests exceed 4096"),
    ({"n_rows": -1}, 1, b"-1 rows"),
    ({"n_free": -1}, 1, b"-1 free blocks"),
    ({"block_size": 0}, 2, b"block_size 0"),
    ({"block_size": 65537}, 2, b"block_size 65537"),
    ({"stride": 3}, 1, b"table_stride 3"),
    ({"max_blocks": 1 << 16, "stride": 1 << 16, "block_size": 1 << 15}, 2, b"positions per row"),
    ({"rows": None}, 1, b"null"),
    ({"lengths": None}, 1, b"null"),
    ({"table": None}, 1, b"null"),
    ({"free": None}, 1, b"null"),
    ({"taken": None}, 1, b"null"),
    ({"after": None}, 1, b"null"),
    ({"ror": None}, 1, b"null"),
    ({"slots": None}, 1, b"null"),
    ({"kv_lengths": None}, 1, b"null"),
])
def test_the_library_refuses_bad_tables(changes: dict, code: int, message: bytes) -> None:
    assert _build(**changes) == code
    assert message in _lib.lib().ayk_last_error()


def _advance(sizes=(64, 128), **kw: object) -> int:
    host = np.asarray(sizes, dtype=np.int32)
    args = dict(lengths=1, n_requests=2, table=1, stride=4, max_blocks=4, free=1, n_free=3, taken=1, after=1,
                block_size=16, positions=1, slots=1, kv_lengths=1, staged=1, capacity=8, sizes=host.ctypes.data,
                n_sizes=host.size, groups=1, cost=160, compute_units=256, stream=None)
    args.update(kw)
    return _lib.lib().ayk_advance_decode_tables(*args.values())


@pytest.mark.parametrize("changes,code,message", [
    ({"staged": None}, 1, b"null"),
    ({"capacity": 1}, 1, b"1 items holds no partition of each of 2 rows"),
    ({"capacity": (1 << 18) + 1}, 2, b"262145 items exceeds 262144"),
    ({"sizes": (64, 64)}, 1, b"size 1, 64"),
    ({"sizes": (100,)}, 1, b"size 0, 100"),
    ({"sizes": (64, (1 << 30) + 64)}, 1, b"up to 2^30"),
    ({"sizes": tuple(range(64, 64 * 34, 64))}, 1, b"33 sizes"),
    ({"groups": 0}, 1, b"0 groups"),
    ({"cost": -1}, 1, b"cost -1"),
    ({"compute_units": 0}, 1, b"0 compute units"),
    ({"n_requests": 5000, "capacity": 5000}, 2, b"5000 requests exceed"),
])
def test_the_library_refuses_bad_advances(changes: dict, code: int, message: bytes) -> None:
    assert _advance(**changes) == code
    assert message in _lib.lib().ayk_last_error()


def test_a_refused_advance_leaves_the_hosts_split() -> None:
    # the split that the last update staged is still the bucket's: a first attend of another head shape
    # stages it again for that shape
    meta = hip_attention.graph_metadata(2, 64, 16, torch.device("cpu"))
    hip_attention.update_graph_metadata(meta, torch.tensor([900, 40], dtype=torch.int32),
                                        torch.arange(1, 129, dtype=torch.int32).view(2, 64))
    staged = list(meta.plan.staged_shape)
    assert staged
    with pytest.raises(BackendError):
        hip_attention.advance_graph_metadata(meta, torch.zeros(2, dtype=torch.int32), _pool())
    assert meta.plan.staged_shape == staged
