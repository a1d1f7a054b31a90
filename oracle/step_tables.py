"""A step's blocks, positions and slots by their rule, request by request -- test infrastructure only.

The rule of ``include/ayaka_hip_tables.h`` in plain integers; its positions and slots are those of
the reference's plan (``python/ayaka/ops/backends/torch/attention.py:64-164``), which
``tests/test_tables_host.py`` checks against ``oracle.paged``.
"""

from __future__ import annotations

import numpy as np

__all__ = ["build"]


def build(rows, lengths, table: np.ndarray, free, taken: int, block: int, n_rows: int) -> dict[str, np.ndarray]:
    """The table, request_of_row, positions, slots, lengths and (taken, short) after the step."""
    table = np.array(table, dtype=np.int64)
    width = table.shape[1]
    request_of_row = np.zeros(n_rows, np.int64)
    positions, slots = np.zeros(n_rows, np.int64), np.zeros(n_rows, np.int64)
    served = np.zeros(len(lengths), np.int64)
    taken = min(max(int(taken), 0), len(free))
    asked, used, short, first = 0, taken, 0, 0
    for b, (count, length) in enumerate(zip(np.asarray(rows).tolist(), np.asarray(lengths).tolist())):
        row, first = first, first + max(count, 0)
        request_of_row[row:first] = b
        able = 0 <= count <= length and 0 < length <= width * block and first <= n_rows
        had = -(-(length - count) // block) if able else 0
        able = able and (had == 0 or table[b, had - 1] != 0)
        need = -(-length // block) - had if able else 0
        asked += need
        if not able or (need and asked > len(free) - taken):
            short += length != 0
            continue
        table[b, had:had + need] = free[taken + asked - need:taken + asked]
        if need:
            used = taken + asked
        served[b] = length
        for j in range(count):
            at = length - count + j
            positions[row + j] = at
            slots[row + j] = table[b, at // block] * block + at % block
    return {"table": table, "request_of_row": request_of_row, "positions": positions, "slots": slots,
            "lengths": served, "after": np.array([used, short])}
