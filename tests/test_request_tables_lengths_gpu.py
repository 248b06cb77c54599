"""GPU tests of request_tables with lengths that no table holds: the call ends, and does what can be done."""

import numpy as np
import pytest
import torch

import prompt_oracle
from lightdelta_b200 import capi
from test_prompt_path_gpu import check_tables, ints, lib

pytestmark = pytest.mark.gpu
BLOCKS, LENGTHS = capi.LD_FAULT_TABLE_BLOCKS, capi.LD_FAULT_TABLE_LENGTHS


def call(query, context, block, width, n_tokens, n_free):
    n = len(query)
    table = torch.full((n, width), 9, dtype=torch.int32, device="cuda")
    cu, used = torch.empty(n + 1, dtype=torch.int32, device="cuda"), ints([0])
    pairs = torch.empty(n, 2, dtype=torch.int32, device="cuda")
    positions, slot_map = (torch.empty(n_tokens, dtype=torch.int64, device="cuda") for _ in range(2))
    free = torch.arange(100, 100 + n_free, dtype=torch.int32, device="cuda")
    start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    lib().request_tables(ints(query), ints(context), free, table, cu, positions, slot_map, pairs, used, block)
    stop.record()
    torch.cuda.synchronize()
    assert capi.fault_flags() == BLOCKS | LENGTHS
    return [t.cpu().numpy() for t in (table, cu, positions, slot_map, pairs, used)], start.elapsed_time(stop)


@pytest.mark.parametrize("n", [1, 40, 4096])
def test_lengths_at_their_largest(n):
    """2^31 - 1 tokens a request in blocks of one: 2^31 new blocks each, of which the rows have four.  The work is bounded by
    the tables, whatever the lengths say (the blocks of 4,096 such requests, counted one by one, would take a minute)."""
    far = 2 ** 31 - 1
    (table, cu, positions, slot_map, pairs, used), took = call([far] * n, [0] * n, 1, 4, 10, 6)
    assert took < 100.0
    # The first request's blocks take the whole free list, of which its row holds four; the others' rows get nothing.
    assert table[0].tolist() == [100, 101, 102, 103] and not table[1:].any()
    assert cu.tolist() == [0] + [far] * n and used.tolist() == [far]
    assert positions.tolist() == list(range(10)) and slot_map.tolist() == [100, 101, 102, 103] + [-1] * 6
    assert not pairs.any()


def test_held_blocks_stay_beside_lengths_that_do_not_fit():
    query, context = [3, 2 ** 31 - 1, 2], [2, 1, 0]
    (table, cu, _, slot_map, pairs, _), _ = call(query, context, 1, 5, 6, 4)
    assert table.tolist() == [[9, 9, 100, 101, 102], [9, 103, 0, 0, 0], [0, 0, 9, 9, 9]]
    assert cu.tolist() == [0, 3, 2 ** 31 - 1, 2 ** 31 - 1]
    assert slot_map.tolist() == [100, 101, 102, 103, -1, -1]
    assert pairs.tolist() == [[102, 9], [0, 9], [0, 0]]


@pytest.mark.parametrize("seed", range(4))
def test_more_blocks_than_entries(seed):
    """Requests of which some have many times their row's blocks, the others fit: against the definition."""
    rng = np.random.default_rng(seed)
    n = int(rng.choice([3, 50, 1500]))
    query = [int(q) for q in rng.integers(0, 12, n)]
    for r in rng.integers(0, n, max(n // 4, 1)):
        query[r] = int(rng.integers(200, 900))
    context = [int(c) for c in rng.integers(0, 10, n)]
    need = sum(-(-(c + q) // 4) - -(-c // 4) for q, c in zip(query, context))
    assert need > 6 * n
    check_tables(query, context, 4, 6, sum(query) // 2, int(rng.choice([need, need // 2])), seed=seed,
                 faults=BLOCKS | LENGTHS)
    assert prompt_oracle.tables(query, context, [1] * need, np.zeros((n, 6)), 0, 4)[5] == need
