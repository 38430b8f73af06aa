"""The plan's part for 8-bit pools, apart from the plan itself (host planner only)."""

from __future__ import annotations

import numpy as np

from miniserve_b200 import _capi
from miniserve_b200.attention import (SeqChunk, _add_kv8, _plan_trees, _plan_with_kv8, plan_batch,
                                      plan_tree_batch, same_launch_shape)
from test_plan_update_cpu import _decode_batch, _info


def test_a_chunk_that_advances_by_whole_pages_keeps_the_shape() -> None:
    # A captured 128-token chunk walks through a preallocated table; a launch over a bf16 pool is the
    # same at every step.
    infos = [_info([SeqChunk(0, 128, 128 * i, list(range(90)))]) for i in range(1, 10)]
    assert all(same_launch_shape(infos[0], b) for b in infos[1:])


def test_the_part_for_8_bit_pools_can_be_added_later() -> None:
    """``_add_kv8`` gives what planning both together gives, for causal steps (with split rows, tensor-core
    items and a shared prefix) and for trees."""
    def table(lo: int, n: int) -> list[int]:
        return list(range(lo, lo + n))

    shared = [SeqChunk(i, 1, 400 + i, table(0, 20) + table(100 + 10 * i, 10)) for i in range(16)]
    batches = [
        [],
        _decode_batch([300, 1000, 77, 4000, 16, 2049]),
        [SeqChunk(0, 300, 512, table(0, 60)), SeqChunk(300, 1, 9000, table(60, 600)),
         SeqChunk(301, 40, 3, table(700, 3))],
        shared + [SeqChunk(16, 65, 0, table(300, 5))],
    ]
    for chunks in batches:
        tokens = sum(c.num_new for c in chunks)
        want, info, kv8 = _plan_with_kv8(chunks, tokens, 148, 0)
        packed, alone = plan_batch(chunks, tokens, 16, 148)
        got, more = _add_kv8(packed, alone, 148, 0)
        assert bytes(more) == bytes(kv8) and np.array_equal(got, want)
    for n in (5, 40):
        trees = [SeqChunk(i * n, n, 700 + i, table(60 * i, 60), parents=[-1] * n) for i in range(3)]
        want, info, kv8 = _plan_trees(trees, 3 * n, 148, 0, _capi.MsKv8Info())
        packed, alone = plan_tree_batch(trees, 3 * n)
        got, more = _add_kv8(packed, alone, 148, 0)
        assert bytes(more) == bytes(kv8) and np.array_equal(got, want)
