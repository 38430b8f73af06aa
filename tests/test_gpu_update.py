"""``AttentionMetadata.update``: which new steps a captured step takes, over either kind of pool.

A launch over a bf16 pool reads nothing of the plan's part for 8-bit pools, so that part decides only
for metadata that an 8-bit call has used.
"""

from __future__ import annotations

import pytest
import torch

from miniserve_b200.attention import SeqChunk, attend, build_attention_metadata, kv_scatter
from miniserve_b200.kv_pool import KV8, allocate_kv_cache
from paged_reference import SCALE, U_BF16, assert_close, attention64

pytestmark = pytest.mark.gpu

KVH = 2
BLOCKS = 100


def pools(dev):
    """The same rows in a bf16 and in an 8-bit pool."""
    g = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.randn(BLOCKS * 16, KVH, 128, device=dev, generator=g).bfloat16() for _ in range(2))
    every = torch.arange(BLOCKS * 16, device=dev)
    out = []
    for dtype in (torch.bfloat16, KV8):
        views = allocate_kv_cache(1, BLOCKS, KVH, dev, dtype=dtype)[1][0]
        kv_scatter(k, v, every, *views)
        out.append(views)
    return out


def prefill(step: int, rows: int = 0) -> list[SeqChunk]:
    """A 128-token chunk that has advanced by whole pages through a preallocated table, beside decode
    rows."""
    chunks = [SeqChunk(0, 128, 128 * step, list(range(90)))]
    return chunks + [SeqChunk(128 + i, 1, 100 + i, list(range(90 - i, 97 - i))) for i in range(rows)]


def queries(dev, n: int) -> torch.Tensor:
    g = torch.Generator(device=dev).manual_seed(2)
    return torch.randn(n, 2 * KVH, 128, device=dev, generator=g).bfloat16()


def check(q, views, chunks, meta, out=None) -> None:
    got = attend(q, *views, meta, SCALE) if out is None else out
    ref, bound, covered = attention64(q, *views, chunks, U_BF16)
    assert_close(got, ref, bound, covered)


@pytest.mark.parametrize("rows", [0, 3])
def test_a_captured_chunk_advances_by_whole_pages(rows: int, cuda_device) -> None:
    """Every step of a chunk of fixed size is taken over a bf16 pool, whose launches do not change, and
    replays as it runs eagerly."""
    dev = cuda_device
    bf16, _ = pools(dev)
    q = queries(dev, 128 + rows)
    slots = torch.zeros(128 + rows, dtype=torch.int64, device=dev)
    meta = build_attention_metadata(prefill(1, rows), slots, 16)
    check(q, bf16, prefill(1, rows), meta)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(q, *bf16, meta, SCALE)
    for step in range(2, 10):
        assert meta.update(prefill(step, rows)), step
        graph.replay()
        fresh = build_attention_metadata(prefill(step, rows), slots, 16)
        assert torch.equal(out, attend(q, *bf16, fresh, SCALE))
        check(q, bf16, prefill(step, rows), meta, out)


def test_an_8_bit_call_after_an_update_of_another_shape(cuda_device) -> None:
    """The part for 8-bit pools belongs to the step that was planned last; once used, it decides too."""
    dev = cuda_device
    bf16, kv8 = pools(dev)
    q = queries(dev, 131)
    slots = torch.zeros(131, dtype=torch.int64, device=dev)
    meta = build_attention_metadata(prefill(1, 3), slots, 16)
    assert meta.update(prefill(2, 3)) and meta.update(prefill(3, 3))
    check(q, bf16, prefill(3, 3), meta)
    check(q, kv8, prefill(3, 3), meta)
    before = meta.plan.clone()
    assert not meta.update(prefill(4, 3))
    assert torch.equal(meta.plan, before)
    check(q, bf16, prefill(3, 3), meta)
    check(q, kv8, prefill(3, 3), meta)
    # Contexts that grow inside their last pages keep both launches; both parts follow.
    grown = [SeqChunk(c.flat_start, c.num_new, c.num_cached + (c.num_new == 1), c.block_table)
             for c in prefill(3, 3)]
    assert meta.update(grown)
    check(q, bf16, grown, meta)
    check(q, kv8, grown, meta)


def test_a_captured_8_bit_chunk_is_refused_another_page_count(cuda_device) -> None:
    dev = cuda_device
    _, kv8 = pools(dev)
    q = queries(dev, 128)
    slots = torch.zeros(128, dtype=torch.int64, device=dev)
    meta = build_attention_metadata(prefill(1), slots, 16)
    graph = torch.cuda.CUDAGraph()
    check(q, kv8, prefill(1), meta)
    torch.cuda.synchronize(dev)
    with torch.cuda.graph(graph):
        out = attend(q, *kv8, meta, SCALE)
    assert not meta.update(prefill(2))
    moved = [SeqChunk(0, 128, 128, list(range(89, -1, -1)))]
    assert meta.update(moved)
    graph.replay()
    check(q, kv8, moved, meta, out)


def test_trees_follow_the_same_rule(cuda_device) -> None:
    """Trees whose cached blocks are read by tensor-core items over a bf16 pool, and whole by kernel F over
    an 8-bit one: a cached length that changes the second's items only is taken until it has been used."""
    dev = cuda_device
    bf16, kv8 = pools(dev)
    parents = [-1] + [i // 2 for i in range(39)]
    q = queries(dev, 41)
    slots = torch.zeros(41, dtype=torch.int64, device=dev)

    def step(cached: int) -> list[SeqChunk]:
        return [SeqChunk(0, 40, cached, list(range(60)), parents=parents),
                SeqChunk(40, 1, 30, [70, 71])]

    meta = build_attention_metadata(step(800), slots, 16, pages_per_split=50)
    assert meta.tree.info.n_tc_items > 0
    check(q, bf16, step(800), meta)
    for cached in (801, 790, 780):
        assert meta.update(step(cached)), cached
        check(q, bf16, step(cached), meta)
    check(q, kv8, step(780), meta)
    check(q, bf16, step(780), meta)
    assert meta.update(step(781))
    check(q, kv8, step(781), meta)


@pytest.mark.parametrize("trees", [False, True])
def test_a_process_without_8_bit_pools_plans_none(trees: bool, cuda_device, monkeypatch) -> None:
    """Neither planned nor uploaded, nor added by an update; the first 8-bit call adds it, which a capture
    cannot."""
    from miniserve_b200 import kv_pool

    dev = cuda_device
    bf16, kv8 = pools(dev)
    monkeypatch.setattr(kv_pool, "_kv8_allocated", False)
    parents = [-1] + [i // 2 for i in range(39)]

    def step(i: int) -> list[SeqChunk]:
        if not trees:
            return prefill(i, 3)
        return [SeqChunk(0, 40, 780 + i, list(range(60)), parents=parents),
                SeqChunk(40, 1, 3000, [i % 7] * 188)]

    n = sum(c.num_new for c in step(1))
    q = queries(dev, n)
    slots = torch.zeros(n, dtype=torch.int64, device=dev)
    meta = build_attention_metadata(step(1), slots, 16)
    metas = [meta] if meta.tree is None else [meta, meta.tree]
    assert all(m.kv8 is None and m.plan.numel() == m.info.total_ints for m in metas)
    check(q, bf16, step(1), meta)
    assert meta.update(step(2)) and all(m.kv8 is None for m in metas)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before it is captured"):
        with torch.cuda.graph(graph):
            attend(q, *kv8, meta, SCALE)
    check(q, kv8, step(2), meta)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(q, *kv8, meta, SCALE)
    swapped = [SeqChunk(c.flat_start, c.num_new, c.num_cached, c.block_table[::-1], c.parents)
               for c in step(2)]
    assert meta.update(swapped)
    graph.replay()
    check(q, kv8, swapped, meta, out)
    check(q, bf16, swapped, meta)
