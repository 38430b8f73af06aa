"""A captured step over selected pages that is updated to steps whose longest row is shorter."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import (allocate_key_bounds, attend_pages, build_attention_metadata, kv_scatter,
                            select_pages, update_key_bounds, update_key_bounds_at)
from miniserve_b200.attention import SeqChunk
from miniserve_b200.kv_pool import KV8, allocate_kv_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, KV8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("pages,pairs", [(65, 1), (577, 1), (65, 40)])
def test_a_longest_row_that_gets_shorter_replays(pages: int, pairs: int, dtype, cuda_device) -> None:
    """Pairs of rows of n + 1 and n - 1 pages, then of n and n (the launches allow for 64 more), then as
    at first: the replay gives what calls with metadata of their own give."""
    dev, kvh = cuda_device, 4
    blocks = 2 * pages
    g = torch.Generator(device=dev).manual_seed(1)
    views = allocate_kv_cache(1, blocks, kvh, dev, dtype=dtype)[1][0]
    k, v = (torch.randn(blocks * 16, kvh, 128, device=dev, generator=g).bfloat16() for _ in range(2))
    kv_scatter(k, v, torch.arange(blocks * 16, device=dev), *views)
    bounds = allocate_key_bounds(1, blocks, kvh, dev)[1][0]
    update_key_bounds_at(*views, bounds, torch.arange(blocks, device=dev),
                         torch.full((blocks,), 16, device=dev))
    q = torch.randn(2 * pairs, 2 * kvh, 128, device=dev, generator=g).bfloat16()
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(2)).tolist()

    def chunks(first: int, second: int) -> list[SeqChunk]:
        """Every pair sees the same pages, its second row behind the first one's."""
        tables = (order[:first], order[first : first + second])
        return [SeqChunk(i, 1, 16 * len(tables[i % 2]) - 1 - i % 7, tables[i % 2]) for i in range(2 * pairs)]

    def metadata(first: int, second: int):
        return build_attention_metadata(chunks(first, second),
                                        torch.zeros(2 * pairs, dtype=torch.int64, device=dev), 16,
                                        pages_per_split=4096)

    def layer(meta):
        update_key_bounds(*views, bounds, meta)
        chosen = select_pages(q, bounds, meta, 11)
        return chosen, attend_pages(q, *views, meta, chosen, 128**-0.5)

    meta = metadata(pages, pages - 2)
    want = layer(meta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(meta)
    for first, second in ((pages - 1, pages - 1), (pages, pages - 2), (pages - 1, pages - 1)):
        assert meta.update(chunks(first, second))
        graph.replay()
        got = [x.clone() for x in out]
        want = layer(metadata(first, second))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        again = layer(meta)
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
