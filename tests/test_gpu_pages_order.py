"""Attention right behind a call that writes whole pages below the cached length."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import attend, build_attention_metadata, clear_pages, kv_scatter
from miniserve_b200.attention import SeqChunk
from miniserve_b200.kv_pool import KV8, allocate_kv_cache
from paged_reference import SCALE, U_BF16, U_F16, assert_close, attention64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, KV8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("new", [1, 5, 20, 200])
@pytest.mark.parametrize("layers", [1, 4])
def test_attend_sees_pages_cleared_right_before_it(layers: int, new: int, dtype, cuda_device) -> None:
    """Half the pages of every table held infinities and are cleared, and the next call attends over them: as
    over zeros, eagerly and as a captured pair."""
    dev = cuda_device
    kvh, blocks = 4, 3000
    g = torch.Generator(device=dev).manual_seed(new)
    pool, views = allocate_kv_cache(layers, blocks, kvh, dev, dtype=dtype)
    for view in views:
        k, v = (torch.randn(blocks * 16, kvh, 128, device=dev, generator=g).bfloat16() for _ in range(2))
        kv_scatter(k, v, torch.arange(blocks * 16, device=dev), *view)
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).tolist()
    chunks, flat, gone = [], 0, order[240:]
    for i in range(4):
        table = order[i * 60 : i * 60 + 60]
        chunks.append(SeqChunk(flat, new, 700 + i, table))
        flat += new
        gone = gone + table[0:43:2]  # pages below the cached length, the last ones of the list
    meta = build_attention_metadata(chunks, torch.zeros(flat, dtype=torch.int64, device=dev), 16)
    q = torch.randn(flat, 2 * kvh, 128, device=dev, generator=g).bfloat16()
    junk = torch.full((len(gone) * 16, kvh, 128), torch.inf, dtype=torch.bfloat16, device=dev)
    at = (torch.tensor(gone, device=dev)[:, None] * 16 + torch.arange(16, device=dev)).flatten()
    for view in views:
        kv_scatter(junk, junk, at, *view)
    before = pool.clone()

    def step() -> torch.Tensor:
        clear_pages(pool, gone)
        return attend(q, *views[-1], meta, SCALE)

    got = []
    for _ in range(5):
        pool.view(torch.uint8).copy_(before.view(torch.uint8))
        got.append(step())
    # Chunks of more than 64 tokens have bf16 weights over either pool.
    u = U_BF16 if dtype == torch.bfloat16 or new > 64 else U_F16
    ref, bound, rows = attention64(q, *views[-1], chunks, u)
    for out in got:
        assert_close(out, ref, bound, rows)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(5):
        pool.view(torch.uint8).copy_(before.view(torch.uint8))
        graph.replay()
        assert torch.equal(out, got[0])
