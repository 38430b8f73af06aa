"""Rows that are moved below a sequence's cached length right before ``attend``."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200.attention import (SeqChunk, attend, build_attention_metadata, kv_gather,
                                      kv_scatter)
from miniserve_b200.kv_pool import KV8, allocate_kv_cache
from paged_reference import SCALE, U_BF16, assert_close, attention64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, KV8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("new", [1, 5, 20, 200])
def test_attend_sees_rows_moved_right_before_it(new: int, dtype, cuda_device) -> None:
    """Many rows are moved, and the next call attends over them: eagerly, and as a captured pair."""
    dev = cuda_device
    kvh, blocks, n = 4, 3000, 1024
    g = torch.Generator(device=dev).manual_seed(new)
    views = allocate_kv_cache(1, blocks, kvh, dev, dtype=dtype)[1][0]
    k, v = (torch.randn(blocks * 16, kvh, 128, device=dev, generator=g).bfloat16() for _ in range(2))
    kv_scatter(k, v, torch.arange(blocks * 16, device=dev), *views)
    table = torch.randperm(n // 16, generator=torch.Generator().manual_seed(1)).tolist()
    chunks, flat = [], 0
    for i in range(4):
        chunks.append(SeqChunk(flat, new, 40 + i, table[i * 16 : i * 16 + 16]))
        flat += new
    meta = build_attention_metadata(chunks, torch.zeros(flat, dtype=torch.int64, device=dev), 16)
    q = torch.randn(flat, 2 * kvh, 128, device=dev, generator=g).bfloat16()
    to = torch.arange(n, device=dev)
    source = [torch.randperm(blocks * 16 - n, device=dev, generator=g)[:n] + n for _ in range(4)]

    def step(src):
        kv_scatter(*kv_gather(src, *views), to, *views, moved=True)
        return attend(q, *views, meta, SCALE)

    outs = [step(src) for src in source for _ in range(5)]
    for i, src in enumerate(source):
        step(src)
        ref, bound, rows = attention64(q, *views, chunks, U_BF16)
        for out in outs[5 * i : 5 * i + 5]:
            assert_close(out, ref, bound, rows)
    src = source[0].clone()
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(src)
    for i in (1, 2, 0):
        src.copy_(source[i])
        graph.replay()
        assert torch.equal(out, outs[5 * i])
