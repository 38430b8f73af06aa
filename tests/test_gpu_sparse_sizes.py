"""Attention over selected pages where queries and keys lie at opposite ends of the range: scores are ordinary
numbers, whatever the sizes of their factors."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import attend_pages, build_attention_metadata, kv_scatter
from miniserve_b200.attention import SeqChunk
from miniserve_b200.kv_pool import KV8, allocate_kv_cache, layer_as_slots
from paged_reference import assert_close
from sparse_reference import SCALE, attend_pages64

pytestmark = pytest.mark.gpu

POOLS = pytest.mark.parametrize("dtype", [torch.bfloat16, KV8], ids=["bf16", "e4m3"])
CHUNKS = [SeqChunk(0, 1, 300, list(range(19))), SeqChunk(1, 3, 90, list(range(19, 25)))]
KVH, BLOCKS = 2, 30


def queries(exponent: int, dev) -> torch.Tensor:
    """[4, 4, 128] of magnitudes up to 2^exponent."""
    g = torch.Generator(device=dev).manual_seed(exponent)
    x = torch.rand(4, 2 * KVH, 128, device=dev, generator=g, dtype=torch.float64) * 2 - 1
    return (x * 0.99 * 2.0**exponent).bfloat16()


def pool(k: torch.Tensor, dtype, dev):
    g = torch.Generator(device=dev).manual_seed(1)
    v = torch.randn(k.shape, device=dev, generator=g).bfloat16()
    views = allocate_kv_cache(1, BLOCKS, KVH, dev, dtype=dtype)[1][0]
    kv_scatter(k, v, torch.arange(BLOCKS * 16, device=dev), *views)
    return views


def metadata(dev):
    return build_attention_metadata(CHUNKS, torch.zeros(4, dtype=torch.int64, device=dev), 16)


@POOLS
@pytest.mark.parametrize("exponent", [-110, -60, 90, 112, 113, 116, 127, 128])
def test_queries_of_any_size(exponent: int, dtype, cuda_device) -> None:
    """Keys (some of their channels zero) as small as the queries are large, or the other way round; the scale
    makes the scores some units wide."""
    dev = cuda_device
    size = -90 if exponent > 0 else 90
    g = torch.Generator(device=dev).manual_seed(2)
    k = torch.randn(BLOCKS * 16, KVH, 128, device=dev, generator=g)
    k *= torch.rand(k.shape, device=dev, generator=g) < 0.7
    views = pool((k * 2.0**size).bfloat16(), dtype, dev)
    q = queries(exponent, dev)
    pages = torch.arange(19, dtype=torch.int32, device=dev).repeat(4, KVH, 1)
    scale = 2.0 ** -(size + exponent)
    out = attend_pages(q, *views, metadata(dev), pages, scale)
    ref, bound, rows = attend_pages64(q, *views, CHUNKS, pages, scale)
    assert bool(torch.isfinite(out[rows]).all())
    assert_close(out, ref, bound, rows)


@POOLS
@pytest.mark.parametrize("scale", [SCALE, 1.0, 2.0**20])
@pytest.mark.parametrize("exponent", [100, 115, 128])
def test_one_key_has_all_the_weight(exponent: int, scale: float, dtype, cuda_device) -> None:
    """Every key but one is zero, and that one's scores are far above 0: the rows are its values, exactly."""
    dev = cuda_device
    q = queries(exponent, dev)
    k = torch.zeros(BLOCKS * 16, KVH, 128, dtype=torch.bfloat16, device=dev)
    at = [17, 19 * 16 + 40]  # one in each sequence, for the first head of the pair
    for slot, row in zip(at, (0, 1)):
        k[slot] = q[row, ::2].sign() * 2.0**-90
    views = pool(k, dtype, dev)
    pages = torch.arange(19, dtype=torch.int32, device=dev).repeat(4, KVH, 1)
    out = attend_pages(q, *views, metadata(dev), pages, scale)
    v = layer_as_slots(views[1])
    for slot, row in zip(at, (0, 1)):
        assert torch.equal(out[row, ::2], v[slot])
