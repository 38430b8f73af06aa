"""The weights of attention over selected pages where the outputs cancel: what their rounding adds shows there.

A weight is held as two bf16 numbers over a bf16 pool (the first loses at most 2^-8 of it, the second 2^-9 of that, and
both are relative to a power of two at most the weight: 2^-17 in all) and as two f16 numbers over an 8-bit one (2^-11,
then 2^-12: 2^-22 is kept as the bound), so that

    |out - exact| <= 2^-8 |out| + A (u + 2 d + n 2^-23 + 2^-20) + n 2^-36 M + n 2^-124,      A = sum_j w_j |v_j|,

with u = 2^-17 or 2^-22; 2^-8: half a bf16 step; d the largest error of a score: 2^-16 of the sum of the magnitudes of
its products, fp32 sums that drop low bits, and 2^-22 of itself, from the exponent's argument (it enters the weights and
their sum, hence twice); n 2^-23: sums of n terms in fp32; 2^-20: ex2.approx and the merge of partial results.  8-bit
pools: f16 ends at 2^-24, and the second number is held 2^12 larger, so that each of n shares may lose 2^-37 of 2^(s + e)
of the row's largest one, M = max_j w_j max|v_j|, whose codes are at least half as large as the largest code; bf16
pools have no such term.  bf16: weights are held 2^-24 smaller, and products below 2^-126 may lose up to 2^-149, which is
2^-125 of the output (8-bit pools: far less).
"""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import attend_pages, build_attention_metadata, kv_scatter
from miniserve_b200.attention import SeqChunk
from miniserve_b200.kv_pool import KV8, allocate_kv_cache, layer_as_slots

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, KV8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("pages", [1, 3, 40])
@pytest.mark.parametrize("width", [2.0**-7, 2.0**-5, 0.5])
def test_values_that_cancel(width: float, pages: int, dtype, cuda_device) -> None:
    """Scores of that width around 0, and every key beside one of nearly the same score and the opposite value."""
    dev, kvh, rows = cuda_device, 3, 8
    g = torch.Generator(device=dev).manual_seed(pages)
    k = torch.randn(pages * 8, kvh, 1, 128, device=dev, generator=g).repeat(1, 1, 2, 1)
    k[:, :, 1] += 0.1 * torch.randn(k[:, :, 1].shape, device=dev, generator=g)
    v = torch.randn(pages * 8, kvh, 1, 128, device=dev, generator=g).repeat(1, 1, 2, 1)
    v[:, :, 1] *= -1
    k, v = (x.transpose(1, 2).flatten(0, 1).bfloat16() for x in (k, v))  # pairs of neighbouring tokens
    views = allocate_kv_cache(1, pages, kvh, dev, dtype=dtype)[1][0]
    kv_scatter(k, v, torch.arange(16 * pages, device=dev), *views)
    q = (torch.randn(rows, 2 * kvh, 128, device=dev, generator=g) * width).bfloat16()
    chunks = [SeqChunk(i, 1, 16 * pages - 1, list(range(pages))) for i in range(rows)]
    meta = build_attention_metadata(chunks, torch.zeros(rows, dtype=torch.int64, device=dev), 16)
    chosen = torch.arange(pages, dtype=torch.int32, device=dev).repeat(rows, kvh, 1)
    scale = 128**-0.5
    out = attend_pages(q, *views, meta, chosen, scale).double()
    ks, vs = (layer_as_slots(x).double().transpose(0, 1)[None] for x in views)  # [1, kv_heads, keys, 128]
    x = q.double().unflatten(1, (kvh, 2))
    s = x @ ks.transpose(-1, -2) * scale
    w = torch.softmax(s, -1)
    want = (w @ vs).flatten(1, 2)
    d = (2.0**-16 * (x.abs() @ ks.abs().transpose(-1, -2)) * scale + 2.0**-22 * s.abs()).amax(-1, keepdim=True)
    n, u = 16 * pages, 2.0**-17 if dtype == torch.bfloat16 else 2.0**-22
    bound = (w @ vs.abs()) * (u + 2 * d + n * 2.0**-23 + 2.0**-20) + n * 2.0**-124
    if dtype != torch.bfloat16:
        bound += n * 2.0**-36 * (w * vs.abs().amax(-1)[:, :, None]).amax(-1, keepdim=True)
    bound = bound.flatten(1, 2) + 2.0**-8 * want.abs()
    over = ((out - want).abs() / bound).max().item()
    assert over <= 1, over
