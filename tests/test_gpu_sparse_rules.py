"""The rules by which pages are selected, from the definition of a score: sum over the channels of the larger of
q lo and q hi, the larger one of a KV head's two query heads."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import build_attention_metadata, select_pages
from miniserve_b200.attention import SeqChunk

pytestmark = pytest.mark.gpu


def selected(q: torch.Tensor, bounds: torch.Tensor, n: int, budget: int) -> torch.Tensor:
    """[rows, kv_heads, budget] of rows that see n pages each, pages in the order of the blocks: the first one,
    the last two, and of the others those with the largest scores.  A page with a bound that is not finite
    counts as infinite; so does a score that is not finite."""
    x, (lo, hi) = q.double().unflatten(1, (-1, 2)), bounds[:n].double().unbind(2)
    lo, hi = (b.transpose(0, 1)[None, :, None] for b in (lo, hi))  # [1, kv_heads, 1, pages, 128]
    s = torch.maximum(x[..., None, :] * lo, x[..., None, :] * hi).sum(-1).amax(2)
    whole = torch.isfinite(bounds[:n]).all(-1).all(-1).T
    s = torch.where(whole & torch.isfinite(s), s, torch.inf)
    s[..., 0] = s[..., -2:] = torch.inf
    # Ties go to the lower page, but the pages that are always kept come first.
    kept = torch.zeros(n, device=s.device)
    kept[0] = kept[-2:] = 1
    order = s.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, kept[order].sort(dim=-1, descending=True, stable=True).indices)
    return order[..., :budget].sort(-1).values.int()


@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("side", [0, 1], ids=["lo", "hi"])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("value", [-torch.inf, torch.inf, torch.nan])
def test_pages_with_a_bound_that_is_not_finite_come_first(value: float, sign: float, side: int, n: int,
                                                          cuda_device) -> None:
    """Whichever side the bound is on and whatever the sign of the query's channel, also where that side is not
    the larger one."""
    dev = cuda_device
    kvh = 3
    g = torch.Generator(device=dev).manual_seed(n)
    x = torch.randn(2, n + 3, kvh, 128, device=dev, generator=g)
    bounds = torch.stack([x.amin(0), x.amax(0)], 2).bfloat16().contiguous()
    q = torch.randn(4, 2 * kvh, 128, device=dev, generator=g).bfloat16()
    q[..., 77] = sign * q[..., 77].abs()
    q[3, :, 77] = 0
    some, clean = [5, n // 2, n - 9], bounds.clone()
    bounds[some, :, side, 77] = value
    if value == (torch.inf if side == 0 else -torch.inf):  # lo <= hi
        bounds[some, :, 1 - side, 77] = value
    chunks = [SeqChunk(i, 1, 16 * n - 1 - i, list(range(n))) for i in range(4)]
    meta = build_attention_metadata(chunks, torch.zeros(4, dtype=torch.int64, device=dev), 16)
    for budget in (5, 6, 20):
        got = select_pages(q, bounds, meta, budget)
        assert torch.equal(got, selected(q, bounds, n, budget)), budget
        if budget > 5:
            assert bool((got[..., None] == torch.tensor(some, device=dev)).any(2).all())
    assert torch.equal(select_pages(q, clean, meta, 20), selected(q, clean, n, 20))
