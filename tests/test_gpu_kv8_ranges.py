"""V rows of very different sizes in an 8-bit pool: whatever finite value a row holds, a query gets the
definition's output from the keys it sees.

The bound is that of ``paged_reference`` plus what f16 loses below its normal range.  A weight times
its row's scale is rounded to f16, whose step below 2^-14 is 2^-24, so a key loses at most half of it,
2^-25, against units in which the row's largest p 2^e is at least 1; a code is at most 448, and the
largest row's own amax at least 224 2^e.  Over n keys that is at most n 2^-24 max_j w_j max|v_j|.
"""

from __future__ import annotations

import random

import pytest
import torch

from miniserve_b200.attention import SeqChunk, attend, build_attention_metadata, kv_scatter
from miniserve_b200.kv_pool import KV8, allocate_kv_cache, layer_as_slots, slots_into_layer
from paged_reference import SCALE, U_F16, assert_close, attention64, visible

pytestmark = pytest.mark.gpu

KVH = 2


def random_tree(rng: random.Random, n: int) -> list[int]:
    return [rng.randint(max(-1, i - 6), i - 1) for i in range(n)]


KINDS = {  # new tokens and whether they are a tree
    "decode": (1, False), "verify": (5, False), "chunk20": (20, False), "chunk40": (40, False),
    "tree12": (12, True), "tree40": (40, True),
}


def setup(dev, kind: str, cached: int, seed: int):
    """One sequence over shuffled blocks: chunk, slots of its positions, K, V (reference layout), q."""
    n, tree = KINDS[kind]
    rng = random.Random(seed)
    blocks = -(-(n + cached) // 16)
    table = rng.sample(range(blocks + 2), blocks)
    chunk = SeqChunk(0, n, cached, table, parents=random_tree(rng, n) if tree else None)
    g = torch.Generator(device=dev).manual_seed(seed)
    k, v = (torch.randn((blocks + 2) * 16, KVH, 128, device=dev, generator=g) for _ in range(2))
    q = torch.randn(n, 2 * KVH, 128, device=dev, generator=g)
    p = torch.arange(n + cached)
    slots = (torch.tensor(table)[p // 16] * 16 + p % 16).to(dev)
    return chunk, slots, k, v, q


def lost(q, views, chunk) -> torch.Tensor:
    """n 2^-24 max_j w_j max|v_j| of every query row, [n, heads, 1]."""
    k, v = layer_as_slots(views[0]), layer_as_slots(views[1])
    p = torch.arange(chunk.context_len)
    slots = (torch.tensor(chunk.block_table)[p // 16] * 16 + p % 16).to(q.device)
    see = visible(chunk).to(q.device)
    out = []
    for h in range(q.shape[1]):
        s = q[:, h].double() @ k[slots, h // 2].double().nan_to_num(0).T * SCALE
        w = torch.softmax(torch.where(see, s, -torch.inf), -1)
        top = v[slots, h // 2].double().nan_to_num(0).abs().amax(-1)
        out.append(chunk.context_len * 2.0**-24 * (w * top).amax(-1))
    return torch.stack(out, 1)[..., None]


def check(dev, chunk, slots, k, v, q, split: int = 0) -> torch.Tensor:
    _, views = allocate_kv_cache(1, k.shape[0] // 16, KVH, dev, dtype=KV8)
    slots_into_layer(views[0][0], k.bfloat16())
    slots_into_layer(views[0][1], v.bfloat16())
    q = q.bfloat16()
    meta = build_attention_metadata([chunk], slots[chunk.num_cached :].contiguous(), 16,
                                    pages_per_split=split)
    got = attend(q, *views[0], meta, SCALE)
    ref, bound, rows = attention64(q, *views[0], [chunk], U_F16)
    assert_close(got, ref, bound + lost(q, views[0], chunk), rows)
    return got


@pytest.mark.parametrize("gap", [20, 26, 30, 60, 100])
@pytest.mark.parametrize("at", [3, 150, 199])
@pytest.mark.parametrize("kind", KINDS)
def test_all_weight_on_a_small_row(kind: str, at: int, gap: int, cuda_device) -> None:
    """Every query's weight rests on one cached key whose V row is 2^gap smaller than the others."""
    dev = cuda_device
    chunk, slots, k, v, q = setup(dev, kind, 200, seed=gap + at)
    sign = torch.where(torch.arange(128, device=dev) % 3 == 0, 1.0, -1.0)
    k *= 0.05
    k[slots[at]] = 8 * sign
    q = sign + 0.1 * q  # scores of about 90 and 0
    v[slots[at]] *= 2.0**-gap
    check(dev, chunk, slots, k, v, q)
    check(dev, chunk, slots, k, v, q, split=3)


@pytest.mark.parametrize("split", [0, 2])
@pytest.mark.parametrize("size", [1e9, 1e30, 1e37])
@pytest.mark.parametrize("kind", [k for k in KINDS if k != "decode"])
def test_a_huge_new_row_reaches_only_the_rows_that_see_it(kind: str, size: float, split: int,
                                                          cuda_device) -> None:
    """The V row of a draft, or of a later token, is huge but finite: its siblings and the tokens before
    it keep their results, and those that see it get its share."""
    dev = cuda_device
    for cached, huge in ((0, -1), (37, -1), (200, 1)):
        chunk, slots, k, v, q = setup(dev, kind, cached, seed=cached)
        row = v[slots[cached + huge % chunk.num_new]]
        row *= size / row.abs().amax()
        v[slots[cached + huge % chunk.num_new]] = row
        check(dev, chunk, slots, k, v, q, split)


@pytest.mark.parametrize("split", [0, 3])
@pytest.mark.parametrize("spread", [4, 12, 30, 55])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_every_size(kind: str, spread: int, split: int, cuda_device) -> None:
    """V rows of sizes 2^-spread .. 2^spread, K rows of sizes that decide the weights sharply or
    hardly at all."""
    dev = cuda_device
    for strength in (0.2, 3.0):
        chunk, slots, k, v, q = setup(dev, kind, 333, seed=spread)
        g = torch.Generator(device=dev).manual_seed(spread)
        v *= 2.0 ** ((2 * torch.rand(v.shape[0], KVH, 1, device=dev, generator=g) - 1) * spread)
        check(dev, chunk, slots, k, v, q * strength, split)


def test_rising_and_falling_sizes(cuda_device) -> None:
    """Sizes that grow, or shrink, by a power of two every few keys over a whole context."""
    dev = cuda_device
    for step in (-0.25, 0.25):
        for kind in ("decode", "chunk40", "tree12"):
            chunk, slots, k, v, q = setup(dev, kind, 600, seed=5)
            v[slots] *= 2.0 ** (step * torch.arange(slots.numel(), device=dev) - 300 * step)[:, None, None]
            check(dev, chunk, slots, k, v, q)


@pytest.mark.parametrize("kind", ["decode", "tree12"])
def test_many_tiny_weights_beside_a_strong_key(kind: str, cuda_device) -> None:
    """131072 keys of weight 2^-20.4 carry 9 % of the output beside one strong key, while a key of no
    weight holds a V row 64 times as large."""
    dev = cuda_device
    chunk, slots, k, v, q = setup(dev, kind, 131072, seed=1)
    sign = torch.where(torch.arange(128, device=dev) % 3 == 0, 1.0, -1.0)
    turn = torch.where(torch.arange(128, device=dev) % 2 == 0, 1.0, -1.0)
    k.zero_()
    k[slots[1]], k[slots[2]] = 1.25 * sign, -1.25 * sign  # scores of +-14.1 = 20.4 ln 2
    v[:] = turn
    v[slots[1]], v[slots[2]] = sign, 64.0
    _, views = allocate_kv_cache(1, k.shape[0] // 16, KVH, dev, dtype=KV8)
    slots_into_layer(views[0][0], k.bfloat16())
    slots_into_layer(views[0][1], v.bfloat16())
    q = sign.expand_as(q).bfloat16()
    meta = build_attention_metadata([chunk], slots[chunk.num_cached :].contiguous(), 16,
                                    pages_per_split=1 << 14)
    got = attend(q, *views[0], meta, SCALE)
    ref, _, _ = attention64(q, *views[0], [chunk], U_F16)
    # Half a bf16 step of an output of at most 1.1; half a step of f16's smallest, 2^-25, of weights of
    # 2^-20.4 that sum to 0.095, all rounded alike; and, in the numerator and in the sum of weights, at
    # most 2048 additions of 16 keys at 2^-23 each (a quarter of the pages per warp).
    limit = 2.0**-8 * 1.1 + 2.0**-4.6 * 0.095 + 2 * 2.0**-12 * 1.1
    assert (got.double() - ref).abs().max().item() <= limit


@pytest.mark.parametrize("kind", ["verify", "chunk20", "tree12"])
def test_a_nan_row_of_no_weight_is_still_seen(kind: str, cuda_device) -> None:
    """A NaN V row among the new tokens whose weight underflows: rows that see it get NaN, as everywhere
    else in the context, and the others nothing of it."""
    dev = cuda_device
    chunk, slots, k, v, q = setup(dev, kind, 200, seed=9)
    sign = torch.where(torch.arange(128, device=dev) % 3 == 0, 1.0, -1.0)
    k *= 0.05
    k[slots[150]] = 8 * sign
    q = sign + 0.1 * q
    v[slots[202]] = float("nan")
    got = check(dev, chunk, slots, k, v, q)
    sees = visible(chunk)[:, 202].to(dev)
    assert bool(sees.any()) and not bool(sees.all())
    assert torch.equal(got.isnan().all(-1).all(-1), sees)


def test_zero_and_unwritten_rows_beside_others(cuda_device) -> None:
    """Zero V rows (the smallest exponent), and slots that were never written, among ordinary ones."""
    dev = cuda_device
    for kind in ("decode", "chunk20", "tree40"):
        chunk, slots, k, v, q = setup(dev, kind, 300, seed=3)
        v[slots[40:90]] = 0.0
        v[slots[7]] *= 2.0**-110  # below the smallest exponent's normal codes
        check(dev, chunk, slots, k, v, q)
        _, views = allocate_kv_cache(1, k.shape[0] // 16, KVH, dev, dtype=KV8)
        kv_scatter(k[slots[100:]].bfloat16(), v[slots[100:]].bfloat16(), slots[100:], *views[0])
        qb = q.bfloat16()
        meta = build_attention_metadata([chunk], slots[chunk.num_cached :].contiguous(), 16)
        got = attend(qb, *views[0], meta, SCALE)
        ref, bound, rows = attention64(qb, *views[0], [chunk], U_F16)
        assert_close(got, ref, bound + lost(qb, views[0], chunk), rows)


@pytest.mark.parametrize("split", [0, 2])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_at_the_end_of_the_range(kind: str, split: int, cuda_device) -> None:
    """V rows of 2e38 and 3e38, one and all of them: every weighted mean is finite, though sums of rows
    are not."""
    dev = cuda_device
    for every in (False, True):
        chunk, slots, k, v, q = setup(dev, kind, 200, seed=11)
        if every:
            v = torch.where(v < 0, -2e38, 2e38)
        else:
            v[slots[[5, 199, 200]]] = 3e38
        got = check(dev, chunk, slots, k, v, q * 0.3, split)
        assert bool(torch.isfinite(got).all())
