"""Attention over trees of drafted tokens on the GPU, through bf16 and 8-bit pools, against a 64-bit
evaluation within the bound of ``paged_reference``."""

from __future__ import annotations

import random

import pytest
import torch

from miniserve_b200.attention import (SeqChunk, attend, build_attention_metadata, kv_gather,
                                      kv_scatter, paged_attention, tree_positions)
from miniserve_b200.kv_pool import KV8, allocate_kv_cache, layer_as_slots, slots_into_layer
from paged_reference import SCALE, U_BF16, U_F16, assert_close, attention64

pytestmark = pytest.mark.gpu

POOLS = {"bf16": (torch.bfloat16, U_BF16), "e4m3": (KV8, U_F16)}


def random_tree(rng: random.Random, n: int, unused: int = 0, back: int = 8) -> list[int]:
    return [rng.randint(max(-1, i - back), i - 1) for i in range(n - unused)] + [-2] * unused


def batch(dev, seqs, kvh: int, pool: str, seed: int = 0):
    """seqs: (new, cached, parents or None).  Every slot of the pool is filled."""
    rng = random.Random(seed)
    need = [-(-(n + c) // 16) for n, c, _ in seqs]
    perm = rng.sample(range(sum(need) + 2), sum(need) + 2)
    at = flat = 0
    chunks = []
    for (n, c, parents), b in zip(seqs, need):
        chunks.append(SeqChunk(flat, n, c, perm[at : at + b], parents=parents))
        at += b
        flat += n
    g = torch.Generator(device=dev).manual_seed(seed)
    _, views = allocate_kv_cache(1, len(perm), kvh, dev, dtype=POOLS[pool][0])
    for view in views[0]:
        x = torch.randn(len(perm) * 16, kvh, 128, device=dev, generator=g)
        x *= torch.exp(0.5 * torch.randn(len(perm) * 16, kvh, 1, device=dev, generator=g))
        slots_into_layer(view, x.bfloat16())
    q = torch.randn(flat, 2 * kvh, 128, device=dev, generator=g).bfloat16()
    return views[0], chunks, q


def slots_of(chunks, dev) -> torch.Tensor:
    return torch.tensor([c.block_table[p // 16] * 16 + p % 16 for c in chunks
                         for p in range(c.num_cached, c.context_len)], device=dev)


def check(views, chunks, q, u: float, split: int = 0) -> torch.Tensor:
    meta = build_attention_metadata(chunks, slots_of(chunks, q.device), 16, pages_per_split=split)
    out = attend(q, *views, meta, SCALE)
    ref, bound, covered = attention64(q, *views, chunks, u)
    assert_close(out, ref, bound, covered)
    return out


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("split", [0, 1, 5])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 63, 64, 65, 100])
def test_random_trees(n: int, split: int, pool: str, cuda_device) -> None:
    """Tile and page borders: trees over 0, 1, 15, 16, 17 and 500 cached tokens (and 512, 645 and 1535,
    whose whole blocks larger trees read on the tensor cores), some positions unused."""
    rng = random.Random(n)
    seqs = [(n, c, random_tree(rng, n, unused=rng.choice([0, 0, n // 4])))
            for c in (0, 1, 15, 16, 17, 500, 512, 645, 1535)]
    views, chunks, q = batch(cuda_device, seqs, 2, pool, seed=n)
    check(views, chunks, q, POOLS[pool][1], split)


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("kvh", [1, 3, 8])
def test_head_counts_and_many_sequences(kvh: int, pool: str, cuda_device) -> None:
    rng = random.Random(kvh)
    seqs = [(n, rng.randint(0, 400), random_tree(rng, n)) for n in
            [rng.choice([1, 4, 8, 16, 30, 60]) for _ in range(40)]]
    views, chunks, q = batch(cuda_device, seqs, kvh, pool, seed=kvh)
    check(views, chunks, q, POOLS[pool][1])


@pytest.mark.parametrize("pool", POOLS)
def test_a_chain_is_a_causal_chunk(pool: str, cuda_device) -> None:
    """Drafts in a chain see what a verify row's tokens see: both paths within their bounds, and in an
    8-bit pool (the same kernel, the same pages per warp) bit for bit."""
    chain = lambda n: list(range(-1, n - 1))  # noqa: E731
    seqs = [(8, 100, chain(8)), (5, 33, chain(5)), (30, 250, chain(30))]
    views, chunks, q = batch(cuda_device, seqs, 2, pool, seed=3)
    tree = check(views, chunks, q, POOLS[pool][1], split=64)
    causal = [SeqChunk(c.flat_start, c.num_new, c.num_cached, c.block_table) for c in chunks]
    plain = check(views, causal, q, POOLS[pool][1], split=64)
    if pool == "e4m3":
        assert torch.equal(tree, plain)


@pytest.mark.parametrize("pool", POOLS)
def test_trees_beside_other_work(pool: str, cuda_device) -> None:
    """One step with trees, decode rows, a short chunk and a prompt chunk, in any order."""
    rng = random.Random(1)
    seqs = [(1, 80, None), (12, 90, random_tree(rng, 12)), (100, 30, None), (40, 77, random_tree(rng, 40)),
            (20, 5, None), (6, 0, random_tree(rng, 6, unused=2)), (3, 300, None)]
    views, chunks, q = batch(cuda_device, seqs, 8, pool, seed=5)
    check(views, chunks, q, U_BF16)
    check(views, chunks, q, U_BF16, split=8)


@pytest.mark.parametrize("pool", POOLS)
def test_unused_positions_may_hold_anything(pool: str, cuda_device) -> None:
    """NaN and infinities in the q, k and v rows of unused drafts and behind the sequence: the other
    rows are as without them, the unused rows zero (also where nothing at all is visible)."""
    dev = cuda_device
    rng = random.Random(2)
    seqs = [(16, 40, random_tree(rng, 16, unused=5)), (8, 0, [-2] * 8), (3, 9, [-2, -1, -2]),
            (33, 3, random_tree(rng, 33, unused=20)), (40, 700, random_tree(rng, 40, unused=30)),
            (20, 600, [-2] * 20)]
    views, chunks, q = batch(dev, seqs, 2, pool, seed=6)
    clean = check(views, chunks, q, U_BF16)
    ks, vs = layer_as_slots(views[0]), layer_as_slots(views[1])
    live = torch.zeros(ks.shape[0], dtype=torch.bool)
    for c in chunks:
        for p in range(c.context_len):
            k = p - c.num_cached
            live[c.block_table[p // 16] * 16 + p % 16] = k < 0 or c.parents[k] != -2
        for k in range(c.num_new):
            if c.parents[k] == -2:
                q[c.flat_start + k] = float("nan") if k % 2 else float("inf")
                assert bool((clean[c.flat_start + k] == 0).all())
    dead = (~live).nonzero().flatten().to(dev)
    ks[dead], vs[dead] = float("nan"), float("inf")
    vs[dead[::2]] = float("nan")
    slots_into_layer(views[0], ks)
    slots_into_layer(views[1], vs)
    assert torch.equal(check(views, chunks, q, U_BF16), clean)
    assert torch.equal(check(views, chunks, q, U_BF16, split=1).isnan(), clean.isnan())


@pytest.mark.parametrize("pool", POOLS)
def test_a_bad_draft_reaches_only_its_descendants(pool: str, cuda_device) -> None:
    """NaN or infinite values of one draft: the rows that see it get them, its siblings do not."""
    dev = cuda_device
    parents = [-1, 0, 0, 1, 1, 2, 2, -1, 7, 3]
    views, chunks, q = batch(dev, [(10, 21, parents), (10, 40, parents)], 2, pool, seed=7)
    ks, vs = layer_as_slots(views[0]), layer_as_slots(views[1])

    def slot(c, k):
        p = c.num_cached + k
        return c.block_table[p // 16] * 16 + p % 16

    vs[slot(chunks[0], 1), 0, 5] = float("nan")
    vs[slot(chunks[0], 1), 0, 77] = float("inf")
    vs[slot(chunks[0], 7), 1, 6] = -float("inf")
    ks[slot(chunks[1], 2), 0, 6] = float("nan")
    slots_into_layer(views[0], ks)
    slots_into_layer(views[1], vs)
    out = check(views, chunks, q, POOLS[pool][1])
    bad = out.isnan().any(-1)
    assert bad[:10, 0].tolist() == [False, True, False, True, True, False, False, False, False, True]
    assert bad[10:, 0].tolist() == [False, False, True, False, False, True, True, False, False, False]


@pytest.mark.parametrize("pool", POOLS)
def test_long_context_is_split(pool: str, cuda_device) -> None:
    rng = random.Random(4)
    views, chunks, q = batch(cuda_device, [(16, 9000, random_tree(rng, 16)),
                                           (50, 6001, random_tree(rng, 50))], 2, pool, seed=8)
    meta = build_attention_metadata(chunks, slots_of(chunks, cuda_device), 16)
    assert meta.tree.info.n_combine > 0
    first = check(views, chunks, q, U_BF16)
    assert torch.equal(check(views, chunks, q, U_BF16), first)


@pytest.mark.parametrize("pool", POOLS)
def test_a_captured_step_takes_new_trees(pool: str, cuda_device) -> None:
    """The tree and the cached length change between replays; update() writes masks and tables into
    the captured plan."""
    dev = cuda_device
    rng = random.Random(9)
    seqs = [(12, 50, random_tree(rng, 12)), (1, 33, None), (12, 97, random_tree(rng, 12))]
    views, chunks, q = batch(dev, seqs, 4, pool, seed=9)
    slots = slots_of(chunks, dev)
    meta = build_attention_metadata(chunks, slots, 16)
    k = torch.randn(25, 4, 128, device=dev).bfloat16()
    paged_attention(q, k, k, *views, meta, SCALE)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, k, k, *views, meta, SCALE)
    for step in (1, 2):
        new = [SeqChunk(c.flat_start, c.num_new, c.num_cached + (0 if c.parents is None else -step),
                        c.block_table, parents=c.parents and random_tree(rng, 12, unused=step))
               for c in chunks]
        k.copy_(torch.randn(25, 4, 128, device=dev))
        q.copy_(torch.randn(25, 8, 128, device=dev))
        assert meta.update(new, slots_of(new, dev))
        graph.replay()
        ref, bound, covered = attention64(q, *views, new, U_BF16)
        assert_close(out, ref, bound, covered)
    assert not meta.update([chunks[1]])


def test_refusals(cuda_device) -> None:
    views, chunks, q = batch(cuda_device, [(3, 5, [-1, 0, 0])], 2, "bf16")
    with pytest.raises(ValueError, match="parent"):
        build_attention_metadata([SeqChunk(0, 3, 5, chunks[0].block_table, parents=[-1, 0, 2])],
                                 slots_of(chunks, cuda_device), 16)
    meta = build_attention_metadata(chunks, slots_of(chunks, cuda_device), 16)
    with pytest.raises(ValueError, match="scale"):
        attend(q, *views, meta, -1.0)
    with pytest.raises(ValueError, match="rows"):
        attend(q[:2], *views, meta, SCALE)


@pytest.mark.parametrize("pool", POOLS)
def test_a_speculative_loop(pool: str, cuda_device) -> None:
    """The operators together, as a server uses them: draft trees are written and attended, a path of
    each is accepted and its rows moved behind the cached tokens, and the next step decodes over
    them.  Every step against the 64-bit evaluation; the moved rows bit for bit."""
    dev = cuda_device
    rng = random.Random(11)
    kvh, g = 4, torch.Generator(device=dev).manual_seed(11)
    perm = rng.sample(range(60), 60)
    tables = [perm[20 * i : 20 * i + 20] for i in range(3)]
    cached = [50, 111, 7]
    _, pools = allocate_kv_cache(1, 60, kvh, dev, dtype=POOLS[pool][0])
    views = pools[0]

    def fresh(n):
        return (torch.randn(n, kvh, 128, device=dev, generator=g).bfloat16(),
                torch.randn(n, kvh, 128, device=dev, generator=g).bfloat16(),
                torch.randn(n, 2 * kvh, 128, device=dev, generator=g).bfloat16())

    k, v, _ = fresh(60 * 16)
    kv_scatter(k, v, torch.arange(960, device=dev), *views)
    for _ in range(3):
        parents = [random_tree(rng, 14) for _ in tables]
        assert [max(tree_positions(c, p)) < c + 14 for c, p in zip(cached, parents)]
        chunks = [SeqChunk(14 * i, 14, cached[i], tables[i], parents=parents[i]) for i in range(3)]
        slots = slots_of(chunks, dev)
        meta = build_attention_metadata(chunks, slots, 16)
        k, v, q = fresh(42)
        out = paged_attention(q, k, v, *views, meta, SCALE)
        ref, bound, covered = attention64(q, *views, chunks, POOLS[pool][1])
        assert_close(out, ref, bound, covered)
        src, dst = [], []
        for i, c in enumerate(chunks):
            path = [rng.randrange(14)]
            while parents[i][path[0]] >= 0:
                path.insert(0, parents[i][path[0]])
            for depth, k_ in enumerate(path):
                src.append(int(slots[14 * i + k_]))
                p = c.num_cached + depth
                dst.append(tables[i][p // 16] * 16 + p % 16)
            cached[i] += len(path)
        before = [layer_as_slots(x)[src] for x in views]
        kv_scatter(*kv_gather(torch.tensor(src, device=dev), *views), torch.tensor(dst, device=dev),
                   *views)
        for x, want in zip(views, before):
            assert torch.equal(layer_as_slots(x)[dst], want)
        chunks = [SeqChunk(i, 1, cached[i], tables[i]) for i in range(3)]
        meta = build_attention_metadata(chunks, slots_of(chunks, dev), 16)
        k, v, q = fresh(3)
        out = paged_attention(q, k, v, *views, meta, SCALE)
        ref, bound, covered = attention64(q, *views, chunks, U_BF16)
        assert_close(out, ref, bound, covered)
        cached = [c + 1 for c in cached]


@pytest.mark.parametrize("pool", POOLS)
def test_graphs_captured_first_and_eager_calls_between(pool: str, cuda_device) -> None:
    """Split tiles count their arrivals in the workspace: graphs captured before any eager call, an eager
    call before their first replay, and replays in any order all find the counters at zero."""
    dev = cuda_device
    rng = random.Random(5)
    warm_views, warm_chunks, warm_q = batch(dev, [(3, 20, [-1, 0, 0])], 2, pool, seed=1)
    check(warm_views, warm_chunks, warm_q, U_BF16)  # loads the kernels
    seqs = [(8, 2500, random_tree(rng, 8)), (40, 1100, random_tree(rng, 40)), (2, 3000, None)]
    views, chunks, q = batch(dev, seqs, 2, pool, seed=11)
    meta = build_attention_metadata(chunks, slots_of(chunks, dev), 16, pages_per_split=24)
    assert meta.tree.info.n_combine > 0
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attend(q, *views, meta, SCALE)
            out2 = attend(q, *views, meta, SCALE)
        graphs.append((g, out, out2))
    eager = attend(q, *views, meta, SCALE).clone()
    ref, bound, covered = attention64(q, *views, chunks, U_BF16)
    assert_close(eager, ref, bound, covered)
    for k in (1, 0, 0, 1):
        g, out, out2 = graphs[k]
        out.fill_(7.0)
        out2.fill_(7.0)
        g.replay()
        assert torch.equal(out, eager) and torch.equal(out2, eager)
        assert torch.equal(attend(q, *views, meta, SCALE), eager)


@pytest.mark.parametrize("pool", POOLS)
def test_two_steps_at_once(pool: str, cuda_device) -> None:
    """Two steps with metadata of their own, on two streams over one pool."""
    dev = cuda_device
    rng = random.Random(6)
    seqs = [(16, 1500, random_tree(rng, 16)), (50, 900, random_tree(rng, 50)), (4, 2000, None)] * 3
    views, chunks, q = batch(dev, seqs, 4, pool, seed=12)
    want = check(views, chunks, q, U_BF16, split=16)
    metas = [build_attention_metadata(chunks, slots_of(chunks, dev), 16, pages_per_split=16)
             for _ in range(2)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize(dev)
    outs = []
    for _ in range(5):
        for meta, stream in zip(metas, streams):
            with torch.cuda.stream(stream):
                outs.append(attend(q, *views, meta, SCALE))
    torch.cuda.synchronize(dev)
    assert all(torch.equal(out, want) for out in outs)


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("n,cached", [(1024, 3), (1024, 530), (1000, 515)])
def test_the_largest_trees(n: int, cached: int, pool: str, cuda_device) -> None:
    rng = random.Random(n + cached)
    seqs = [(n, cached, random_tree(rng, n, unused=rng.choice([0, 9]), back=40)), (3, 40, [-1, 0, 0])]
    views, chunks, q = batch(cuda_device, seqs, 1, pool, seed=n)
    check(views, chunks, q, POOLS[pool][1])


@pytest.mark.parametrize("pool", POOLS)
def test_pools_beyond_32_bit_offsets(pool: str, cuda_device) -> None:
    """The same rows in the first and in the last blocks of a pool of more than 4 GiB: read back and
    attended (decode, a short and a long chunk, small and larger trees), the results are the same."""
    dev = cuda_device
    kvh, rng = 8, random.Random(13)
    page = 4128 if pool == "e4m3" else 8192
    blocks = (1 << 32) // (page * kvh) + 200
    _, layers = allocate_kv_cache(1, blocks, kvh, dev, dtype=POOLS[pool][0])
    views = layers[0]
    seqs = [(1, 300, None), (20, 30, None), (90, 40, None), (9, 100, random_tree(rng, 9)),
            (40, 700, random_tree(rng, 40))]
    outs, rows = [], []
    g = torch.Generator(device=dev).manual_seed(13)
    tokens = sum(n + c for n, c, _ in seqs)
    k = torch.randn(tokens, kvh, 128, device=dev, generator=g).bfloat16()
    v = torch.randn(tokens, kvh, 128, device=dev, generator=g).bfloat16()
    q = torch.randn(sum(n for n, _, _ in seqs), 2 * kvh, 128, device=dev, generator=g).bfloat16()
    need = sum(-(-(n + c) // 16) for n, c, _ in seqs)
    assert blocks * page * kvh > 1 << 32 and need < 150
    for first in (0, blocks - need):
        at, flat, chunks = first, 0, []
        for n, c, parents in seqs:
            nb = -(-(n + c) // 16)
            chunks.append(SeqChunk(flat, n, c, list(range(at, at + nb)), parents=parents))
            at += nb
            flat += n
        slots = torch.tensor([c.block_table[p // 16] * 16 + p % 16 for c in chunks
                              for p in range(c.context_len)], device=dev)
        kv_scatter(k, v, slots, *views)
        torch.cuda.synchronize(dev)
        rows.append(kv_gather(slots, *views))
        meta = build_attention_metadata(chunks, slots_of(chunks, dev), 16)
        outs.append(attend(q, *views, meta, SCALE))
    assert torch.equal(outs[0], outs[1]) and not bool(outs[0].isnan().any())
    assert torch.equal(rows[0][0], rows[1][0]) and torch.equal(rows[0][1], rows[1][1])
    if pool == "bf16":
        assert torch.equal(rows[1][0], k) and torch.equal(rows[1][1], v)


@pytest.mark.parametrize("pool", POOLS)
def test_empty_calls(pool: str, cuda_device) -> None:
    dev = cuda_device
    _, layers = allocate_kv_cache(1, 2, 2, dev, dtype=POOLS[pool][0])
    none = torch.empty(0, 2, 128, dtype=torch.bfloat16, device=dev)
    slots = torch.empty(0, dtype=torch.int64, device=dev)
    kv_scatter(none, none, slots, *layers[0])
    assert kv_gather(slots, *layers[0])[0].shape == (0, 2, 128)
    meta = build_attention_metadata([], slots, 16)
    q = torch.empty(0, 4, 128, dtype=torch.bfloat16, device=dev)
    assert attend(q, *layers[0], meta, SCALE).shape == q.shape
