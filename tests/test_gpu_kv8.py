"""The 8-bit pool on the GPU: rows quantised as they are written, read back, and attended through.

Writes and reads are compared bit for bit with the definition (``quantise_rows``); attention with a
64-bit evaluation over the values the pool stands for, within the bound of ``paged_reference``.
"""

from __future__ import annotations

import random
from types import SimpleNamespace

import pytest
import torch

from miniserve_b200 import _capi
from miniserve_b200.attention import (SeqChunk, attend, build_attention_metadata, kv_gather,
                                      kv_scatter, paged_attention)
from miniserve_b200.kv_pool import KV8, allocate_kv_cache, layer_as_slots, slots_into_layer
from miniserve_b200.qwen3_attention import Qwen3Attention, qk_norm_rope_scatter
from miniserve_b200.workloads import rope_tables
from paged_reference import SCALE, U_F16, assert_close, attention64

pytestmark = pytest.mark.gpu


def status() -> int:
    return _capi.device_status(int(torch.cuda.current_stream().cuda_stream))


def rows(dev, n: int, kvh: int, seed: int, spread: float = 1.0) -> torch.Tensor:
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(n, kvh, 128, device=dev, generator=g)
    return (x * torch.exp(spread * torch.randn(n, kvh, 1, device=dev, generator=g))).bfloat16()


def special_rows(dev) -> torch.Tensor:
    """Rows where the quantiser can go wrong: zeros, one tiny or huge value, the borders of a binade,
    values on a rounding tie, subnormals, infinities, NaN."""
    x = torch.zeros(20, 128, device=dev)
    x[1, 5] = 448
    x[2, 5] = 450
    x[3, 127] = -2.0**-133
    x[4, 0] = 3.3895313892515355e38
    x[5, :] = -3.3895313892515355e38
    x[6] = torch.linspace(-448, 448, 128, device=dev)
    x[7] = torch.arange(128, device=dev) * 2.0**-9  # ties of the subnormal grid
    x[7, 0] = 448
    x[8] = 2.0 ** (torch.arange(128, device=dev).float() - 100)
    x[9] = 1.0625 * 2.0 ** (torch.arange(128, device=dev) % 9 - 4).float()  # ties of normal codes
    x[10, 64] = float("nan")
    x[11, 127] = float("inf")
    x[12, 0] = -float("inf")
    x[13, :] = float("nan")
    x[14, 3] = -0.0
    x[15, :] = 2.0**-120
    x[16, :] = 1.7578125 * 2.0**-95
    x[17, :] = 232 * 2.0**120
    x[18] = torch.randn(128, device=dev, generator=torch.Generator(device=dev).manual_seed(1)) * 1e30
    x[19, ::2] = 1.0
    return x.bfloat16()


# ---- write and read back ------------------------------------------------------------------------


@pytest.mark.parametrize("kvh", [1, 2, 3, 8])
@pytest.mark.parametrize("tokens", [1, 2, 17, 301, 3001])
def test_scatter_writes_exactly_the_definition(tokens: int, kvh: int, cuda_device) -> None:
    """The whole pool, written and unwritten slots, bit for bit; K and V as views of a wider row."""
    dev = cuda_device
    blocks = tokens // 16 + 3
    g = torch.Generator(device=dev).manual_seed(tokens + kvh)
    slots = torch.randperm(blocks * 16, device=dev, generator=g)[:tokens]
    old_k, old_v = rows(dev, blocks * 16, kvh, 5), rows(dev, blocks * 16, kvh, 6)
    for pad in (0, 4, 8):  # row strides that allow 16-byte loads, and one that does not
        wide = torch.zeros(tokens, 2 * kvh * 128 + pad, device=dev, dtype=torch.bfloat16)
        k = wide[:, : kvh * 128].unflatten(1, (kvh, 128))
        v = wide[:, kvh * 128 : 2 * kvh * 128].unflatten(1, (kvh, 128))
        k.copy_(rows(dev, tokens, kvh, 1, 3.0))
        v.copy_(rows(dev, tokens, kvh, 2, 3.0))
        pool, views = allocate_kv_cache(2, blocks, kvh, dev, dtype=KV8)
        want, wviews = allocate_kv_cache(2, blocks, kvh, dev, dtype=KV8)
        for (kc, vc) in (views[1], wviews[1]):
            slots_into_layer(kc, old_k)
            slots_into_layer(vc, old_v)
        new_k, new_v = old_k.clone(), old_v.clone()
        new_k[slots], new_v[slots] = k, v
        slots_into_layer(wviews[1][0], new_k)
        slots_into_layer(wviews[1][1], new_v)
        kv_scatter(k, v, slots, *views[1])
        assert torch.equal(pool.view(torch.uint8), want.view(torch.uint8))
        gk, gv = kv_gather(slots, *views[1])
        assert torch.equal(gk, layer_as_slots(views[1][0])[slots])
        assert torch.equal(gv, layer_as_slots(views[1][1])[slots])
        # Written back, the rows stand for the same values.
        kv_scatter(gk, gv, slots, *views[1])
        assert torch.equal(kv_gather(slots, *views[1])[0], gk)


def test_scatter_of_special_rows(cuda_device) -> None:
    dev = cuda_device
    x = special_rows(dev)
    k = torch.stack([x, x.flip(0)], 1)  # [20, 2, 128]
    pool, views = allocate_kv_cache(1, 2, 2, dev, dtype=KV8)
    want, wviews = allocate_kv_cache(1, 2, 2, dev, dtype=KV8)
    full = torch.zeros(32, 2, 128, device=dev, dtype=torch.bfloat16)
    full[:20] = k
    slots_into_layer(wviews[0][0], full)
    slots_into_layer(wviews[0][1], full.flip(1))
    kv_scatter(full, full.flip(1).contiguous(), torch.arange(32, device=dev), *views[0])
    assert torch.equal(pool.view(torch.uint8), want.view(torch.uint8))
    gk, _ = kv_gather(torch.arange(20, device=dev), *views[0])
    ref = layer_as_slots(wviews[0][0])[:20]
    assert torch.equal(gk.isnan(), ref.isnan())
    assert torch.equal(gk.nan_to_num(1.0), ref.nan_to_num(1.0))
    assert bool(gk[10, 0].isnan().all()) and bool(gk[11, 0].isnan().all())
    assert bool(torch.isfinite(gk[4, 0]).all())


def test_slots_outside_the_pool(cuda_device) -> None:
    """A write to such a slot is skipped, a read gives zeros, and both set the status bit."""
    dev = cuda_device
    pool, views = allocate_kv_cache(1, 3, 2, dev, dtype=KV8)
    x = rows(dev, 4, 2, 3)
    before = None
    for slots in ([5, 48, -1, 7], [5, 1 << 40, -(1 << 40), 7]):
        s = torch.tensor(slots, device=dev)
        kv_scatter(x, x, s, *views[0])
        assert status() == _capi.DEV_BAD_SLOT
        k, v = kv_gather(s, *views[0])
        assert status() == _capi.DEV_BAD_SLOT
        assert bool((k[1:3] == 0).all()) and bool((v[1:3] == 0).all())
        assert bool((k[0] != 0).any()) and bool((k[3] != 0).any())
        now = pool.view(torch.uint8).clone()
        assert before is None or torch.equal(before, now)
        before = now
    bpool, bviews = allocate_kv_cache(1, 3, 2, dev)
    k, v = kv_gather(torch.tensor([48, 1], device=dev), *bviews[0])
    assert status() == _capi.DEV_BAD_SLOT and bool((k == 0).all())


@pytest.mark.parametrize("kvh", [1, 3, 8])
@pytest.mark.parametrize("n", [0, 1, 5, 333, 4001])
def test_gather_from_a_bf16_pool(n: int, kvh: int, cuda_device) -> None:
    """Any order, repeats, NaN and infinities: the pool's bits."""
    dev = cuda_device
    _, views = allocate_kv_cache(1, 40, kvh, dev)
    k, v = rows(dev, 640, kvh, 1), rows(dev, 640, kvh, 2)
    k[3, 0, 7], v[9, 0, 1] = float("nan"), float("inf")
    slots_into_layer(views[0][0], k)
    slots_into_layer(views[0][1], v)
    g = torch.Generator(device=dev).manual_seed(n)
    slots = torch.randint(0, 640, (n,), device=dev, generator=g)
    wide = torch.full((n, 2 * kvh * 128 + 8), 7.0, device=dev, dtype=torch.bfloat16)
    ko = wide[:, : kvh * 128].unflatten(1, (kvh, 128))
    vo = wide[:, kvh * 128 : 2 * kvh * 128].unflatten(1, (kvh, 128))
    gk, gv = kv_gather(slots, *views[0], k_out=ko, v_out=vo)
    assert gk.data_ptr() == ko.data_ptr()
    assert torch.equal(gk.view(torch.int16), k[slots].view(torch.int16))
    assert torch.equal(gv.view(torch.int16), v[slots].view(torch.int16))
    assert bool((wide[:, 2 * kvh * 128 :] == 7.0).all())
    if n:
        a, b = kv_gather(slots, *views[0])
        assert torch.equal(a.view(torch.int16), gk.contiguous().view(torch.int16))
        assert torch.equal(b.view(torch.int16), gv.contiguous().view(torch.int16))


@pytest.mark.parametrize("pad", [0, 4], ids=["16_byte_form", "8_byte_form"])
def test_kernel_a_quantises_the_rows_it_would_store(pad: int, cuda_device) -> None:
    dev = cuda_device
    t, h, kvh = 77, 16, 8
    g = torch.Generator(device=dev).manual_seed(3)
    width = (h + 2 * kvh) * 128
    wide = torch.zeros(t, width + pad, device=dev, dtype=torch.bfloat16)
    qkv = wide[:, :width]
    qkv.copy_(torch.randn(t, width, device=dev, generator=g) * 2)
    qkv[5, 17 * 128 + 3] = float("nan")  # a key row, and a value row
    qkv[6, 26 * 128 + 3] = float("inf")
    qw = (1 + 0.2 * torch.randn(128, device=dev, generator=g)).bfloat16()
    cos, sin = rope_tables(128, t, 1e6, dev)
    slots = torch.randperm(96, device=dev, generator=g)[:t]
    _, bf = allocate_kv_cache(1, 6, kvh, dev)
    pool, v8 = allocate_kv_cache(1, 6, kvh, dev, dtype=KV8)
    want, w8 = allocate_kv_cache(1, 6, kvh, dev, dtype=KV8)
    q0 = qk_norm_rope_scatter(qkv, qw, qw, 1e-6, cos, sin, slots, *bf[0], h)
    q1 = qk_norm_rope_scatter(qkv, qw, qw, 1e-6, cos, sin, slots, *v8[0], h)
    assert torch.equal(q0, q1)
    k, v = kv_gather(slots, *bf[0])
    kv_scatter(k, v, slots, *w8[0])
    assert torch.equal(pool.view(torch.uint8), want.view(torch.uint8))


# ---- attention ------------------------------------------------------------------------------------


def batch(dev, seqs, kvh: int, seed: int = 0, shared: int = 0, spread: float = 0.5, q_scale=1.0):
    """Pool (every slot filled, free ones with leftovers), chunks and queries for (new, cached) rows;
    the first ``shared`` blocks are common to every sequence."""
    rng = random.Random(seed)
    need = [-(-(n + c) // 16) for n, c in seqs]
    total = shared + sum(max(0, b - shared) for b in need)
    perm = rng.sample(range(total + 3), total + 3)
    at, flat, chunks = shared, 0, []
    for (n, c), b in zip(seqs, need):
        own = max(0, b - shared)
        chunks.append(SeqChunk(flat, n, c, perm[:min(b, shared)] + perm[at : at + own]))
        at += own
        flat += n
    _, views = allocate_kv_cache(1, total + 3, kvh, dev, dtype=KV8)
    slots_into_layer(views[0][0], rows(dev, (total + 3) * 16, kvh, seed + 1, spread))
    slots_into_layer(views[0][1], rows(dev, (total + 3) * 16, kvh, seed + 2, spread))
    g = torch.Generator(device=dev).manual_seed(seed + 3)
    q = (torch.randn(flat, 2 * kvh, 128, device=dev, generator=g) * q_scale).bfloat16()
    return views[0], chunks, q


def slot_map(chunks, dev) -> torch.Tensor:
    out = []
    for c in chunks:
        for p in range(c.num_cached, c.context_len):
            out.append(c.block_table[p // 16] * 16 + p % 16)
    return torch.tensor(out, device=dev, dtype=torch.int64)


def check(views, chunks, q, split: int = 0, u: float = U_F16) -> torch.Tensor:
    meta = build_attention_metadata(chunks, slot_map(chunks, q.device), 16, pages_per_split=split)
    out = attend(q, *views, meta, SCALE)
    ref, bound, covered = attention64(q, *views, chunks, u)
    assert_close(out, ref, bound, covered)
    return out


DECODE = [
    [(1, 0)], [(1, 1)], [(1, 14)], [(1, 15)], [(1, 16)], [(1, 47)], [(1, 500)], [(1, 4000)],
    [(2, 0)], [(3, 13)], [(4, 15)], [(5, 16)], [(7, 40)], [(8, 1)], [(8, 505)],
    [(1, 700), (8, 3), (2, 31), (1, 0), (5, 64)],
]


@pytest.mark.parametrize("split", [0, 1, 3])
@pytest.mark.parametrize("seqs", DECODE, ids=lambda s: "_".join(f"{n}over{c}" for n, c in s))
def test_decode_and_verify_rows(seqs, split: int, cuda_device) -> None:
    views, chunks, q = batch(cuda_device, seqs, 3, seed=len(seqs))
    check(views, chunks, q, split)


@pytest.mark.parametrize("split", [0, 2])
@pytest.mark.parametrize("n", [9, 15, 16, 17, 31, 32, 33, 40, 48, 63, 64])
def test_chunks_of_up_to_64_tokens(n: int, split: int, cuda_device) -> None:
    views, chunks, q = batch(cuda_device, [(n, 0), (n, 7), (n, 130), (1, 50)], 2, seed=n)
    check(views, chunks, q, split)


@pytest.mark.parametrize("kvh", [1, 4, 8])
def test_prompt_chunks_on_the_tensor_cores(kvh: int, cuda_device) -> None:
    """Chunks of more than 64 tokens over expanded pages, beside decode rows and short chunks; P is
    bf16 there.  Also with forced splits (partials from both kernels)."""
    views, chunks, q = batch(cuda_device, [(65, 0), (1, 77), (300, 41), (129, 500), (20, 9)], kvh,
                             seed=kvh)
    for split in (0, 8):
        check(views, chunks, q, split, u=2.0**-8)


def test_many_rows_and_long_rows(cuda_device) -> None:
    rng = random.Random(5)
    seqs = [(rng.choice([1, 1, 2, 5]), rng.randint(0, 700)) for _ in range(90)]
    views, chunks, q = batch(cuda_device, seqs + [(1, 5000), (3, 9001)], 2, seed=9)
    check(views, chunks, q)


@pytest.mark.parametrize("num", [16, 40])
def test_shared_prefix_groups(num: int, cuda_device) -> None:
    """Verify rows over a shared 20-block prefix: planned as a cascade group, whose prefix is expanded
    once and merged in the rows' epilogue."""
    rng = random.Random(num)
    seqs = [(5, 320 + rng.randint(0, 200)) for _ in range(num)]
    views, chunks, q = batch(cuda_device, seqs, 8, seed=num, shared=20)
    meta = build_attention_metadata(chunks, slot_map(chunks, q.device), 16)
    assert meta.info.n_cascade == 1
    check(views, chunks, q, u=2.0**-8)


def test_wide_ranges_of_values(cuda_device) -> None:
    """Rows of very different sizes (exponents 60 binades apart), strong queries."""
    views, chunks, q = batch(cuda_device, [(1, 900), (4, 333)], 2, seed=4, spread=3.0, q_scale=3.0)
    check(views, chunks, q)
    kc, vc = views
    n = kc.shape[0] * 16
    v = rows(cuda_device, n, 2, 8)
    v[::3] *= 2.0**-50
    v[1::3] *= 2.0**20
    slots_into_layer(vc, v)
    check(views, chunks, q)


def test_zero_rows(cuda_device) -> None:
    views, chunks, q = batch(cuda_device, [(1, 100), (3, 20)], 2, seed=6)
    slots_into_layer(views[1], torch.zeros(views[1].shape[0] * 16, 2, 128, device=cuda_device).bfloat16())
    assert bool((check(views, chunks, q) == 0).all())
    q.zero_()
    check(views, chunks, q)
    # A zero-filled pool stands for zeros.
    _, fresh = allocate_kv_cache(1, views[0].shape[0], 2, cuda_device, dtype=KV8)
    assert bool((check(fresh[0], chunks, q) == 0).all())


def test_nan_rows_reach_exactly_the_rows_that_see_them(cuda_device) -> None:
    """A visible NaN row makes the output NaN; one behind the sequence's end, or behind a verify row's
    own position, does not."""
    dev = cuda_device
    views, chunks, q = batch(dev, [(4, 40), (1, 20), (12, 60), (1, 37)], 2, seed=7)
    ks, vs = layer_as_slots(views[0]), layer_as_slots(views[1])

    def slot(c, p):
        return c.block_table[p // 16] * 16 + p % 16

    nan = float("nan")
    vs[slot(chunks[0], 42), 0] = nan     # seen by tokens 2 and 3 of the first sequence
    ks[slot(chunks[2], 66), 1] = nan     # seen by tokens 6.. of the third
    vs[slot(chunks[2], 71), 0] = nan     # seen by its last token
    for p in range(21, 32):              # behind the second sequence's end
        vs[slot(chunks[1], p)] = nan
        ks[slot(chunks[1], p)] = nan
    vs[slot(chunks[3], 5), 1] = float("inf")  # a whole row of NaN in 8 bits
    slots_into_layer(views[0], ks)
    slots_into_layer(views[1], vs)
    out = check(views, chunks, q)
    assert not bool(out[4].isnan().any()) and not bool(out[:2].isnan().any())
    assert bool(out[2, :2].isnan().all()) and not bool(out[2, 2:].isnan().any())
    q[17, 3] = nan  # a NaN query touches its own head's row alone
    q[4, 0, 9] = float("inf")
    check(views, chunks, q)


def test_uninitialised_pool_rows_are_not_read(cuda_device) -> None:
    """Codes of every bit pattern behind the sequences' ends."""
    dev = cuda_device
    views, chunks, q = batch(dev, [(1, 3), (9, 3), (5, 18)], 1, seed=8)
    ref = check(views, chunks, q)
    used = torch.zeros(views[0].shape[0] * 16, dtype=torch.bool)
    for c in chunks:
        for p in range(c.context_len):
            used[c.block_table[p // 16] * 16 + p % 16] = True
    for cache in views:
        raw = cache.view(torch.uint8)
        for s in (~used).nonzero().flatten().tolist():
            raw[s // 16, 0, s % 16] = torch.arange(128, device=dev, dtype=torch.uint8) + 128 * (s % 2)
    meta = build_attention_metadata(chunks, slot_map(chunks, dev), 16)
    assert torch.equal(attend(q, *views, meta, SCALE), ref)


def test_blocks_outside_the_pool_read_as_zeros(cuda_device) -> None:
    dev = cuda_device
    views, chunks, q = batch(dev, [(1, 70), (100, 40)], 2, seed=10)
    meta = build_attention_metadata(chunks, slot_map(chunks, dev), 16)
    for c, i in ((chunks[0], 2), (chunks[1], 3)):
        blk = c.block_table[i]
        z_k, z_v = layer_as_slots(views[0]), layer_as_slots(views[1])
        z_k[blk * 16 : blk * 16 + 16] = 0
        z_v[blk * 16 : blk * 16 + 16] = 0
        slots_into_layer(views[0], z_k)
        slots_into_layer(views[1], z_v)
        c.block_table[i] = 1 << 29
    bad = build_attention_metadata(chunks, meta.slot_mapping, 16)
    ref = attend(q, *views, meta, SCALE)
    assert status() == 0
    got = attend(q, *views, bad, SCALE)
    assert status() == _capi.DEV_BAD_BLOCK
    assert torch.equal(got, ref)


def test_rows_without_a_sequence_keep_their_contents(cuda_device) -> None:
    """Strided q and out; rows that no chunk covers, and the columns between rows, stay as they were."""
    dev = cuda_device
    views, chunks, q = batch(dev, [(1, 70), (3, 40), (70, 3)], 2, seed=11)
    t = q.shape[0] + 4
    wide_q = torch.zeros(t, 4 * 128 + 8, device=dev, dtype=torch.bfloat16)
    wide_o = torch.full((t, 4 * 128 + 16), 3.0, device=dev, dtype=torch.bfloat16)
    qv, ov = (w[:, : 4 * 128].unflatten(1, (4, 128)) for w in (wide_q, wide_o))
    qv[: q.shape[0]] = q
    slots = torch.cat([slot_map(chunks, dev), torch.zeros(4, device=dev, dtype=torch.int64)])
    meta = build_attention_metadata(chunks, slots, 16)
    assert attend(qv, *views, meta, SCALE, out=ov).data_ptr() == wide_o.data_ptr()
    ref, bound, covered = attention64(q, *views, chunks, 2.0**-8)
    assert_close(ov, ref, bound, covered)
    assert bool((wide_o[q.shape[0] :] == 3.0).all()) and bool((wide_o[:, 4 * 128 :] == 3.0).all())


def test_attend_refuses(cuda_device) -> None:
    dev = cuda_device
    views, chunks, q = batch(dev, [(2, 70)], 2, seed=12)
    meta = build_attention_metadata(chunks, slot_map(chunks, dev), 16)
    with pytest.raises(ValueError, match="scale"):
        attend(q, *views, meta, 0.0)
    with pytest.raises(ValueError, match="rows"):
        attend(q[:1], *views, meta, SCALE)
    with pytest.raises(ValueError, match="num_heads"):
        attend(q[:, :3], *views, meta, SCALE, out=torch.empty_like(q)[:, :3])
    with pytest.raises(ValueError, match="the pool on"):
        attend(q.cpu(), *views, meta, SCALE, out=torch.empty_like(q))


# ---- streams, graphs, modules -----------------------------------------------------------------------


def test_another_stream_and_a_captured_graph(cuda_device) -> None:
    """paged_attention on a side stream, then captured and replayed twice with new inputs in its
    buffers (decode rows, a short chunk and a prompt chunk; the plan updated in place)."""
    dev = cuda_device
    views, chunks, q = batch(dev, [(1, 70), (20, 40), (90, 30), (1, 300)], 8, seed=13)
    t = q.shape[0]
    meta = build_attention_metadata(chunks, slot_map(chunks, dev), 16)
    k, v = rows(dev, t, 8, 31), rows(dev, t, 8, 32)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        eager = paged_attention(q, k, v, *views, meta, SCALE)
    torch.cuda.current_stream(dev).wait_stream(side)
    ref, bound, covered = attention64(q, *views, chunks, 2.0**-8)
    assert_close(eager, ref, bound, covered)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, k, v, *views, meta, SCALE)
    for seed in (41, 42):
        k.copy_(rows(dev, t, 8, seed))
        v.copy_(rows(dev, t, 8, seed + 10))
        q.copy_(rows(dev, t, 16, seed + 20))
        longer = [SeqChunk(c.flat_start, c.num_new, c.num_cached + (seed - 40 if c.num_new == 1 else 0),
                           c.block_table) for c in chunks]
        assert meta.update(longer, slot_map(longer, dev))
        graph.replay()
        ref, bound, covered = attention64(q, *views, longer, 2.0**-8)
        assert_close(out, ref, bound, covered)
        assert torch.equal(out, paged_attention(q, k, v, *views, meta, SCALE))
    fewer = chunks[:2] + [SeqChunk(21, 91, 30, chunks[2].block_table + [0]), chunks[3]]
    assert not meta.update(fewer)


def test_results_repeat_bit_for_bit(cuda_device) -> None:
    views, chunks, q = batch(cuda_device, [(1, 3000), (5, 900), (33, 100), (80, 20)], 4, seed=14)
    meta = build_attention_metadata(chunks, slot_map(chunks, cuda_device), 16)
    first = attend(q, *views, meta, SCALE)
    for _ in range(5):
        assert torch.equal(attend(q, *views, meta, SCALE), first)


def test_qwen3_attention_on_an_8_bit_pool(cuda_device) -> None:
    """The drop-in module with the fused projection asked for: an 8-bit pool takes the projection and
    kernel A, and its output is o_proj of the attention over the stored rows."""
    dev = cuda_device
    torch.manual_seed(0)
    cfg = SimpleNamespace(num_attention_heads=16, num_key_value_heads=8, head_dim=128,
                          hidden_size=256, rms_norm_eps=1e-6, fused_qkv=True)
    mod = Qwen3Attention(cfg).to(dev, torch.bfloat16)
    views, chunks, _ = batch(dev, [(1, 70), (5, 40), (70, 3)], 8, seed=15)
    t = sum(c.num_new for c in chunks)
    slots = slot_map(chunks, dev)
    meta = build_attention_metadata(chunks, slots, 16)
    cos_t, sin_t = rope_tables(128, 200, 1e6, dev)
    pos = torch.cat([torch.arange(c.num_cached, c.context_len) for c in chunks]).to(dev)
    x = torch.randn(t, 256, device=dev).bfloat16()
    with torch.no_grad():
        out = mod(x, cos_t[pos], sin_t[pos], *views, meta)
        q = qk_norm_rope_scatter(mod.qkv_proj(x), mod.q_norm.weight, mod.k_norm.weight, 1e-6,
                                 cos_t[pos], sin_t[pos], slots, *views, 16)
        att = check(views, chunks, q, u=2.0**-8)
        assert torch.equal(out, mod.o_proj(att.reshape(t, -1)))
