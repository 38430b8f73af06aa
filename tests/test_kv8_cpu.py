"""The 8-bit pool and the tree planner on the host: layout, the quantiser's definition, plans, and
what the entry points refuse (before any CUDA call)."""

from __future__ import annotations

import ctypes as C
import random

import numpy as np
import pytest
import torch

from miniserve_b200 import _capi, tree_positions
from miniserve_b200.attention import (SeqChunk, _plan_trees, _plan_with_kv8, attend, kv_gather,
                                      kv_scatter, plan_tree_batch)
from miniserve_b200.kv_pool import (KV8, KV8_PAGE_BYTES, _kv8_parts, allocate_kv_cache,
                                    check_layer_views, kv8_bytes_per_token, layer_as_slots,
                                    quantise_rows, slots_into_layer)
from paged_reference import tree_mask


def _pool(blocks: int = 5, kvh: int = 3):
    pool, views = allocate_kv_cache(2, blocks, kvh, "cpu", dtype=KV8)
    return pool, views[1]


def test_layout_and_size() -> None:
    pool, (k, v) = _pool()
    assert pool.shape == (2, 5, 3, KV8_PAGE_BYTES) and KV8_PAGE_BYTES == 4128
    assert check_layer_views(k, v, kv8=True) == (5, 3)
    assert v.data_ptr() - k.data_ptr() == 2048
    assert kv8_bytes_per_token(28, 8) == 2 * 28 * 8 * 129
    assert bool((layer_as_slots(k) == 0).all())
    # slot 37 = block 2, token 5; its 16-byte chunk 6 lies at chunk 6 ^ 3, its exponent in byte 5.
    x = torch.randn(80, 3, 128).bfloat16()
    slots_into_layer(k, x)
    codes, e = quantise_rows(x)
    got, exps = _kv8_parts(k)
    assert torch.equal(got[2, 1, 5, 6 ^ 3], codes[37, 1, 96:112].view(torch.uint8))
    assert exps[2, 1, 5] == e[37, 1]
    raw = pool[1, 2, 1].view(torch.uint8)
    assert raw[4096 + 5] == e[37, 1]


def test_views_of_the_other_kind_are_refused() -> None:
    _, (k, v) = _pool()
    with pytest.raises(ValueError, match="bf16"):
        check_layer_views(k, v)
    with pytest.raises(ValueError, match="V half"):
        check_layer_views(k, k, kv8=True)
    with pytest.raises(ValueError, match="strides"):
        check_layer_views(k[:, :2], v[:, :2], kv8=True)
    _, bf = allocate_kv_cache(1, 5, 3, "cpu")
    with pytest.raises(ValueError, match="V half"):
        check_layer_views(bf[0][0], bf[0][0], kv8=True)


@pytest.mark.parametrize("top,exponent", [
    (448.0, 0), (450.0, 1), (447.0, 0), (1.0, -8), (1.75, -8), (1.7578125, -7), (0.0, -100),
    (2.0**-133, -100), (3.3895313892515355e38, 120), (2.0**127, 119), (1.9921875 * 2**126, 119),
])
def test_exponent_is_the_smallest_that_fits(top: float, exponent: int) -> None:
    x = torch.zeros(1, 128).bfloat16()
    x[0, 7] = -top
    codes, b = quantise_rows(x)
    assert int(b[0]) - 127 == exponent
    held = codes.double() * 2.0**exponent
    assert bool(torch.isfinite(held.to(torch.bfloat16)).all())
    if exponent < 120 and top > 2.0**-60:
        assert abs(held[0, 7].item() + top) <= top * 2.0**-4  # half an e4m3 step


def test_quantised_values_are_within_half_a_step_and_stable() -> None:
    torch.manual_seed(0)
    x = (torch.randn(4096, 128) * torch.exp(3 * torch.randn(4096, 1))).bfloat16()
    codes, b = quantise_rows(x)
    scale = 2.0 ** (b.double() - 127)[:, None]
    held = codes.double() * scale
    # Half a step: 2^-4 of a normal code, 2^-10 of the scale below 2^-6.
    assert bool(((held - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0**-4,
                                                             scale * 2.0**-10)).all())
    assert torch.equal(held.to(torch.bfloat16).double(), held)  # reading back rounds nothing
    c2, b2 = quantise_rows(held.to(torch.bfloat16))
    assert torch.equal(c2.double() * 2.0 ** (b2.double() - 127)[:, None], held)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_row_with_a_non_finite_value_stands_for_nan(bad: float) -> None:
    _, (k, _) = _pool()
    x = torch.randn(80, 3, 128).bfloat16()
    x[4, 2, 100] = bad
    slots_into_layer(k, x)
    got = layer_as_slots(k)
    assert bool(got[4, 2].isnan().all()) and not bool(got[3].isnan().any())


# ---- plans ---------------------------------------------------------------------------------------


def _chunk(flat: int, n: int, c: int, first: int, parents=None) -> SeqChunk:
    return SeqChunk(flat, n, c, list(range(first, first + -(-(n + c) // 16))), parents=parents)


def _random_parents(rng: random.Random, n: int, unused: int = 0) -> list[int]:
    return [rng.randint(max(-1, i - 6), i - 1) for i in range(n - unused)] + [-2] * unused


@pytest.mark.parametrize("n", [1, 8, 16, 17, 31, 32, 33, 64, 100, 256])
@pytest.mark.parametrize("split", [0, 1, 3, 40])
def test_tree_plan_covers_every_page_once(n: int, split: int) -> None:
    """Every tile's pages are read once, by kernel F's items or (the cached whole 128-key blocks of trees
    of more than 16 drafts over 512 tokens and more, as the planner chooses) by tensor-core items; the partial rows of a
    combine record are those its items write."""
    rng = random.Random(n)
    chunks, flat, at = [], 0, 7
    for cached in (0, 15, 16, 511, 512, 700, 5000):
        parents = _random_parents(rng, n, unused=n // 5)
        c = _chunk(flat, n, cached, at, parents)
        at += len(c.block_table)
        flat += n
        chunks.append(c)
    packed, info = plan_tree_batch(chunks, flat, 16, 148, split)
    assert packed.size == info.total_ints
    count = len(chunks)
    # (Without a given split, trees of up to 32 drafts keep their cached blocks where that is faster.)
    could = n > 16 and (n > 32 or split > 0 or info.n_tc_items > 0)
    has_prefix = [could and c.num_cached >= 512 for c in chunks]
    seqs = packed[: (count + sum(has_prefix)) * 8].reshape(-1, 8)
    narrow = packed[info.off_decode :][: 8 * info.n_decode_items].reshape(-1, 8)
    wide = packed[info.off_tile :][: 8 * info.n_tile_items].reshape(-1, 8)
    tcs = packed[info.off_tc :][: 8 * info.n_tc_items].reshape(-1, 8)
    combine = packed[info.off_combine :][: 8 * info.n_combine].reshape(-1, 8)
    assert all(it[2] <= 16 for it in narrow) and all(16 < it[2] <= 32 for it in wide)
    pages: dict[tuple[int, int], list[int]] = {}
    written: dict[int, int] = {}  # partial row -> how often
    arrive = [0] * info.n_combine
    for s, tok0, nq, pb, pe, part, rec, flag in np.concatenate([narrow, wide]).tolist():
        assert tok0 % 32 == 0 and pb < pe and (part >= 0) == (flag != 0)
        pages.setdefault((s, tok0), []).extend(range(pb, pe))
        if part >= 0:
            assert flag == (3 if has_prefix[s] else 2)
            assert combine[rec, :3].tolist() == [s, tok0, nq]
            arrive[rec] += 1
            for r in range(2 * nq):
                written[part + r] = written.get(part + r, 0) + 1
    for vs, tok0, nq, pb, pe, part, tok_b, n_b in tcs.tolist():
        s = [i for i in range(count) if has_prefix[i]][vs - count]
        assert seqs[vs, 0] == chunks[s].flat_start and seqs[vs, 4] == seqs[s, 4]
        assert seqs[vs, 2] == chunks[s].num_cached // 128 * 128
        assert n_b == 0 and tok0 % 64 == 0 and nq == min(64, n - tok0)
        assert pb % 8 == 0 and pe % 8 == 0 and pb < pe and pe * 16 <= chunks[s].num_cached
        for t0 in range(tok0, tok0 + nq, 32):
            pages.setdefault((s, t0), []).extend(range(pb, pe))
        for r in range(2 * nq):
            written[part + r] = written.get(part + r, 0) + 1
    assert set(written.values()) <= {1} and len(written) == info.part_rows
    merged: dict[int, int] = {}
    for k, (s, tok0, nq, row0, parts, stride, arrivals, _) in enumerate(combine.tolist()):
        assert arrivals == arrive[k] and (parts == arrivals or has_prefix[s])
        for p in range(parts):
            for r in range(2 * nq):
                merged[row0 + p * stride + r] = 1
    assert merged == written
    for i, c in enumerate(chunks):
        assert seqs[i, 0] == c.flat_start and seqs[i, 2] == c.num_cached
        for tok0 in range(0, n, 32):
            last = c.num_cached + min(n, tok0 + 32)
            assert sorted(pages[(i, tok0)]) == list(range(-(-last // 16)))
        words = int(seqs[i, 7])
        mask = packed[seqs[i, 6] : seqs[i, 6] + n * words].view(np.uint32).reshape(n, words)
        bits = np.unpackbits(mask.view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
        assert np.array_equal(bits, tree_mask(c.parents).numpy())
        tab = packed[info.off_tables + seqs[i, 4] :][: len(c.block_table)]
        assert tab.tolist() == c.block_table


@pytest.mark.parametrize("n", [1, 16, 17, 48, 100])
@pytest.mark.parametrize("split", [0, 1, 3, 40])
def test_tree_plans_kv8_part_covers_every_page_once(n: int, split: int) -> None:
    """Over an 8-bit pool kernel F reads every page of a tile itself, larger trees' cached blocks too."""
    chunks, flat, at = [], 0, 7
    for cached in (0, 15, 511, 512, 5000):
        chunks.append(_chunk(flat, n, cached, at, list(range(-1, n - 1))))
        at += len(chunks[-1].block_table)
        flat += n
    packed, info, kv8 = _plan_trees(chunks, flat, 148, split, _capi.MsKv8Info())
    assert packed.size == kv8.total_ints >= info.total_ints and kv8.n_pages == 0
    items = [packed[off:][: 8 * count].reshape(-1, 8)
             for off, count in ((kv8.off_narrow, kv8.n_narrow), (kv8.off_wide, kv8.n_wide))]
    assert all(it[2] <= 16 for it in items[0]) and all(16 < it[2] <= 32 for it in items[1])
    combine = packed[kv8.off_combine :][: 8 * kv8.n_combine].reshape(-1, 8)
    pages: dict[tuple[int, int], list[int]] = {}
    used: set[int] = set()
    arrive = [0] * kv8.n_combine
    for s, tok0, nq, pb, pe, part, rec, flag in np.concatenate(items).tolist():
        pages.setdefault((s, tok0), []).extend(range(pb, pe))
        assert (part >= 0) == (flag == 2) and flag in (0, 2)
        if part >= 0:
            k = (part - combine[rec, 3]) // (2 * nq)
            assert combine[rec, :3].tolist() == [s, tok0, nq] and combine[rec, 5] == 2 * nq
            assert 0 <= k < combine[rec, 4] and (part - combine[rec, 3]) % (2 * nq) == 0
            rows = set(range(part, part + 2 * nq))
            assert not rows & used and max(rows) < info.part_rows + kv8.part_rows
            used |= rows
            arrive[rec] += 1
    assert arrive == combine[:, 4].tolist() == combine[:, 6].tolist()
    for i, c in enumerate(chunks):
        for tok0 in range(0, n, 32):
            last = c.num_cached + min(n, tok0 + 32)
            assert sorted(pages.pop((i, tok0))) == list(range(-(-last // 16)))
    assert not pages


@pytest.mark.parametrize("parents,what", [
    ([-1, 1, 0], "draft 1 has parent 1"), ([0, -1], "draft 0 has parent 0"),
    ([-1, -3], "draft 1 has parent -3"), ([-2, 0], "draft 1 has parent 0"), ([-1, 2, -1], "draft 1"),
])
def test_tree_plan_refuses_bad_parents(parents, what: str) -> None:
    with pytest.raises(ValueError, match=what):
        plan_tree_batch([_chunk(0, len(parents), 20, 0, parents)], len(parents))


def test_tree_plan_refuses_bad_batches() -> None:
    with pytest.raises(ValueError, match="one parent per new token"):
        plan_tree_batch([_chunk(0, 3, 20, 0, [-1, 0])], 3)
    with pytest.raises(ValueError, match="blocks"):
        plan_tree_batch([SeqChunk(0, 2, 40, [1, 2], parents=[-1, 0])], 2)
    with pytest.raises(ValueError, match="flat_start"):
        plan_tree_batch([_chunk(1, 2, 4, 0, [-1, 0])], 2)
    with pytest.raises(ValueError, match="more than 1024"):
        plan_tree_batch([_chunk(0, 1025, 0, 0, [-1] * 1025)], 1025)
    none = plan_tree_batch([], 0)[1]
    assert none.n_tile_items == 0 and none.n_decode_items == 0


def test_tree_plan_reports_a_small_buffer() -> None:
    lib = _capi.load()
    one = np.array([1], np.int32)
    zero = np.zeros(1, np.int32)
    off = np.array([0, 1], np.int64)
    out = np.empty(4, np.int32)
    rc = lib.ms_tree_plan_build(1, zero.ctypes.data, one.ctypes.data, zero.ctypes.data,
                                off.ctypes.data, zero.ctypes.data, (-one).ctypes.data, 1, 16, 148, 0,
                                out.ctypes.data, out.size, C.byref(_capi.MsPlanInfo()))
    assert rc == _capi.MS_ERR_CAPACITY


def test_tree_positions_are_depths() -> None:
    assert tree_positions(100, [-1, 0, 0, 1, -1, 4, -2]) == [100, 101, 101, 102, 100, 101, 100]


def test_kv8_part_maps_every_page_of_tensor_core_items() -> None:
    """The expanded pages: each tensor-core record's table becomes a run of the identity, and the map
    gives the pool blocks in the same order; other records keep their tables."""
    chunks, flat, at = [], 0, 3
    for n, c in ((1, 50), (200, 70), (8, 3), (65, 0), (30, 9)):
        chunks.append(_chunk(flat, n, c, at))
        at += len(chunks[-1].block_table)
        flat += n
    packed, info, kv8 = _plan_with_kv8(chunks, flat, 148, 0)
    assert kv8.n_pages == -(-270 // 16) + -(-65 // 16)
    assert kv8.off_seqs >= info.total_ints and packed.size == kv8.total_ints
    seqs = packed[kv8.off_seqs :][: len(chunks) * 8].reshape(-1, 8)
    plain = packed[info.off_seqs :][: len(chunks) * 8].reshape(-1, 8)
    for i, c in enumerate(chunks):
        if c.num_new > 64:
            tab = packed[kv8.off_tables + seqs[i, 4] :][: len(c.block_table)]
            assert packed[kv8.off_map + tab].tolist() == c.block_table
            assert np.array_equal(np.delete(seqs[i], [4, 5]), np.delete(plain[i], [4, 5]))
        else:
            assert np.array_equal(seqs[i], plain[i])
    lib = _capi.load()
    need = lib.ms_kv8_workspace_bytes(C.byref(info), C.byref(kv8), 8)
    part = ((info.part_rows + kv8.part_rows) * 129 * 4 + 4 * kv8.n_combine) * 8
    assert need == -(-part // 1024) * 1024 + kv8.n_pages * 8 * 8192
    _, short, none = _plan_with_kv8(chunks[:1], 1, 148, 0)
    assert none.n_pages == 0 and short.n_tc_items == 0


def test_kv8_struct_matches_the_header() -> None:
    assert C.sizeof(_capi.MsKv8Info) == 56


@pytest.mark.parametrize("split", [0, 1, 3])
def test_kv8_part_covers_every_row_once(split: int) -> None:
    """Kernel F's items over an 8-bit pool: every tile of up to 32 tokens of the sequences with up to
    64 new ones reads its pages once, splits name their record; cascade rows read their own pages."""
    chunks, flat, at = [], 0, 3
    for n, c in [(1, 0), (1, 4000), (8, 15), (16, 16), (17, 40), (33, 700), (64, 3), (65, 20)]:
        chunks.append(_chunk(flat, n, c, at))
        at += len(chunks[-1].block_table)
        flat += n
    prefix = list(range(at, at + 20))
    at += 20
    for i in range(16):
        own = list(range(at, at + 3))
        at += 3
        chunks.append(SeqChunk(flat, 5, 330 + i, prefix + own))
        flat += 5
    packed, info, kv8 = _plan_with_kv8(chunks, flat, 148, split)
    assert info.n_cascade == 1
    items = np.concatenate([packed[kv8.off_narrow :][: 8 * kv8.n_narrow].reshape(-1, 8),
                            packed[kv8.off_wide :][: 8 * kv8.n_wide].reshape(-1, 8)])
    combine = packed[kv8.off_combine :][: 8 * kv8.n_combine].reshape(-1, 8)
    pages: dict[tuple[int, int], list[int]] = {}
    used: set[int] = set()
    for s, tok0, nq, pb, pe, part, f6, f7 in items.tolist():
        pages.setdefault((s, tok0), []).extend(range(pb, pe))
        if f7 == 2:
            assert combine[f6, :3].tolist() == [s, tok0, nq] and combine[f6, 5] == 2 * nq
            rows = set(range(part, part + 2 * nq))
            assert min(rows) >= info.part_rows and max(rows) < info.part_rows + kv8.part_rows
            assert not rows & used
            used |= rows
        else:
            assert part == -1 and f7 == (1 if s >= 8 else 0)
    want = {}
    for i, c in enumerate(chunks):
        for tok0 in range(0, c.num_new if c.num_new <= 64 else 0, 32):
            last = c.num_cached + min(c.num_new, tok0 + 32)
            want[(i, tok0)] = list(range(20 if i >= 8 else 0, -(-last // 16)))
    assert {k: sorted(v) for k, v in pages.items()} == want


# ---- refusals, before any CUDA call -----------------------------------------------------------------


def test_entry_points_refuse_bad_arguments() -> None:
    lib = _capi.load()
    buf = torch.zeros(8192, dtype=torch.uint8)
    p = (buf.data_ptr() + 15) // 16 * 16
    assert lib.ms_kv_scatter_kv8(p, 128, p, 128, -1, 1, p, p, 1, None) == _capi.MS_ERR_ARG
    assert lib.ms_kv_scatter_kv8(p, 128, p, 128, 1, 1, p, None, 1, None) == _capi.MS_ERR_ARG
    assert lib.ms_kv_scatter_kv8(p, 128, p, 128, 1, 1, p, p + 8, 1, None) == _capi.MS_ERR_LAYOUT
    assert lib.ms_kv_scatter_kv8(p, 120, p, 128, 1, 1, p, p, 1, None) == _capi.MS_ERR_ARG
    assert lib.ms_kv_scatter_kv8(p + 2, 128, p, 128, 1, 1, p, p, 1, None) == _capi.MS_ERR_ARG
    assert lib.ms_kv_gather_kv8(p, 1, 1, p, 1, p, 128, p + 8, 128, None) == _capi.MS_ERR_ARG
    assert lib.ms_kv_gather(p, 1, 1, p, p, 1, p, 128, p, 128, None) == _capi.MS_ERR_LAYOUT
    assert lib.ms_kv_gather_kv8(p, 0, 1, None, 0, None, 0, None, 0, None) == _capi.MS_OK
    assert lib.ms_qk_norm_rope_scatter_kv8(None, 0, 4, 15, 8, None, None, 1e-6, None, None, 0, None,
                                           0, None, None, 0, None, 0, None) == _capi.MS_ERR_ARG
    _, info = plan_tree_batch([_chunk(0, 2, 4, 0, [-1, 0])], 2)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        rc = lib.ms_tree_attention(p, 256, p, 256, 2, 1, p, p, 1, p, C.byref(info), None, 0, scale,
                                   None)
        assert rc == _capi.MS_ERR_ARG and b"scale" in lib.ms_last_error()
    rc = lib.ms_tree_attention(p, 256, p, 256, 3, 1, p, p, 1, p, C.byref(info), None, 0, 1.0, None)
    assert rc == _capi.MS_ERR_ARG and b"num_heads" in lib.ms_last_error()
    args = (p, 256, p, 256, 2, 1, p, 1, p, C.byref(info))
    rc = lib.ms_tree_attention_kv8(*args, None, None, 0, 1.0, None)
    assert rc == _capi.MS_ERR_ARG and b"8-bit part" in lib.ms_last_error()
    rc = lib.ms_paged_attention_kv8(*args, None, None, 0, 1.0, None)
    assert rc == _capi.MS_ERR_ARG and b"ms_tree_plan_build" in lib.ms_last_error()
    rc = lib.ms_paged_attention(p, 256, p, 256, 2, 1, p, p, 1, p, C.byref(info), None, 0, 1.0, None)
    assert rc == _capi.MS_ERR_ARG and b"ms_tree_plan_build" in lib.ms_last_error()
    _, info, kv8 = _plan_with_kv8([_chunk(0, 100, 4, 0)], 100, 148, 0)
    args = (p, 256, p, 256, 2, 1, p, 1, p, C.byref(info))
    rc = lib.ms_tree_attention_kv8(*args, C.byref(kv8), None, 0, 1.0, None)
    assert rc == _capi.MS_ERR_ARG and b"ms_tree_plan_build" in lib.ms_last_error()
    rc = lib.ms_paged_attention_kv8(*args, None, None, 0, 1.0, None)
    assert rc == _capi.MS_ERR_ARG and b"8-bit part" in lib.ms_last_error()
    rc = lib.ms_paged_attention_kv8(*args, C.byref(kv8), None, 0, 1.0, None)
    assert rc == _capi.MS_ERR_ARG and b"workspace" in lib.ms_last_error()


def test_python_wrappers_refuse_bad_arguments() -> None:
    _, (k_cache, v_cache) = _pool()
    k = torch.zeros(4, 3, 128, dtype=torch.bfloat16)
    slots = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="4 rows but 3 slots"):
        kv_scatter(k, k, slots[:3], k_cache, v_cache)
    with pytest.raises(ValueError, match="int64"):
        kv_scatter(k, k, slots.int(), k_cache, v_cache)
    with pytest.raises(ValueError, match=r"\[T, 3, 128\]"):
        kv_scatter(k[:, :2], k[:, :2], slots, k_cache, v_cache)
    with pytest.raises(RuntimeError, match="CUDA only"):
        kv_scatter(k, k, slots, k_cache, v_cache)
    with pytest.raises(RuntimeError, match="CUDA only"):
        kv_gather(slots, k_cache, v_cache)
    with pytest.raises(ValueError, match="int64"):
        kv_gather(slots.int(), k_cache, v_cache)
    with pytest.raises(ValueError, match="V half"):
        attend(torch.zeros(1, 6, 128), k_cache, k_cache, None, 1.0)
