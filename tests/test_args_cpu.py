"""Calls over a bf16 pool whose tensors do not fit each other are refused before anything is launched
(the 8-bit pool's refusals are in test_kv8_cpu.py)."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import _capi
from miniserve_b200.attention import (AttentionMetadata, SeqChunk, attend,
                                      build_attention_metadata, kv_gather, kv_scatter, plan_batch)
from miniserve_b200.kv_pool import KV8, allocate_kv_cache
from miniserve_b200.qwen3_attention import qk_norm_rope_scatter, qkv_proj_norm_rope_scatter

KVH = 8


class NoLaunch:
    """The library with every entry point answering as if it had launched."""

    def __init__(self) -> None:
        self.calls: list[str] = []

    def __getattr__(self, name: str):
        def call(*args):
            self.calls.append(name)
            return _capi.MS_OK
        return call


@pytest.fixture
def lib(monkeypatch):
    """CPU tensors pass for the GPU's; nothing runs."""
    from miniserve_b200 import attention, qwen3_attention

    fake = NoLaunch()
    monkeypatch.setattr(_capi, "load", lambda path=None: fake)
    monkeypatch.setattr(attention, "_stream", lambda device: 0)
    monkeypatch.setattr(qwen3_attention, "_stream", lambda device: 0)
    return fake


def views(dtype=torch.bfloat16, device="cpu"):
    return allocate_kv_cache(1, 4, KVH, torch.device(device), dtype=dtype)[1][0]


def rows(n: int, heads: int = KVH) -> torch.Tensor:
    return torch.zeros(n, heads, 128, dtype=torch.bfloat16)


def test_scatter_and_gather(lib) -> None:
    pool = views()
    slots = torch.zeros(4, dtype=torch.int64)
    kv_scatter(rows(4), rows(4), slots, *pool)
    kv_scatter(rows(3), rows(3), slots, *pool)  # a longer slot mapping, as in a padded step
    assert lib.calls == ["ms_kv_scatter"] * 2
    bad = [
        (rows(5), rows(5), slots, "5 rows but 4 slots"),
        (rows(4), rows(3), slots, r"\[T, 8, 128\]"),
        (rows(4), rows(5), slots, r"\[T, 8, 128\]"),
        (rows(4, 7), rows(4, 7), slots, r"\[T, 8, 128\]"),
        (rows(4, 16), rows(4, 16), slots, r"\[T, 8, 128\]"),
        (rows(4), rows(4), slots.int(), "int64"),
        (rows(4), rows(4), torch.zeros(8, dtype=torch.int64)[::2], "contiguous"),
        (rows(4).float(), rows(4).float(), slots, "bf16"),
    ]
    for k, v, s, what in bad:
        with pytest.raises(ValueError, match=what):
            kv_scatter(k, v, s, *pool)
    with pytest.raises(ValueError, match="slots"):
        kv_gather(slots, *pool, k_out=rows(3), v_out=rows(3))
    with pytest.raises(ValueError, match="int64"):
        kv_gather(slots.int(), *pool)
    assert lib.calls == ["ms_kv_scatter"] * 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, KV8])
def test_kernel_a(dtype, lib) -> None:
    pool = views(dtype)
    qkv = torch.zeros(4, 4096, dtype=torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16)
    table = torch.zeros(4, 128)
    slots = torch.zeros(4, dtype=torch.int64)

    def call(qkv=qkv, w=w, cos=table, sin=table, slots=slots, **kw):
        return qk_norm_rope_scatter(qkv, w, w, 1e-6, cos, sin, slots, *pool, 16, **kw)

    call()
    call(positions=slots, q_out=rows(5, 16))
    n = len(lib.calls)
    assert n == 2
    bad = [
        (dict(slots=slots[:3]), "4 rows but slot_mapping has 3"),
        (dict(slots=slots.int()), "slot_mapping must be contiguous int64"),
        (dict(slots=torch.zeros(8, dtype=torch.int64)[::2]), "contiguous"),
        (dict(positions=slots[:1]), "4 rows but positions has 1"),
        (dict(positions=slots.int()), "positions must be contiguous int64"),
        (dict(w=w[:64]), "128 values"),
        (dict(cos=table, sin=table[:2]), "same positions"),
        (dict(cos=table[:, :64], sin=table[:, :64]), "rows of 128"),
        (dict(q_out=rows(3, 16)), "q_out"),
        (dict(q_out=rows(4, 8)), "q_out"),
    ]
    for kw, what in bad:
        with pytest.raises(ValueError, match=what):
            call(**kw)
    assert len(lib.calls) == n


def test_kernel_e(lib) -> None:
    pool = views()
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    weight = torch.zeros(4096, 256, dtype=torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16)
    table = torch.zeros(4, 128)
    slots = torch.zeros(4, dtype=torch.int64)
    qkv_proj_norm_rope_scatter(x, weight, w, w, 1e-6, table, table, slots, *pool, 16)
    for s, kw, what in ((slots[:3], {}, "4 rows but"), (slots.int(), {}, "int64"),
                        (slots, {"q_out": rows(2, 16)}, "q_out")):
        with pytest.raises(ValueError, match=what):
            qkv_proj_norm_rope_scatter(x, weight, w, w, 1e-6, table, table, s, *pool, 16, **kw)
    assert len(lib.calls) == 1


def _meta(chunks: list[SeqChunk], num_tokens: int) -> AttentionMetadata:
    packed, info = plan_batch(chunks, num_tokens)
    return AttentionMetadata(torch.zeros(num_tokens, dtype=torch.int64), torch.from_numpy(packed), info,
                             num_tokens, _packed=packed)


def test_attend(monkeypatch) -> None:
    from miniserve_b200 import attention

    pool = views()
    # Five slots, of which the step's sequences use three rows.
    meta = _meta([SeqChunk(0, 1, 20, [0, 1]), SeqChunk(1, 2, 3, [2])], 5)
    fake = NoLaunch()
    monkeypatch.setattr(_capi, "load", lambda path=None: fake)
    monkeypatch.setattr(attention, "_stream", lambda device: 0)
    attend(rows(5, 16), *pool, meta, 1.0)
    attend(rows(3, 16), *pool, meta, 1.0)
    attend(rows(9, 16), *pool, meta, 1.0, out=rows(3, 16))
    n = len(fake.calls)
    for q, out, what in (
        (rows(2, 16), None, "3 rows"),
        (rows(5, 16), rows(2, 16), "3 rows"),
        (rows(5, 16), rows(5, 8), "heads"),
        (rows(5, 16).float(), None, "bf16"),
    ):
        with pytest.raises(ValueError, match=what):
            attend(q, *pool, meta, 1.0, out=out)
    assert len(fake.calls) == n


def test_without_a_gpu() -> None:
    pool = views()
    slots = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA only"):
        kv_scatter(rows(4), rows(4), slots, *pool)
    with pytest.raises(RuntimeError, match="CUDA only"):
        kv_gather(slots, *pool)
    with pytest.raises(RuntimeError, match="CUDA only"):
        attend(rows(4, 16), *pool, _meta([SeqChunk(0, 1, 20, [0, 1])], 4), 1.0)


@pytest.mark.gpu
def test_tensors_on_the_host(cuda_device) -> None:
    """A host tensor among device ones is refused."""
    pool = views(device=cuda_device)
    qkv = torch.zeros(4, 4096, dtype=torch.bfloat16, device=cuda_device)
    w = torch.ones(128, dtype=torch.bfloat16, device=cuda_device)
    table = torch.zeros(4, 128, device=cuda_device)
    slots = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    for kw in (dict(slots=slots.cpu()), dict(w=w.cpu()), dict(cos=table.cpu()), dict(qkv=qkv.cpu())):
        args = dict(qkv=qkv, w=w, cos=table, slots=slots) | kw
        with pytest.raises(ValueError, match="pool's device"):
            qk_norm_rope_scatter(args["qkv"], args["w"], args["w"], 1e-6, args["cos"], args["cos"],
                                 args["slots"], *pool, 16)
    k = rows(4).to(cuda_device)
    for a, s in ((k, slots.cpu()), (k.cpu(), slots)):
        with pytest.raises(ValueError, match="the pool on"):
            kv_scatter(a, a, s, *pool)
    q = rows(4, 16).to(cuda_device)
    meta = build_attention_metadata([SeqChunk(0, 1, 20, [0, 1])], slots, 16)
    for a, out in ((q.cpu(), q), (q, q.cpu())):
        with pytest.raises(ValueError, match="the pool on"):
            attend(a, *pool, meta, 1.0, out=out)
