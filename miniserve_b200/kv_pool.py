"""The paged KV pool in the layout the sm_100a kernels read.

Replaces ``ModelRunner.allocate_kv_cache`` (src/miniserve/runner/model_runner.py:77-94).  The
reference pool is ``[layers, 2, slots, kv_heads, head_dim]``: one token's heads are contiguous,
so one KV head's 16-token block is 16 scattered 256-byte rows.  Here the pool is

    [layers, num_blocks, kv_heads, 2 (K, V), 2 (d // 64), 16 (token), 64 (d % 64)]  bf16

so that K and V of one (block, head) form one contiguous 8 KiB page pair that a single TMA box
moves into shared memory, already split into 128-byte rows for the swizzled layout the tensor
cores read.  Slot semantics are unchanged: slot = block * 16 + offset in the block.

Like the reference, the pool is zero-filled: masked-out keys of a partial last block are still
multiplied by a zero weight, and uninitialised memory could hold NaN bit patterns.

The 8-bit pool (``dtype=torch.float8_e4m3fn``) holds every (token, KV head) row of K and of V as 128
e4m3 codes and one exponent byte, 129 bytes instead of 256:

    [layers, num_blocks, kv_heads, 4128]   (K: 16 rows of 128 codes; V: the same; 16 + 16 exponents)

A row with exponent byte b stands for its codes times 2^(b - 127); b is chosen when the row is written
(``kv_scatter``, kernel A), from the row's largest magnitude.  The 16-byte chunks of row t are stored
at chunk ^ (t % 2 + 2 (t // 4)), which the kernels read without bank conflicts; ``layer_as_slots`` gives the
values a layer stands for.  Attention takes V rows of any finite sizes side by side: a key's share is lost
only where its softmax weight is below fp32's range (2^-126 of the row's largest), or where it adds less than
2^-25 of the row's largest share.  (Chunks of more than 64 tokens, which run over bf16 copies of the pages,
may overflow where they see V rows beyond 2^119, as over a bf16 pool.)
"""

from __future__ import annotations

import torch
from torch import Tensor

BLOCK_SIZE = 16
HEAD_DIM = 128
KV8 = torch.float8_e4m3fn  # dtype of an 8-bit pool
KV8_ROWS_BYTES = BLOCK_SIZE * HEAD_DIM  # K (or V) codes of one (block, head)
KV8_PAGE_BYTES = 2 * KV8_ROWS_BYTES + 2 * BLOCK_SIZE  # with the exponent bytes


def kv_bytes_per_token(num_layers: int, num_kv_heads: int, head_dim: int = HEAD_DIM,
                       dtype_bytes: int = 2) -> int:
    """K and V of every layer for one token (qwen3.py:60-62): 112 KiB for Qwen3-0.6B in bf16."""
    return 2 * num_layers * num_kv_heads * head_dim * dtype_bytes


def kv8_bytes_per_token(num_layers: int, num_kv_heads: int) -> int:
    """The same for an 8-bit pool: 128 codes and an exponent byte per row (56.4 KiB for Qwen3-0.6B)."""
    return 2 * num_layers * num_kv_heads * (HEAD_DIM + 1)


_kv8_allocated = False


def kv8_in_use() -> bool:
    """Whether this process has allocated an 8-bit pool: steps are then planned for both kinds of
    pool, else for bf16 ones only (a step of cascade groups takes a tenth less to plan and upload)."""
    return _kv8_allocated


def allocate_kv_cache(
    num_layers: int,
    num_blocks: int,
    num_kv_heads: int,
    device: torch.device | str,
    dtype: torch.dtype = torch.bfloat16,
    zero: bool = True,
) -> tuple[Tensor, list[tuple[Tensor, Tensor]]]:
    """Allocate the pool and return ``(pool, [(k_cache, v_cache) per layer])``.

    Each per-layer view has shape ``[num_blocks, kv_heads, 2, 16, 64]``; ``v_cache`` starts
    4 KiB after ``k_cache`` inside every (block, head) page pair.  With
    ``dtype=torch.float8_e4m3fn`` the pool is the 8-bit one and a layer's views are
    ``[num_blocks, kv_heads, 16, 128]`` e4m3 codes (their exponent bytes lie behind them in the pool):
    every function that takes a layer's views takes either kind, except the fused projection.
    """
    if dtype == KV8:
        global _kv8_allocated
        _kv8_allocated = True
        raw = (torch.zeros if zero else torch.empty)(
            (num_layers, num_blocks, num_kv_heads, KV8_PAGE_BYTES), dtype=torch.uint8,
            device=device)
        pool = raw.view(KV8)
        size = (num_blocks, num_kv_heads, BLOCK_SIZE, HEAD_DIM)
        stride = (num_kv_heads * KV8_PAGE_BYTES, KV8_PAGE_BYTES, HEAD_DIM, 1)
        layer = num_blocks * num_kv_heads * KV8_PAGE_BYTES
        return pool, [(pool.as_strided(size, stride, i * layer),
                       pool.as_strided(size, stride, i * layer + KV8_ROWS_BYTES))
                      for i in range(num_layers)]
    if dtype != torch.bfloat16:
        raise ValueError("the sm_100a kernels read a bf16 pool, or an 8-bit one (torch.float8_e4m3fn)")
    shape = (num_layers, num_blocks, num_kv_heads, 2, 2, BLOCK_SIZE, HEAD_DIM // 2)
    pool = (torch.zeros if zero else torch.empty)(shape, dtype=dtype, device=device)
    views = [(pool[i, :, :, 0], pool[i, :, :, 1]) for i in range(num_layers)]
    return pool, views


def is_kv8(k_cache: Tensor) -> bool:
    """Whether a layer's view belongs to an 8-bit pool."""
    return k_cache is not None and k_cache.dtype == KV8


def _check_kv8_views(k_cache: Tensor, v_cache: Tensor) -> tuple[int, int]:
    shape = k_cache.shape
    if len(shape) != 4 or shape[2] != BLOCK_SIZE or shape[3] != HEAD_DIM:
        raise ValueError(
            "k_cache must be a layer view of miniserve_b200.kv_pool.allocate_kv_cache "
            f"([blocks, kv_heads, 16, 128] of an 8-bit pool); got shape {tuple(shape)}"
        )
    nb, kvh = shape[0], shape[1]
    want = (kvh * KV8_PAGE_BYTES, KV8_PAGE_BYTES, HEAD_DIM, 1)
    if k_cache.stride() != want or v_cache.stride() != want:
        raise ValueError(f"KV pool views have strides {k_cache.stride()}, expected {want}")
    if (v_cache.dtype != KV8 or v_cache.shape != shape
            or v_cache.data_ptr() != k_cache.data_ptr() + KV8_ROWS_BYTES):
        raise ValueError("v_cache must be the V half of the same pool as k_cache")
    return nb, kvh


def check_layer_views(k_cache: Tensor, v_cache: Tensor, kv8: bool = False) -> tuple[int, int]:
    """Validate one layer's (k_cache, v_cache) views; return ``(num_blocks, num_kv_heads)``.  An
    8-bit pool's views pass only where the caller says it takes them (``kv8``)."""
    if kv8 and is_kv8(k_cache):
        return _check_kv8_views(k_cache, v_cache)
    if k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise ValueError("KV pool views must be bf16")
    shape = k_cache.shape
    if len(shape) != 5 or shape[2:] != (2, BLOCK_SIZE, HEAD_DIM // 2):
        raise ValueError(
            "k_cache must be a layer view of miniserve_b200.kv_pool.allocate_kv_cache "
            f"([blocks, kv_heads, 2, 16, 64]); got shape {tuple(shape)}"
        )
    nb, kvh = shape[0], shape[1]
    page = BLOCK_SIZE * HEAD_DIM  # elements of one K (or V) page
    want = (kvh * 2 * page, 2 * page, page // 2, HEAD_DIM // 2, 1)
    if k_cache.stride() != want or v_cache.stride() != want:
        raise ValueError(f"KV pool views have strides {k_cache.stride()}, expected {want}")
    if v_cache.shape != shape or v_cache.data_ptr() != k_cache.data_ptr() + 2 * page:
        raise ValueError("v_cache must be the V half of the same pool as k_cache")
    return nb, kvh


def _kv8_parts(view: Tensor) -> tuple[Tensor, Tensor]:
    """Codes ``[blocks, kv_heads, 16, 8, 16]`` (uint8, chunks as stored) and exponent bytes ``[blocks,
    kv_heads, 16]`` of a K or V view of an 8-bit pool, both sharing its memory."""
    nb, kvh = view.shape[0], view.shape[1]
    pos = view.storage_offset() % KV8_PAGE_BYTES  # 0: K, KV8_ROWS_BYTES: V
    if pos not in (0, KV8_ROWS_BYTES):
        raise ValueError("not a K or V view of an 8-bit pool")
    base = view.view(torch.uint8)
    codes = base.unflatten(-1, (8, 16))
    at = view.storage_offset() - pos + 2 * KV8_ROWS_BYTES + (BLOCK_SIZE if pos else 0)
    exps = base.as_strided((nb, kvh, BLOCK_SIZE), (kvh * KV8_PAGE_BYTES, KV8_PAGE_BYTES, 1), at)
    return codes, exps


def _kv8_order(device: torch.device) -> Tensor:
    """``[16, 8]``: where row t's chunk i is stored (i ^ (t % 2 + 2 (t // 4)))."""
    t = torch.arange(BLOCK_SIZE, device=device)[:, None]
    return torch.arange(8, device=device)[None, :] ^ (t % 2 + 2 * (t // 4))


def layer_as_slots(view: Tensor) -> Tensor:
    """A copy of one layer's K (or V) view in the reference layout ``[slots, kv_heads, 128]`` (bf16;
    for an 8-bit pool the values its rows stand for)."""
    nb, kvh = view.shape[0], view.shape[1]
    if is_kv8(view):
        codes, exps = _kv8_parts(view)
        order = _kv8_order(view.device)[None, None, :, :, None].expand_as(codes)
        vals = torch.gather(codes, 3, order).flatten(-2).view(KV8).float()
        scale = (exps.to(torch.int32) << 23).view(torch.float32)  # 2^(b - 127); 255: infinity
        vals = (vals * scale[..., None]).to(torch.bfloat16)
        vals = torch.where((exps == 255)[..., None], float("nan"), vals)
        return vals.permute(0, 2, 1, 3).reshape(nb * BLOCK_SIZE, kvh, HEAD_DIM)
    return view.permute(0, 3, 1, 2, 4).reshape(nb * BLOCK_SIZE, kvh, HEAD_DIM)


def quantise_rows(x: Tensor) -> tuple[Tensor, Tensor]:
    """The 8-bit form of rows ``[..., 128]``: e4m3 codes and exponent bytes (uint8), as the kernels
    store them.  The exponent e = b - 127 is the smallest integer in [-100, 120] with max|x| 2^-e <=
    448; a row with a NaN or an infinity gets b = 255 and zero codes."""
    y = x.float()
    ok = torch.isfinite(y).all(-1)
    y = torch.where(ok[..., None], y, 0.0)
    mant, expo = torch.frexp(y.abs().amax(-1))  # 448 = 0.875 * 2^9
    e = (expo - 9 + (mant > 0.875).to(expo.dtype)).clamp(-100, 120)
    e = torch.where(mant == 0, -100, e)
    limit = torch.where(e == 120, 240.0, 448.0)[..., None]  # c 2^120 stays a bf16 value
    z = y * ((127 - e) << 23).view(torch.float32)[..., None]
    codes = torch.minimum(torch.maximum(z, -limit), limit).to(KV8)
    return codes, torch.where(ok, e + 127, 255).to(torch.uint8)


def slots_into_layer(view: Tensor, slots_layout: Tensor) -> None:
    """Fill one layer's K (or V) view from a reference-layout ``[slots, kv_heads, 128]`` tensor."""
    nb, kvh = view.shape[0], view.shape[1]
    if is_kv8(view):
        codes, exps = _kv8_parts(view)
        rows = slots_layout.reshape(nb, BLOCK_SIZE, kvh, HEAD_DIM).permute(0, 2, 1, 3)
        c, b = quantise_rows(rows)
        c = c.view(torch.uint8).reshape(nb, kvh, BLOCK_SIZE, 8, 16)
        order = _kv8_order(view.device)[None, None, :, :, None].expand_as(c)
        codes.copy_(torch.gather(c, 3, order))  # the order is its own inverse
        exps.copy_(b)
        return
    src = slots_layout.reshape(nb, BLOCK_SIZE, kvh, 2, HEAD_DIM // 2).permute(0, 2, 3, 1, 4)
    view.copy_(src)
