"""Sparse attention for decode: every query token attends over a few pages that a cheap score selects.

No reference counterpart.  A page is the 16 tokens of one block, of one KV head.  Beside the pool lies
another paged tensor, the key bounds (``allocate_key_bounds``): for each page and channel the smallest and
the largest key value, a sixteenth of a bf16 pool's bytes.  Per layer and step:

    update_key_bounds(k_cache, v_cache, bounds, meta)    # after the step's rows are written
    pages = select_pages(q, bounds, meta, budget)
    out = attend_pages(q, k_cache, v_cache, meta, pages, scale)

``Qwen3Attention`` makes these calls where its ``sparse_budget`` and ``key_bounds`` are set.  Sequences of
at most ``SHORT_QUERY`` new tokens (decode and verify rows) are sparse; longer chunks and draft trees of
the same step are attended in full by ``attend_pages``.  Either kind of pool serves.
"""

from __future__ import annotations

import ctypes as C

import torch
from torch import Tensor

from . import _capi
from .attention import (AttentionMetadata, _check_slots, _on_own_device, _rows, _stream, attend)
from .kv_pool import HEAD_DIM, check_layer_views, is_kv8

MAX_BUDGET = 4096  # pages that a query token may keep
MAX_SELECT_PAGES = 49152  # pages that one may choose from (786432 tokens)


def allocate_key_bounds(num_layers: int, num_blocks: int, num_kv_heads: int,
                        device: torch.device | str) -> tuple[Tensor, list[Tensor]]:
    """Zero-filled key bounds ``[layers, num_blocks, kv_heads, 2 (lo, hi), 128]`` bf16 and each layer's
    view of them."""
    bounds = torch.zeros((num_layers, num_blocks, num_kv_heads, 2, HEAD_DIM), dtype=torch.bfloat16,
                         device=device)
    return bounds, list(bounds.unbind(0))


def _check_bounds(bounds: Tensor) -> tuple[int, int]:
    """(blocks, KV heads) of a layer's key bounds."""
    shape = bounds.shape
    if (len(shape) != 4 or shape[2] != 2 or shape[3] != HEAD_DIM or bounds.dtype is not torch.bfloat16
            or not bounds.is_contiguous()):
        raise ValueError(f"bounds must be a layer of allocate_key_bounds (bf16 [blocks, kv_heads, 2, "
                         f"{HEAD_DIM}]); got {bounds.dtype} {tuple(shape)}")
    nb, kvh, _, _ = shape
    return nb, kvh


def _check_pool(k_cache: Tensor, v_cache: Tensor, bounds: Tensor) -> tuple[int, int]:
    """The pool's views and its bounds; (blocks, KV heads)."""
    nb, kvh = check_layer_views(k_cache, v_cache, kv8=True)
    blocks, heads = _check_bounds(bounds)
    if blocks != nb or heads != kvh:
        raise ValueError(f"bounds of {blocks} blocks and {heads} KV heads, the pool has {nb} and {kvh}")
    return nb, kvh


def _other_device(index: int, **tensors: Tensor) -> ValueError:
    name, t = next((n, t) for n, t in tensors.items() if t.get_device() != index)
    return ValueError(f"{name} is on {t.device}, other arguments on cuda:{index}")


def update_key_bounds(k_cache: Tensor, v_cache: Tensor, bounds: Tensor, meta: AttentionMetadata) -> None:
    """The bounds of every page that the step's new tokens lie on, over the page's tokens up to the end of
    its sequence.  Call it for every layer and step once the step's rows are in the pool (prompt chunks
    included), so that later steps can select among the pages.

    A page keeps what it got until a step writes to it again; rows that are moved below a sequence's
    cached length (accepted drafts) want ``update_key_bounds_at`` for their blocks."""
    nb, kvh = _check_pool(k_cache, v_cache, bounds)
    dev, index = k_cache.device, k_cache.get_device()
    if bounds.get_device() != index or meta.plan.get_device() != index:
        raise _other_device(index, bounds=bounds, meta=meta.plan)
    lib = _capi.load()
    fn = lib.ms_key_bounds_step_kv8 if is_kv8(k_cache) else lib.ms_key_bounds_step
    for part in (meta, meta.tree):
        if part is not None and part.info.num_seqs > 0:
            rc = _on_own_device(fn, dev, k_cache.data_ptr(), nb, kvh, part.plan.data_ptr(),
                                C.byref(part.info), bounds.data_ptr(), _stream(dev))
            _capi.check(rc, "update_key_bounds")


def update_key_bounds_at(k_cache: Tensor, v_cache: Tensor, bounds: Tensor, blocks: Tensor,
                         rows: Tensor) -> None:
    """The bounds of the blocks ``blocks`` (int64 vector) over their first ``rows`` tokens each (int64
    vector).  Entries with a negative block or without rows are skipped.  The blocks of one call differ
    from each other."""
    nb, kvh = _check_pool(k_cache, v_cache, bounds)
    n = _check_slots(blocks)
    if _check_slots(rows) != n:
        raise ValueError(f"{n} blocks but {rows.shape[0]} row counts")
    dev, index = k_cache.device, k_cache.get_device()
    if not bounds.get_device() == blocks.get_device() == rows.get_device() == index:
        raise _other_device(index, bounds=bounds, blocks=blocks, rows=rows)
    lib = _capi.load()
    fn = lib.ms_key_bounds_kv8 if is_kv8(k_cache) else lib.ms_key_bounds
    rc = _on_own_device(fn, dev, k_cache.data_ptr(), nb, kvh, blocks.data_ptr(), rows.data_ptr(), n,
                        bounds.data_ptr(), _stream(dev))
    _capi.check(rc, "update_key_bounds_at")


def _check_rows_of_step(rows: int, meta: AttentionMetadata) -> None:
    if rows < meta.num_tokens and rows < (need := meta.rows_needed()):
        raise ValueError(f"q must have the step's {need} rows")


def _check_pages(pages: Tensor, rows: int, kvh: int, budget: int | None = None) -> int:
    shape = pages.shape
    if (len(shape) != 3 or shape[0] < rows or shape[1] != kvh or pages.dtype is not torch.int32
            or not pages.is_contiguous() or (budget is not None and shape[2] != budget)):
        want = "budget" if budget is None else budget
        raise ValueError(f"pages must be contiguous int32 [{rows}, {kvh}, {want}]; got {pages.dtype} "
                         f"{tuple(shape)}")
    return shape[2]


def select_pages(q: Tensor, bounds: Tensor, meta: AttentionMetadata, budget: int, first: int = 1,
                 last: int = 2, out: Tensor | None = None) -> Tensor:
    """The pages that each query token of the step's short rows keeps, ``[T, kv_heads, budget]`` int32:
    indices into its sequence's block table in ascending order, -1 behind.

    A token that sees at most ``budget`` pages keeps them all.  Else it keeps the ``first`` first and the
    ``last`` last ones (its own page is the last) and of those between the ones with the highest scores,
    max over the KV head's two query heads of sum_d max(q_d lo_d, q_d hi_d), compared as exactly as 64 bits
    give them; equal scores go to the lower page, and a score that is not finite counts as infinite, as does
    that of any page with a bound that is not finite.
    Rows of longer chunks and of trees are left untouched (undefined).  Calls that use one metadata share its
    scratch, so they are ordered on the GPU (one stream, or events).  The scratch is the product of the step's
    sequences, the most new tokens of a short row (up to 8), the KV heads and the most pages that a short row
    sees, 4.25 bytes each: one very long row makes it large for every row of its step."""
    nb, kvh = _check_bounds(bounds)
    q_stride, (t, heads, _) = _rows(q, "q"), q.shape
    if heads != 2 * kvh:
        raise ValueError(f"q must have {2 * kvh} heads for bounds of {kvh} KV heads, not {heads}")
    if not 1 <= budget <= MAX_BUDGET or first < 0 or last < 1 or first + last > budget:
        raise ValueError(f"need 1 <= budget <= {MAX_BUDGET}, first >= 0, last >= 1 and first + last <= "
                         f"budget; got {budget}, {first} and {last}")
    dev, index, plan = bounds.device, bounds.get_device(), meta.plan
    if q.get_device() != index or plan.get_device() != index:
        raise _other_device(index, q=q, meta=plan)
    _check_rows_of_step(t, meta)
    if out is None:
        out = torch.empty(t, kvh, budget, dtype=torch.int32, device=dev)
    else:
        _check_pages(out, t, kvh, budget)
        if out.get_device() != index:
            raise _other_device(index, out=out)
    most_new, most_pages = meta.short_rows()
    if most_new:
        if most_pages > MAX_SELECT_PAGES:
            raise ValueError(f"a row sees up to {most_pages} pages; at most {MAX_SELECT_PAGES} can be "
                             "chosen from")
        ws = meta.select_workspace(kvh, dev)
        rc = _on_own_device(
            _capi.load().ms_select_pages, dev, q.data_ptr(), q_stride, heads, kvh,
            bounds.data_ptr(), nb, plan.data_ptr(), C.byref(meta.info), most_new, most_pages,
            budget, first, last, out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(dev))
        _capi.check(rc, "select_pages")
    return out


def attend_pages(q: Tensor, k_cache: Tensor, v_cache: Tensor, meta: AttentionMetadata, pages: Tensor,
                 scale: float, out: Tensor | None = None) -> Tensor:
    """``attend`` where the query tokens of short rows see only the keys of their ``pages`` (``[T,
    kv_heads, budget]`` int32, as ``select_pages`` gives them or of the caller's own choice).

    Entries that the token does not see (negative, or behind its own page) are skipped in any place; a page
    named twice counts twice; a row without pages gives zeros.  Longer chunks and trees see all that they
    see in ``attend``.  Rows not covered by ``meta`` are left untouched.

    Over an 8-bit pool a key adds nothing where its weight times its value row's size is below 2^-36 of the
    largest such product of the query token, and a query's channels below 2^-27 of its largest one lose bits."""
    nb, kvh = check_layer_views(k_cache, v_cache, kv8=True)
    dev, index, plan = k_cache.device, k_cache.get_device(), meta.plan
    q_stride, shape = _rows(q, "q"), q.shape
    if not q.get_device() == plan.get_device() == pages.get_device() == index:
        raise _other_device(index, q=q, meta=plan, pages=pages)
    _check_rows_of_step(shape[0], meta)
    budget = _check_pages(pages, shape[0], kvh)
    if not 1 <= budget <= MAX_BUDGET:
        raise ValueError(f"pages must have 1 to {MAX_BUDGET} entries per row, not {budget}")
    if out is None:
        out = torch.empty_like(q)
        out_stride = out.stride(0)
    else:
        if out.shape[1:] != shape[1:] or out.shape[0] < shape[0]:
            raise ValueError("out must have q's shape")
        out_stride = _rows(out, "out")
        if out.get_device() != index:
            raise _other_device(index, out=out)
    scale = float(scale)
    rest = meta.rest()
    most_new, _ = meta.short_rows()
    if most_new:
        lib = _capi.load()
        rows = (q.data_ptr(), q_stride, out.data_ptr(), out_stride, shape[1], kvh)
        step = (nb, plan.data_ptr(), C.byref(meta.info), most_new, pages.data_ptr(), budget, scale,
                _stream(dev))
        if is_kv8(k_cache):
            rc = _on_own_device(lib.ms_attend_pages_kv8, dev, *rows, k_cache.data_ptr(), *step)
        else:
            rc = _on_own_device(lib.ms_attend_pages, dev, *rows, k_cache.data_ptr(), v_cache.data_ptr(),
                                *step)
        _capi.check(rc, "attend_pages")
    if rest is not None:
        attend(q, k_cache, v_cache, rest, scale, out)
    return out


