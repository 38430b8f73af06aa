"""Drop-in replacement for MiniServe's attention backend (src/miniserve/attention/backends.py).

Same names and call shapes as the reference module:

* ``SeqChunk(flat_start, num_new, num_cached, block_table)``            (backends.py:36-47)
* ``build_attention_metadata(chunks, slot_mapping, block_size)``       (backends.py:80-98)
* ``paged_attention(q, k, v, k_cache, v_cache, meta, scale) -> [T, H, D]`` (backends.py:145-197)
* ``SHORT_QUERY`` and ``MAX_GATHER_TOKENS`` (backends.py:32-33; the runner's profiler imports the
  latter, model_runner.py:21,111).

What changes underneath: the metadata is one packed int32 plan built by the native planner and
uploaded with a single pinned, non-blocking copy; the KV pool uses the layout of
``miniserve_b200.kv_pool``; the scatter and the attention are hand-written sm_100a kernels that
read the pool in place (no gather copy, no padding, no masks in memory).  Everything runs on the
caller's current CUDA stream and never synchronises; errors surface as ``ValueError`` /
``RuntimeError`` like the reference's.

Beyond the reference: the pool may be the 8-bit one (``allocate_kv_cache(...,
dtype=torch.float8_e4m3fn)``), which ``kv_scatter``, ``attend`` and ``paged_attention`` take like the
bf16 one; ``kv_gather`` reads rows of either back; and a chunk's new tokens may be a tree of drafted
tokens (``SeqChunk.parents``).
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field
from itertools import chain

import numpy as np
import torch
from torch import Tensor

from . import _capi
from .kv_pool import BLOCK_SIZE, HEAD_DIM, check_layer_views, is_kv8, kv8_in_use

SHORT_QUERY = 8  # rows with at most this many new tokens take the decode kernel
MAX_GATHER_TOKENS = 16384  # kept for the runner's profiler; nothing is gathered here


@dataclass
class SeqChunk:
    """What attention needs to know about one scheduled sequence (backends.py:36-47)."""

    flat_start: int  # where its new tokens start in the flattened batch
    num_new: int  # new tokens this step (its queries)
    num_cached: int  # tokens already in the KV cache before this step
    block_table: list[int]
    # A tree of drafts instead of a causal chunk: draft k's parent among the new tokens (an earlier
    # one), -1 for a child of the last cached token, UNUSED_DRAFT for a position without a draft.
    # Draft k's K/V lie at position num_cached + k; it sees the cached tokens, its ancestors and
    # itself.  An unused position sees nothing, is seen by none, and its output row is zero.
    parents: list[int] | None = None

    @property
    def context_len(self) -> int:
        return self.num_cached + self.num_new


UNUSED_DRAFT = -2


def tree_positions(num_cached: int, parents: list[int]) -> list[int]:
    """RoPE position of each draft of a tree: ``num_cached`` plus its depth (unused positions get
    ``num_cached``)."""
    depth: list[int] = []
    for k, p in enumerate(parents):
        if not UNUSED_DRAFT <= p < k or (p >= 0 and parents[p] == UNUSED_DRAFT):
            raise ValueError(f"draft {k} has parent {p} (want an earlier draft in use, -1 for the last "
                             f"cached token, or {UNUSED_DRAFT} for an unused position)")
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return [num_cached + d for d in depth]


@dataclass
class AttentionMetadata:
    """The per-step plan, built once and shared by every layer (backends.py:67-71)."""

    slot_mapping: Tensor  # [T] int64 slot of each new token, on the device
    plan: Tensor  # packed int32 plan on the device
    info: _capi.MsPlanInfo  # host-side description of the plan
    num_tokens: int
    _workspace: dict[tuple, Tensor] = field(default_factory=dict, repr=False)
    _num_sms: int = field(default=148, repr=False)
    _pages_per_split: int = field(default=0, repr=False)
    # The plan's part for 8-bit pools: its description, and the device plan with it behind (None: not
    # built for the present step).  Once a call has used it, a captured graph may hold it.
    kv8: _capi.MsKv8Info | None = field(default=None, repr=False)
    _plan8: Tensor | None = field(default=None, repr=False)
    _kv8_used: bool = field(default=False, repr=False)
    _packed: np.ndarray | None = field(default=None, repr=False)  # the plan on the host, without it
    # The sequences whose new tokens are trees of drafts, planned apart (None: there are none).
    tree: AttentionMetadata | None = field(default=None, repr=False)
    # Calls over selected pages: what their launches take from the step (see short_rows), and the sequences
    # that they attend in full, planned apart; None until a call has asked.
    _short: tuple[int, int] | None = field(default=None, repr=False)
    _rest: AttentionMetadata | None = field(default=None, repr=False)
    _no_rest: bool = field(default=False, repr=False)

    def update(self, chunks: list[SeqChunk], slot_mapping: Tensor | None = None) -> bool:
        """Plan a new step into this metadata's device buffers, for CUDA-graph replay.

        A graph captured over calls that use this metadata keeps the addresses of its plan and
        slot mapping and the launch shapes derived from ``info`` (grid sizes, section offsets,
        workspace size).  When the new step's plan has the same shape (same item counts, offsets
        and split workspace: for example, the same batch again, or contexts that grew inside their
        last pages), its plan and, if given, its slot mapping are copied into the existing buffers
        on the current stream (after the work already queued there, so no kernel of the previous
        step sees them) and True is returned.  Otherwise nothing changes and False is returned:
        build new metadata and capture again.  What a launch over an 8-bit pool adds to the shape
        (the pages that its tensor-core items read) counts once this metadata has been used for one.
        A launch over selected pages takes the most new tokens of the step's short rows and a bound of the
        pages that they see (``short_rows``): once this metadata has been used for one, the first has to be
        the same and the second is not to grow past the bound.
        No reference counterpart (MiniServe captures no graphs).
        """
        if slot_mapping is not None and tuple(slot_mapping.shape) != tuple(self.slot_mapping.shape):
            return False
        plain, trees = _split_trees(chunks)
        if bool(trees) != (self.tree is not None):
            return False
        new = [(self, self._replan(plain))]
        if self.tree is not None:
            new.append((self.tree, self.tree._replan(trees)))
        if self._rest is not None:
            new.append((self._rest, self._rest._replan([c for c in plain if c.num_new > SHORT_QUERY])))
        if any(plan is None for _, plan in new):
            return False
        if self._short is not None:
            most_new, most_pages = _short_rows(*new[0][1][:2])
            if most_new != self._short[0] or most_pages > self._short[1]:
                return False
        if self._no_rest and any(c.num_new > SHORT_QUERY for c in plain):
            return False
        for meta, plan in new:
            meta._write(*plan)
        if slot_mapping is not None and slot_mapping.data_ptr() != self.slot_mapping.data_ptr():
            self.slot_mapping.copy_(slot_mapping, non_blocking=True)
        return True

    def _replan(self, chunks: list[SeqChunk]
                ) -> tuple[np.ndarray, _capi.MsPlanInfo, _capi.MsKv8Info | None] | None:
        """The plan of a new step, or None if it launches differently.  A part for 8-bit pools that
        launches differently is left out where no call has used it: the next one builds it anew."""
        kv8 = None if self.kv8 is None else _capi.MsKv8Info()
        if self.info.is_tree:
            packed, info, kv8 = _plan_trees(chunks, self.num_tokens, self._num_sms,
                                            self._pages_per_split, kv8)
        else:
            packed, info, kv8 = _plan(chunks, self.num_tokens, BLOCK_SIZE, self._num_sms,
                                      self._pages_per_split, kv8)
        if not same_launch_shape(info, self.info):
            return None
        if kv8 is not None and (bytes(kv8) != bytes(self.kv8)
                                or info.n_tc_combine != self.info.n_tc_combine):
            if self._kv8_used:
                return None
            packed, kv8 = packed[: info.total_ints], None
        return packed, info, kv8

    def _write(self, packed: np.ndarray, info: _capi.MsPlanInfo, kv8: _capi.MsKv8Info | None) -> None:
        """A plan of the same launch shape into this metadata's buffers."""
        base = int(info.total_ints)
        host = torch.from_numpy(packed).pin_memory()
        if kv8 is not None:
            self._plan8.copy_(host, non_blocking=True)
        if self._plan8 is not self.plan or kv8 is None:
            self.plan[:base].copy_(host[:base], non_blocking=True)
        if kv8 is None:
            self._plan8 = None
        self.info, self.kv8, self._packed = info, kv8, packed[:base]

    def for_kv8(self) -> tuple[Tensor, _capi.MsKv8Info]:
        """The device plan with its part for 8-bit pools, and that part's description."""
        if self.kv8 is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the step has no plan for 8-bit pools (it was planned before the "
                                   "process had one, or updated since): call it once before it is "
                                   "captured")
            packed, self.kv8 = _add_kv8(self._packed, self.info, self._num_sms,
                                        self._pages_per_split)
            self._plan8 = _upload_plan(packed, self.plan.device)
        self._kv8_used = True
        return self._plan8, self.kv8

    def short_rows(self) -> tuple[int, int]:
        """Most new tokens of the sequences of at most SHORT_QUERY of them (0: there are none), and a bound of
        the pages that one of them sees (the most of them in steps of 64, of the step that first asked): what
        a launch over their selected pages depends on."""
        if self._short is None:
            self._short = _short_rows(self._packed, self.info)
        return self._short

    def select_workspace(self, num_kv_heads: int, device: torch.device) -> Tensor:
        """Scratch of ``select_pages`` for this step: the scores of the short rows' pages."""
        key = (device, num_kv_heads, "select")
        ws = self._workspace.get(key)
        if ws is None:
            most_new, most_pages = self.short_rows()
            need = int(_capi.load().ms_select_workspace_bytes(
                self.info.num_seqs, most_new, most_pages, num_kv_heads))
            ws = self._workspace[key] = torch.empty(need, dtype=torch.uint8, device=device)
        return ws

    def rest(self) -> AttentionMetadata | None:
        """The step without the sequences of at most SHORT_QUERY new tokens (None: nothing is left, which a
        step of the same launch shape shares)."""
        if self._rest is None and not self._no_rest:
            long = _long_chunks(self._packed, self.info)
            self._no_rest = not long and self.tree is None
            if self._no_rest:
                return None
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the step's longer chunks have no plan of their own yet: call "
                                   "attend_pages once before it is captured")
            packed, info, _ = _plan(long, self.num_tokens, BLOCK_SIZE, self._num_sms,
                                    self._pages_per_split, None)
            self._rest = AttentionMetadata(
                self.slot_mapping, _upload_plan(packed, self.plan.device), info, self.num_tokens,
                _num_sms=self._num_sms, _pages_per_split=self._pages_per_split, _packed=packed,
                tree=self.tree)
        return self._rest

    def rows_needed(self) -> int:
        """Rows of q and out that the planned sequences reach (``num_tokens`` counts the slots)."""
        seqs = _seq_records(self._packed, self.info)
        last = int((seqs[:, 0] + seqs[:, 1]).max()) if seqs.shape[0] else 0
        return last if self.tree is None else max(last, self.tree.rows_needed())

    def workspace(self, num_kv_heads: int, device: torch.device, kv8: bool = False,
                  counters: bool = False) -> Tensor | None:
        """Scratch for this step (allocated once, reused by every layer): split-KV partials, with
        ``counters`` the arrival counters of split tiles behind them (zeroed here, left at zero by
        every call), and for an 8-bit pool the expanded pages of tensor-core items.  Allocated while
        the stream is captured, a workspace with counters is that call's own: its zeroing is a node
        of the graph, which runs only when that graph does."""
        key = (device, -num_kv_heads if kv8 else num_kv_heads)  # a tensor's device has its index
        ws = self._workspace.get(key)
        if ws is not None:
            return ws
        if kv8:
            need = int(_capi.load().ms_kv8_workspace_bytes(
                C.byref(self.info), C.byref(self.for_kv8()[1]), num_kv_heads))
        else:
            need = int(self.info.workspace_bytes_per_kv_head) * num_kv_heads
        if need == 0:
            return None
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        if counters:
            rows = int(self.info.part_rows) + (int(self.kv8.part_rows) if kv8 else 0)
            n = int(self.kv8.n_combine if kv8 else self.info.n_combine)
            at = rows * (HEAD_DIM + 1) * 4 * num_kv_heads
            if n:
                ws[at : at + n * 4 * num_kv_heads].zero_()
                if torch.cuda.is_current_stream_capturing():
                    return ws
        self._workspace[key] = ws
        return ws


def _seq_records(packed: np.ndarray, info: _capi.MsPlanInfo) -> np.ndarray:
    """``[num_seqs, 8]``: first row, new tokens, cached tokens, context, table's offset and length."""
    n = int(info.num_seqs)
    return packed[info.off_seqs :][: 8 * n].reshape(n, 8)


def _short_rows(packed: np.ndarray, info: _capi.MsPlanInfo) -> tuple[int, int]:
    seqs = _seq_records(packed, info)
    short = seqs[(seqs[:, 1] > 0) & (seqs[:, 1] <= SHORT_QUERY)]
    if not short.shape[0]:
        return 0, 0
    pages = -(-int(short[:, 3].max()) // BLOCK_SIZE)
    return int(short[:, 1].max()), -(-pages // 64) * 64


def _long_chunks(packed: np.ndarray, info: _capi.MsPlanInfo) -> list[SeqChunk]:
    """The chunks of more than SHORT_QUERY new tokens that a plan holds."""
    seqs = _seq_records(packed, info)
    tables = packed[info.off_tables :]
    return [SeqChunk(int(r[0]), int(r[1]), int(r[2]), tables[r[4] : r[4] + r[5]].tolist())
            for r in seqs[seqs[:, 1] > SHORT_QUERY]]


_SM_COUNT: dict[int, int] = {}


def _num_sms(device: torch.device) -> int:
    if device.type != "cuda":
        raise RuntimeError("miniserve_b200 attention runs on CUDA only (no CPU fallback)")
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _SM_COUNT:
        _SM_COUNT[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return _SM_COUNT[idx]


def plan_batch(
    chunks: list[SeqChunk],
    num_tokens: int,
    block_size: int = BLOCK_SIZE,
    num_sms: int = 148,
    pages_per_split: int = 0,
) -> tuple[np.ndarray, _capi.MsPlanInfo]:
    """Run the native planner on the host; returns ``(packed int32 plan, info)``."""
    packed, info, _ = _plan(chunks, num_tokens, block_size, num_sms, pages_per_split, None)
    return packed, info


def _plan_with_kv8(chunks: list[SeqChunk], num_tokens: int, num_sms: int, pages_per_split: int
                   ) -> tuple[np.ndarray, _capi.MsPlanInfo, _capi.MsKv8Info]:
    """The plan with the part an 8-bit pool needs behind it, so that one plan (and one upload)
    serves either kind of pool."""
    kv8 = _capi.MsKv8Info()
    return _plan(chunks, num_tokens, BLOCK_SIZE, num_sms, pages_per_split, kv8)


def _plan(chunks: list[SeqChunk], num_tokens: int, block_size: int, num_sms: int,
          pages_per_split: int, kv8: _capi.MsKv8Info | None):
    lib = _capi.load()
    n = len(chunks)
    flat = np.fromiter((c.flat_start for c in chunks), dtype=np.int32, count=n)
    new = np.fromiter((c.num_new for c in chunks), dtype=np.int32, count=n)
    cached = np.fromiter((c.num_cached for c in chunks), dtype=np.int32, count=n)
    lens = np.fromiter((len(c.block_table) for c in chunks), dtype=np.int64, count=n)
    offsets = np.zeros(n + 1, dtype=np.int64)
    np.cumsum(lens, out=offsets[1:])
    total = int(offsets[-1])
    tables = np.fromiter(chain.from_iterable(c.block_table for c in chunks), dtype=np.int32,
                         count=total)
    cap = int(lib.ms_plan_capacity(n, num_tokens, total))
    out = np.empty(cap + (int(lib.ms_kv8_plan_capacity(n, total)) if kv8 is not None else 0),
                   dtype=np.int32)
    info = _capi.MsPlanInfo()
    rc = lib.ms_plan_build(
        n, flat.ctypes.data, new.ctypes.data, cached.ctypes.data, offsets.ctypes.data,
        tables.ctypes.data if total else None, num_tokens, block_size, num_sms, pages_per_split,
        out.ctypes.data, cap, C.byref(info),
    )
    _capi.check(rc, "build_attention_metadata")
    if kv8 is None:
        return out[: info.total_ints], info, None
    rc = lib.ms_kv8_plan_build(out.ctypes.data, out.size, C.byref(info), num_sms, pages_per_split,
                               C.byref(kv8))
    _capi.check(rc, "build_attention_metadata")
    return out[: kv8.total_ints], info, kv8


def _add_kv8(packed: np.ndarray, info: _capi.MsPlanInfo, num_sms: int, pages_per_split: int
             ) -> tuple[np.ndarray, _capi.MsKv8Info]:
    """A packed plan with the part for 8-bit pools behind it."""
    lib = _capi.load()
    n = int(info.num_seqs)
    seqs = packed[info.off_seqs :][: 8 * n].reshape(n, 8)  # fields 1 and 5: new tokens, table length
    new = np.ascontiguousarray(seqs[:, 1])
    entries = int(seqs[:, 5].sum(dtype=np.int64))
    more = (lib.ms_tree_plan_capacity(n, new.ctypes.data, entries) if info.is_tree
            else lib.ms_kv8_plan_capacity(n, entries))
    out = np.empty(packed.size + int(more), dtype=np.int32)
    out[: packed.size] = packed
    kv8 = _capi.MsKv8Info()
    rc = lib.ms_kv8_plan_build(out.ctypes.data, out.size, C.byref(info), num_sms, pages_per_split,
                               C.byref(kv8))
    _capi.check(rc, "build_attention_metadata")
    return out[: kv8.total_ints], kv8


def plan_tree_batch(
    chunks: list[SeqChunk],
    num_tokens: int,
    block_size: int = BLOCK_SIZE,
    num_sms: int = 148,
    pages_per_split: int = 0,
) -> tuple[np.ndarray, _capi.MsPlanInfo]:
    """Run the native planner of draft trees on the host (every chunk has ``parents``); returns
    ``(packed int32 plan, info)``."""
    if block_size != BLOCK_SIZE:
        raise ValueError(f"block_size must be {BLOCK_SIZE}")
    packed, info, _ = _plan_trees(chunks, num_tokens, num_sms, pages_per_split, None)
    return packed, info


def _plan_trees(chunks: list[SeqChunk], num_tokens: int, num_sms: int, pages_per_split: int,
                kv8: _capi.MsKv8Info | None):
    lib = _capi.load()
    n = len(chunks)
    for i, c in enumerate(chunks):
        if c.parents is None or len(c.parents) != c.num_new:
            raise ValueError(f"tree sequence {i}: parents must name one parent per new token "
                             f"({c.num_new})")
    flat = np.fromiter((c.flat_start for c in chunks), dtype=np.int32, count=n)
    new = np.fromiter((c.num_new for c in chunks), dtype=np.int32, count=n)
    cached = np.fromiter((c.num_cached for c in chunks), dtype=np.int32, count=n)
    lens = np.fromiter((len(c.block_table) for c in chunks), dtype=np.int64, count=n)
    offsets = np.zeros(n + 1, dtype=np.int64)
    np.cumsum(lens, out=offsets[1:])
    total = int(offsets[-1])
    tables = np.fromiter(chain.from_iterable(c.block_table for c in chunks), dtype=np.int32,
                         count=total)
    parents = np.fromiter(chain.from_iterable(c.parents or [] for c in chunks), dtype=np.int32)
    cap = int(lib.ms_tree_plan_capacity(n, new.ctypes.data, total))
    out = np.empty(cap, dtype=np.int32)
    info = _capi.MsPlanInfo()
    rc = lib.ms_tree_plan_build(
        n, flat.ctypes.data, new.ctypes.data, cached.ctypes.data, offsets.ctypes.data,
        tables.ctypes.data if total else None, parents.ctypes.data, num_tokens, BLOCK_SIZE,
        num_sms, pages_per_split, out.ctypes.data, cap, C.byref(info),
    )
    _capi.check(rc, "build_attention_metadata")
    if kv8 is None:
        return out[: info.total_ints], info, None
    rc = lib.ms_kv8_plan_build(out.ctypes.data, cap, C.byref(info), num_sms, pages_per_split,
                               C.byref(kv8))
    _capi.check(rc, "build_attention_metadata")
    return out[: kv8.total_ints], info, kv8


def _split_trees(chunks: list[SeqChunk]) -> tuple[list[SeqChunk], list[SeqChunk]]:
    trees = [c for c in chunks if c.parents is not None]
    return ([c for c in chunks if c.parents is None], trees) if trees else (chunks, trees)


def prepare_arrays(num_new: np.ndarray, num_cached: np.ndarray, table_offsets: np.ndarray,
                   tables: np.ndarray, positions_out: np.ndarray, slots_out: np.ndarray
                   ) -> tuple[np.ndarray, int]:
    """``ms_prepare_step`` over CSR arrays (int32 num_new / num_cached / tables, int64
    table_offsets of length n + 1) into caller buffers (contiguous int64, e.g. pinned host
    memory).  Returns ``(flat_start int32, num_tokens)``."""
    lib = _capi.load()
    n = int(num_new.shape[0])
    for arr, dt, name in ((num_new, np.int32, "num_new"), (num_cached, np.int32, "num_cached"),
                          (table_offsets, np.int64, "table_offsets"), (tables, np.int32, "tables"),
                          (positions_out, np.int64, "positions_out"),
                          (slots_out, np.int64, "slots_out")):
        if arr.dtype != dt or not arr.flags.c_contiguous:
            raise ValueError(f"{name} must be a contiguous {np.dtype(dt).name} array")
    if num_cached.shape[0] != n or table_offsets.shape[0] != n + 1:
        raise ValueError("num_cached / table_offsets do not match num_new")
    tokens = int(num_new.sum(dtype=np.int64))
    if positions_out.shape[0] < tokens or slots_out.shape[0] < tokens:
        raise ValueError(f"positions_out / slots_out must be contiguous int64 arrays of >= {tokens} "
                         "elements")
    flat = np.empty(n, dtype=np.int32)
    got = C.c_int32(0)
    rc = lib.ms_prepare_step(
        n, num_new.ctypes.data, num_cached.ctypes.data, table_offsets.ctypes.data,
        tables.ctypes.data if tables.size else None, BLOCK_SIZE, flat.ctypes.data,
        positions_out.ctypes.data, slots_out.ctypes.data,
        min(positions_out.shape[0], slots_out.shape[0]), C.byref(got))
    _capi.check(rc, "prepare_step")
    return flat, got.value


def prepare_step(
    scheduled: list[tuple[int, int, list[int]]],
    *,
    positions_out: np.ndarray | None = None,
    slots_out: np.ndarray | None = None,
) -> tuple[list[SeqChunk], np.ndarray, np.ndarray]:
    """The attention inputs of ``ModelRunner.prepare`` (model_runner.py:162-205) in one native
    pass (``ms_prepare_step``).  ``scheduled`` holds ``(num_new, num_cached, block_table)`` per
    sequence in batch order; returns ``(chunks, positions, slot_mapping)`` with int64 positions
    and slots (``table[p // 16] * 16 + p % 16``) in flat-batch order.  Optional ``*_out`` arrays
    (int64, e.g. views of pinned host tensors) receive the results without new allocations."""
    n = len(scheduled)
    new = np.fromiter((s[0] for s in scheduled), dtype=np.int32, count=n)
    cached = np.fromiter((s[1] for s in scheduled), dtype=np.int32, count=n)
    lens = np.fromiter((len(s[2]) for s in scheduled), dtype=np.int64, count=n)
    offsets = np.zeros(n + 1, dtype=np.int64)
    np.cumsum(lens, out=offsets[1:])
    total = int(offsets[-1])
    tables = np.fromiter(chain.from_iterable(s[2] for s in scheduled), dtype=np.int32, count=total)
    tokens = int(new.sum(dtype=np.int64))
    positions = positions_out if positions_out is not None else np.empty(tokens, dtype=np.int64)
    slots = slots_out if slots_out is not None else np.empty(tokens, dtype=np.int64)
    flat, got = prepare_arrays(new, cached, offsets, tables, positions, slots)
    chunks = [SeqChunk(int(flat[i]), int(new[i]), int(cached[i]), list(scheduled[i][2]))
              for i in range(n)]
    return chunks, positions[:got], slots[:got]


def build_attention_metadata(
    chunks: list[SeqChunk],
    slot_mapping: Tensor,
    block_size: int,
    *,
    pages_per_split: int = 0,
) -> AttentionMetadata:
    """Plan one step and upload it (one pinned H2D copy, no sync).  backends.py:80-98.

    The plan serves bf16 pools, and 8-bit ones once the process has allocated one; a step planned before
    that gets their part with its first call over one."""
    device = slot_mapping.device
    num_sms = _num_sms(device)  # raises for a non-CUDA device: there is no CPU path
    if block_size != BLOCK_SIZE:
        raise ValueError(f"block_size must be {BLOCK_SIZE}")
    num_tokens = int(slot_mapping.shape[0])
    plain, trees = _split_trees(chunks)
    slots = slot_mapping if slot_mapping.dtype == torch.int64 else slot_mapping.to(torch.int64)
    slots = slots.contiguous()

    def part() -> _capi.MsKv8Info | None:
        return _capi.MsKv8Info() if kv8_in_use() else None

    def metadata(packed: np.ndarray, info: _capi.MsPlanInfo, kv8: _capi.MsKv8Info | None
                 ) -> AttentionMetadata:
        plan = _upload_plan(packed, device)
        return AttentionMetadata(slots, plan, info, num_tokens, _num_sms=num_sms,
                                 _pages_per_split=pages_per_split, kv8=kv8,
                                 _plan8=None if kv8 is None else plan,
                                 _packed=packed[: info.total_ints])

    meta = metadata(*_plan(plain, num_tokens, BLOCK_SIZE, num_sms, pages_per_split, part()))
    if trees:
        meta.tree = metadata(*_plan_trees(trees, num_tokens, num_sms, pages_per_split, part()))
    return meta


def same_launch_shape(a: _capi.MsPlanInfo, b: _capi.MsPlanInfo) -> bool:
    """Whether two plans launch the same kernels with the same arguments apart from the plan's
    contents: every field of the plan description is equal except the total page count (a
    statistic no launch reads) and the count of tensor-core combine records, which only a launch
    over an 8-bit pool reads (``AttentionMetadata.update`` compares it for those)."""
    return all(getattr(a, name) == getattr(b, name)
               for name, _ in _capi.MsPlanInfo._fields_
               if name not in ("total_pages", "n_tc_combine", "reserved"))


def _upload_plan(packed: np.ndarray, device: torch.device) -> Tensor:
    """The step's one host-to-device copy: the packed plan, through pinned memory, non-blocking
    (the reference's ``to_device``, utils.py:11-20)."""
    return torch.from_numpy(packed).pin_memory().to(device, non_blocking=True)


def _stream(device: torch.device) -> int:
    """The current stream of a tensor's device, as the library takes it (torch's own accessor of the
    raw handle: a Stream object per call costs two microseconds)."""
    index = device.index  # a CUDA tensor's device always has one
    if index is None:
        raise RuntimeError("miniserve_b200 attention runs on CUDA only (no CPU fallback)")
    return torch._C._cuda_getCurrentRawStream(index)


def _rows(t: Tensor, name: str) -> int:
    """Row stride (elements) of a [T, heads, 128] tensor whose heads are packed in each row."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != HEAD_DIM or stride[2] != 1 or stride[1] != HEAD_DIM:
        raise ValueError(f"{name} must be [T, heads, {HEAD_DIM}] with contiguous heads")
    if t.dtype is not torch.bfloat16:
        raise ValueError(f"{name} must be bf16")
    return stride[0]


def kv_scatter(k: Tensor, v: Tensor, slot_mapping: Tensor, k_cache: Tensor, v_cache: Tensor,
               moved: bool = False) -> None:
    """Write this step's K/V rows into their slots (backends.py:159-160).  Into an 8-bit pool each
    row is quantised as it is written (see ``kv_pool``).  ``moved``: the rows are not the step's own but lie
    below the cached length of sequences that the next call may attend over.

    The slots of one call differ from each other, as for ``index_copy_``: what a slot named twice
    holds afterwards is undefined (an 8-bit one may pair one row's codes with the other's exponent).
    ``attend`` over a bf16 pool may read rows below a sequence's ``num_cached`` while the call before it
    on the stream still runs: it waits for rows that are written with ``moved`` (a launch more), and a step
    that writes its own rows in between needs no flag."""
    nb, kvh = check_layer_views(k_cache, v_cache, kv8=True)
    kv8 = is_kv8(k_cache)
    dev = _check_rows_args(k, v, slot_mapping, k_cache, kvh, spare_slots=not kv8)
    t = k.shape[0]
    rows = (k.data_ptr(), _rows(k, "k"), v.data_ptr(), _rows(v, "v"), t, kvh,
            slot_mapping.data_ptr(), k_cache.data_ptr())
    lib = _capi.load()
    if kv8:
        rc = _on_own_device(lib.ms_kv_scatter_kv8, dev, *rows, nb, _stream(dev))
    else:
        stream = _stream(dev)
        rc = _on_own_device(lib.ms_kv_scatter, dev, *rows, v_cache.data_ptr(), nb, stream)
        if moved and rc == _capi.MS_OK:
            rc = _on_own_device(lib.ms_kv_moved, dev, stream)
    _capi.check(rc, "kv_scatter")


def _on_own_device(fn, device: torch.device, *args) -> int:
    """Call the library, which launches on the current device, with the tensors' own device current."""
    index = device.index
    if index is None or torch._C._cuda_getDevice() == index:
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


def _check_rows_args(k: Tensor, v: Tensor, slots: Tensor, k_cache: Tensor, kvh: int,
                     spare_slots: bool = False) -> torch.device:
    """Rows and their slots fit each other and the pool (with ``spare_slots`` slots behind the last row
    are ignored); returns the pool's device."""
    shape = k.shape
    if len(shape) != 3 or shape != v.shape or shape[1] != kvh:
        raise ValueError(f"k and v must both be [T, {kvh}, {HEAD_DIM}]")
    n = _check_slots(slots)
    if n != shape[0] and (n < shape[0] or not spare_slots):
        raise ValueError(f"{shape[0]} rows but {n} slots")
    dev = k_cache.device
    index = k_cache.get_device()
    if not (k.get_device() == index and v.get_device() == index and slots.get_device() == index):
        raise ValueError(f"k, v and slots are on {k.device}, {v.device} and {slots.device}, "
                         f"the pool on {dev}")
    return dev


def _check_slots(slots: Tensor) -> int:
    """The length of a vector of slots."""
    shape = slots.shape
    if slots.dtype != torch.int64 or len(shape) != 1 or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int64 vector")
    return shape[0]


def kv_gather(slots: Tensor, k_cache: Tensor, v_cache: Tensor, k_out: Tensor | None = None,
              v_out: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Rows ``slots`` (int64 vector, any order, repeats allowed) of a layer's pool as bf16
    ``(k, v)``, each ``[len(slots), kv_heads, 128]``.  No reference counterpart.

    What it is for: after a verify step the accepted drafts' rows are read and written to the
    positions they take in the sequence (``kv_scatter(*kv_gather(from_slots, ...), to_slots, ...,
    moved=True)``; the rows are read before any is written, so the two sets may overlap), or a
    sequence's rows are handed to another cache.  From an 8-bit pool the values are exact, and writing
    them back stores the same values again.  A slot outside the pool reads as zeros (and sets the device
    status bit).
    """
    nb, kvh = check_layer_views(k_cache, v_cache, kv8=True)
    n = _check_slots(slots)
    ours = k_out is None and v_out is None
    if k_out is None:
        k_out = k_cache.new_empty((n, kvh, HEAD_DIM), dtype=torch.bfloat16)
    if v_out is None:
        v_out = torch.empty_like(k_out)
    if ours and k_cache.is_cuda and slots.device == k_cache.device:  # rows that need no checking
        dev = k_cache.device
        k_stride = v_stride = kvh * HEAD_DIM
    else:
        dev = _check_rows_args(k_out, v_out, slots, k_cache, kvh)
        k_stride, v_stride = _rows(k_out, "k_out"), _rows(v_out, "v_out")
    outs = (k_out.data_ptr(), k_stride, v_out.data_ptr(), v_stride, _stream(dev))
    lib = _capi.load()
    if is_kv8(k_cache):
        rc = _on_own_device(lib.ms_kv_gather_kv8, dev, slots.data_ptr(), n, kvh, k_cache.data_ptr(),
                            nb, *outs)
    else:
        rc = _on_own_device(lib.ms_kv_gather, dev, slots.data_ptr(), n, kvh, k_cache.data_ptr(),
                            v_cache.data_ptr(), nb, *outs)
    _capi.check(rc, "kv_gather")
    return k_out, v_out


def attend(q: Tensor, k_cache: Tensor, v_cache: Tensor, meta: AttentionMetadata, scale: float,
           out: Tensor | None = None) -> Tensor:
    """Attention of every planned query row through the pool (backends.py:161-197); draft trees
    and an 8-bit pool included.

    Rows not covered by ``meta`` are left untouched (undefined, like ``torch.empty_like``).  Scores are held
    in fp32: rows that see any beyond 2^29 in magnitude may come out wrong or NaN.
    """
    nb, kvh = check_layer_views(k_cache, v_cache, kv8=True)
    dev = k_cache.device
    shape = q.shape
    q_stride = _rows(q, "q")
    index = k_cache.get_device()
    if q.get_device() != index or meta.plan.get_device() != index:
        raise ValueError(f"q and meta are on {q.device} and {meta.plan.device}, the pool on {dev}")
    need = meta.num_tokens
    if shape[0] < need and shape[0] < (need := meta.rows_needed()):
        raise ValueError(f"q must have the step's {need} rows")
    if out is None:
        out = torch.empty_like(q)
        out_stride = out.stride(0)
    else:
        out_stride = _rows(out, "out")
        if out.get_device() != index:
            raise ValueError(f"out is on {out.device}, the pool on {dev}")
        if out.shape[1:] != shape[1:] or (out.shape[0] < need and out.shape[0] < meta.rows_needed()):
            raise ValueError(f"out must have q's heads and the step's {meta.rows_needed()} rows")
    kv8 = is_kv8(k_cache)
    scale = float(scale)
    lib = _capi.load()
    stream = _stream(dev)
    q_args = (q.data_ptr(), q_stride, out.data_ptr(), out_stride, shape[1], kvh)
    info, tree = meta.info, meta.tree
    if tree is None or info.n_decode_items or info.n_tile_items or info.n_tc_items:
        if kv8:
            plan8, info8 = meta.for_kv8()
        ws = meta.workspace(kvh, dev, kv8, kv8)
        ws_args = (0, 0) if ws is None else (ws.data_ptr(), ws.numel())
        if kv8:
            rc = _on_own_device(
                lib.ms_paged_attention_kv8, dev, *q_args, k_cache.data_ptr(), nb,
                plan8.data_ptr(), C.byref(info), C.byref(info8), *ws_args, scale, stream)
        else:
            rc = _on_own_device(
                lib.ms_paged_attention, dev, *q_args, k_cache.data_ptr(), v_cache.data_ptr(), nb,
                meta.plan.data_ptr(), C.byref(info), *ws_args, scale, stream)
        _capi.check(rc, "paged_attention")
    if tree is not None:
        if kv8:
            plan8, info8 = tree.for_kv8()
        ws = tree.workspace(kvh, dev, kv8, True)
        ws_args = (0, 0) if ws is None else (ws.data_ptr(), ws.numel())
        if kv8:
            rc = _on_own_device(
                lib.ms_tree_attention_kv8, dev, *q_args, k_cache.data_ptr(), nb,
                plan8.data_ptr(), C.byref(tree.info), C.byref(info8), *ws_args, scale, stream)
        else:
            rc = _on_own_device(
                lib.ms_tree_attention, dev, *q_args, k_cache.data_ptr(), v_cache.data_ptr(), nb,
                tree.plan.data_ptr(), C.byref(tree.info), *ws_args, scale, stream)
        _capi.check(rc, "paged_attention")
    return out


def paged_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    meta: AttentionMetadata,
    scale: float,
) -> Tensor:
    """Write this step's keys and values into the cache, then attend through it.

    q: [T, heads, 128]; k, v: [T, kv_heads, 128]; caches: layer views of the pool.
    Returns [T, heads, 128] (backends.py:145-158).
    """
    kv_scatter(k, v, meta.slot_mapping, k_cache, v_cache)
    return attend(q, k_cache, v_cache, meta, scale)
