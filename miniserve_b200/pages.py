"""Whole pages of a cache: copied, cleared, and counted while sequences fork, end and move together.

No reference counterpart (its block manager shares pages between sequences with equal prefixes, and never
copies one).  ``copy_pages`` and ``clear_pages`` work on any paged tensor ``[layers, num_blocks, ...]``: a
pool of either kind, key bounds.  ``CachePages`` keeps the free list and the reference counts for a host that
has no block manager of its own, or wants forks and compaction beside it.
"""

from __future__ import annotations

import math
import struct
from collections import Counter
from collections.abc import Sequence
from itertools import chain

import numpy as np
from torch import Tensor

from . import _capi
from .attention import _on_own_device, _stream
from .kv_pool import BLOCK_SIZE


def _paged(pool: Tensor) -> tuple[int, int, int]:
    """(layers, blocks, bytes of a block) of a paged tensor."""
    shape = pool.shape
    if len(shape) < 3 or not pool.is_contiguous():
        raise ValueError("pool must be a contiguous paged tensor [layers, num_blocks, ...]")
    # Not the stride of a block: where there is one block, a contiguous tensor may have any.
    return shape[0], shape[1], math.prod(shape[2:]) * pool.element_size()


def _block_list(blocks: Sequence[int] | np.ndarray, name: str) -> tuple[bytes, int]:
    """Block numbers as the library reads them (host memory; it checks that the pool has them), and how
    many."""
    try:
        if isinstance(blocks, np.ndarray):
            if blocks.ndim != 1 or (blocks.size and blocks.dtype.kind not in "iu"):
                raise TypeError
            if blocks.size and not 0 <= int(blocks.min()) <= int(blocks.max()) < 1 << 31:
                raise struct.error
            return blocks.astype(np.int32).tobytes(), blocks.size
        if isinstance(blocks, (bytes, bytearray, str)):
            raise TypeError
        n = len(blocks)
        # The fastest way from a list of Python integers to an array: 1000 of them 22 us, array("i") 34.
        return struct.pack(f"{n}i", *blocks), n
    except TypeError:
        raise ValueError(f"{name} must be a list of block numbers") from None
    except struct.error:
        raise ValueError(f"{name} must be a list of block numbers of the pool's blocks") from None


def copy_pages(pool: Tensor, src: Sequence[int] | np.ndarray, dst: Sequence[int] | np.ndarray) -> None:
    """Copy block ``src[i]`` of every layer to block ``dst[i]``.  The lists are host memory (a captured
    call keeps them).  No block is written twice, or both written and read, by one call; one block may go
    to several.  ``attend`` waits for the copies."""
    layers, blocks, page = _paged(pool)
    (s, n), (d, places) = _block_list(src, "src"), _block_list(dst, "dst")
    if n != places:
        raise ValueError(f"{n} blocks to copy but {places} places")
    if n == 0 or layers == 0:
        return
    dev = pool.device
    rc = _on_own_device(_capi.load().ms_copy_pages, dev, pool.data_ptr(), blocks * page, page, layers,
                        blocks, s, d, n, _stream(dev))
    _capi.check(rc, "copy_pages")


def clear_pages(pool: Tensor, blocks: Sequence[int] | np.ndarray) -> None:
    """Fill the listed blocks of every layer with zeros: a page that held an infinity or a NaN passes
    neither on to the next sequence that is given it.  ``attend`` waits for it."""
    layers, num_blocks, page = _paged(pool)
    b, n = _block_list(blocks, "blocks")
    if n == 0 or layers == 0:
        return
    dev = pool.device
    rc = _on_own_device(_capi.load().ms_clear_pages, dev, pool.data_ptr(), num_blocks * page, page, layers,
                        num_blocks, b, n, _stream(dev))
    _capi.check(rc, "clear_pages")


class CachePages:
    """The pages of one or more paged tensors of as many blocks (a pool and its key bounds): which are
    free, and how many block tables hold each.  Copies and clearing are queued on the current stream."""

    def __init__(self, *tensors: Tensor) -> None:
        if not tensors:
            raise ValueError("CachePages needs a paged tensor")
        sizes = {_paged(t)[1] for t in tensors}
        if len(sizes) != 1:
            raise ValueError(f"paged tensors of different numbers of blocks: {sorted(sizes)}")
        # What a copy would refuse, or do to a page that another tensor's copy still reads, is refused here: the
        # counts change before the copies are queued.
        for t in tensors:
            if _paged(t)[2] % 16 or t.data_ptr() % 16:
                raise ValueError("paged tensors need pages of whole multiples of 16 bytes on 16-byte boundaries")
        spans = sorted((str(t.device), t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                       for t in tensors)
        if any(a[0] == b[0] and b[1] < a[2] for a, b in zip(spans, spans[1:])):
            raise ValueError("paged tensors must not share memory")
        self.tensors = tensors
        self.num_blocks = sizes.pop()
        self._free = list(range(self.num_blocks - 1, -1, -1))  # the lowest is taken first
        self._held: Counter[int] = Counter()  # tables that hold a page

    @property
    def num_free(self) -> int:
        return len(self._free)

    def holders(self, block: int) -> int:
        """How many block tables hold a page."""
        return self._held[block]

    def allocate(self, count: int) -> list[int]:
        """``count`` free pages, held once each."""
        if count < 0 or count > len(self._free):
            raise RuntimeError(f"{count} pages wanted, {len(self._free)} free")
        taken = [self._free.pop() for _ in range(count)]
        self._held.update(taken)
        return taken

    def _check_held(self, named: Counter[int]) -> None:
        for block, times in named.items():
            if self._held[block] < times:
                raise ValueError(f"block {block} is held by {self._held[block]} tables, named {times} times")

    def fork(self, tables: Sequence[Sequence[int]], num_tokens: Sequence[int], copies: int = 1
             ) -> list[list[list[int]]]:
        """``copies`` new block tables for each sequence's first ``num_tokens`` tokens.  Whole pages are
        shared, the page that would still be written to is copied (one launch for all of them per tensor):
        the forks and their origin can all be continued.  Raises with nothing changed where the free pages do
        not suffice."""
        if len(tables) != len(num_tokens) or copies < 0:
            raise ValueError("fork needs one token count per table, and copies >= 0")
        for table, n in zip(tables, num_tokens):
            if n < 0 or len(table) * BLOCK_SIZE < n:
                raise ValueError(f"a table of {len(table)} pages does not hold {n} tokens")
            self._check_held(Counter(table[: -(-n // BLOCK_SIZE)]))
        partial = [n % BLOCK_SIZE != 0 for n in num_tokens]
        fresh = self.allocate(sum(partial) * copies)
        src, out, at = [], [], 0
        for table, n, part in zip(tables, num_tokens, partial):
            whole = list(table[: n // BLOCK_SIZE])
            forks = []
            for _ in range(copies):
                self._held.update(whole)
                forks.append(whole + fresh[at : at + part])
                at += part
            if part:
                src += [table[n // BLOCK_SIZE]] * copies
            out.append(forks)
        for t in self.tensors:
            copy_pages(t, src, fresh)
        return out

    def free(self, tables: Sequence[Sequence[int]], clear: bool = True) -> list[int]:
        """Give up block tables.  Pages that no other table holds become free and, with ``clear``, are
        filled with zeros; returns them."""
        named = Counter(chain.from_iterable(tables))
        self._check_held(named)
        self._held.subtract(named)
        gone = sorted((b for b in named if self._held[b] == 0), reverse=True)
        for b in gone:
            del self._held[b]
        self._free += gone
        if clear:
            for t in self.tensors:
                clear_pages(t, gone)
        return gone

    def compact(self, tables: Sequence[Sequence[int]], clear: bool = True) -> list[list[int]]:
        """Move the pages in use to the lowest block numbers and return ``tables`` (all that are held)
        rewritten.  Only pages that lie behind are moved; with ``clear`` the places they leave are filled
        with zeros."""
        if Counter(chain.from_iterable(tables)) != self._held:
            raise ValueError("compact needs every block table that is held, as often as it is")
        live = len(self._held)
        src = sorted(b for b in self._held if b >= live)
        dst = sorted(b for b in self._free if b < live)
        for t in self.tensors:
            copy_pages(t, src, dst)
            if clear:
                clear_pages(t, src)
        to = dict(zip(src, dst))
        self._held = Counter({to.get(b, b): n for b, n in self._held.items()})
        self._free = list(range(self.num_blocks - 1, live - 1, -1))
        return [[to.get(b, b) for b in table] for table in tables]
