"""Views of paged tensors: what the calls over whole pages take for a page."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import _capi, pages
from miniserve_b200.pages import CachePages, clear_pages, copy_pages


class Calls:
    """The library, which keeps the arguments of its calls and launches nothing."""

    def __init__(self) -> None:
        self.made: list[tuple] = []

    def __getattr__(self, name: str):
        return lambda *args: self.made.append((name, *args)) or _capi.MS_OK


@pytest.fixture
def lib(monkeypatch) -> Calls:
    fake = Calls()
    monkeypatch.setattr(_capi, "load", lambda path=None: fake)
    monkeypatch.setattr(pages, "_stream", lambda device: 0)
    return fake


def test_a_view_of_one_block_has_pages_of_its_own_size(lib) -> None:
    """A tensor of one layer and one block counts as contiguous whatever its strides: its page is 32 bytes, not
    the 10 pages that lie between it and the next block of such a view."""
    pool = torch.zeros(1, 10, 2, 16, dtype=torch.uint8)
    view = pool[:, ::10]
    assert view.is_contiguous() and view.stride(1) == 320
    clear_pages(view, [0])
    copy_pages(view, [0], [0])
    for name, base, layer, page, layers, blocks, *_ in lib.made:
        assert (base, layer, page, layers, blocks) == (pool.data_ptr(), 32, 32, 1, 1), name
    one = torch.zeros(3, 1, 2, 16, dtype=torch.uint8)
    for tensor in (one, one.as_strided(one.shape, (32, 7, 16, 1)), torch.zeros(3, 4, 8).bfloat16()[:, 1:2][:1]):
        lib.made.clear()
        clear_pages(tensor, [0])
        size = tensor[0, 0].numel() * tensor.element_size()
        assert lib.made[0][2:6] == (size, size, tensor.shape[0], 1)


def test_tensors_whose_pages_cannot_be_moved_are_refused_at_first(lib) -> None:
    """Not when a fork or an end of a sequence has already changed the counts."""
    for odd in (torch.zeros(1, 8, 24, dtype=torch.uint8), torch.zeros(3, 8, 4, dtype=torch.bfloat16),
                torch.zeros(8 * 32 + 1, dtype=torch.uint8)[1:].view(1, 8, 32)):
        with pytest.raises(ValueError, match="16"):
            CachePages(torch.zeros(2, 8, 32, dtype=torch.uint8), odd)
    CachePages(torch.zeros(2, 8, 32, dtype=torch.uint8), torch.zeros(3, 8, 16, dtype=torch.uint8))
    assert lib.made == []


def test_tensors_that_share_memory_are_refused(lib) -> None:
    """``compact`` moves and clears one tensor after the other: a tensor given twice would lose its pages."""
    pool = torch.zeros(4, 8, 32, dtype=torch.uint8)
    for more in ((pool,), (pool[1:3],), (torch.zeros(1, 8, 16), pool[3:]), (pool.view(torch.int16),)):
        with pytest.raises(ValueError, match="share memory"):
            CachePages(pool, *more)
    pages = CachePages(pool[:2], pool[2:])
    table = pages.allocate(3)
    pages.free([table[:2]])
    assert pages.compact([table[2:]]) == [[0]]
    assert [name for name, *_ in lib.made] == ["ms_clear_pages"] * 2 + ["ms_copy_pages", "ms_clear_pages"] * 2
