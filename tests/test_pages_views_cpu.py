"""Views of paged tensors: what the calls over whole pages take for a page."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import _capi, pages
from miniserve_b200.pages import clear_pages, copy_pages


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
