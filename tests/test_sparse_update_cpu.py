"""Later steps that a captured step over selected pages takes: what its launches depend on bounds them."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import attention
from miniserve_b200.attention import AttentionMetadata, SeqChunk, plan_batch


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch) -> None:
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    def write(self, packed, info, kv8) -> None:
        self.info, self._packed = info, packed[: int(info.total_ints)]

    monkeypatch.setattr(AttentionMetadata, "_write", write)


def step(lengths) -> AttentionMetadata:
    c = chunks(lengths)
    packed, info = plan_batch(c, len(c), 16, 148, pages_per_split=4096)
    return AttentionMetadata(torch.zeros(len(c), dtype=torch.int64), torch.from_numpy(packed), info, len(c),
                             _pages_per_split=4096, _packed=packed)


def chunks(lengths) -> list[SeqChunk]:
    """Decode rows of as many pages in all, whatever their lengths."""
    return [SeqChunk(i, 1, n - 1, list(range(p))) for i, (n, p) in enumerate(lengths)]


def test_a_longest_row_that_gets_shorter_is_taken() -> None:
    """Rows of 65 and 63 pages, then of 64 and 64: fewer pages than the launches allow for."""
    meta = step([(1030, 65), (1000, 63)])
    assert meta.short_rows() == (1, 128)
    assert meta.update(chunks([(1020, 64), (1020, 64)]))
    # The bound stays the launches', and they take the longer row again.
    assert meta.short_rows() == (1, 128)
    assert meta.update(chunks([(1030, 65), (1000, 63)]))
    # Beyond the bound.
    assert not meta.update(chunks([(2060, 129), (8, 1)]))
    meta = step([(1020, 64), (1020, 64)])
    assert meta.short_rows() == (1, 64)
    assert not meta.update(chunks([(1030, 65), (1000, 63)]))
