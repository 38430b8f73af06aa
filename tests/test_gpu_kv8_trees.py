"""Draft trees over an 8-bit pool, where kernel F alone runs, at f16's rounding of the weights (2^-11), not
at that of the bf16 kernels beside it."""

from __future__ import annotations

import random

import pytest
import torch

from miniserve_b200.attention import SeqChunk, attend, build_attention_metadata
from paged_reference import SCALE, U_F16, assert_close, attention64
from test_gpu_tree import batch, random_tree, slots_of

pytestmark = pytest.mark.gpu


def close(out, q, views, chunks) -> None:
    ref, bound, rows = attention64(q, *views, chunks, U_F16)
    assert_close(out, ref, bound, rows)


@pytest.mark.parametrize("split", [0, 9])
def test_beside_decode_rows_and_short_chunks(split: int, cuda_device) -> None:
    rng = random.Random(1)
    seqs = [(12, 300, random_tree(rng, 12)), (1, 700, None), (40, 90, None), (33, 610, random_tree(rng, 33)),
            (3, 1500, None), (63, 1100, random_tree(rng, 63, unused=9)), (17, 0, random_tree(rng, 17))]
    views, chunks, q = batch(cuda_device, seqs, 4, "e4m3", seed=21)
    meta = build_attention_metadata(chunks, slots_of(chunks, cuda_device), 16, pages_per_split=split)
    close(attend(q, *views, meta, SCALE), q, views, chunks)


def test_long_contexts_and_large_trees(cuda_device) -> None:
    rng = random.Random(2)
    seqs = [(24, 9000, random_tree(rng, 24)), (7, 12000, random_tree(rng, 7)),
            (200, 2000, random_tree(rng, 200))]
    views, chunks, q = batch(cuda_device, seqs, 2, "e4m3", seed=22)
    meta = build_attention_metadata(chunks, slots_of(chunks, cuda_device), 16)
    close(attend(q, *views, meta, SCALE), q, views, chunks)


def test_replays_of_a_captured_step(cuda_device) -> None:
    dev = cuda_device
    rng = random.Random(3)
    seqs = [(20, 900, random_tree(rng, 20)), (9, 333, random_tree(rng, 9)), (2, 700, None)]
    views, chunks, q = batch(dev, seqs, 4, "e4m3", seed=23)
    meta = build_attention_metadata(chunks, slots_of(chunks, dev), 16, pages_per_split=16)
    attend(q, *views, meta, SCALE)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(q, *views, meta, SCALE)
    for step in (1, 2, 3):
        new = [SeqChunk(c.flat_start, c.num_new, c.num_cached - (0 if c.parents is None else step),
                        c.block_table, parents=c.parents and random_tree(rng, c.num_new, unused=step))
               for c in chunks]
        q.copy_(torch.randn(q.shape, device=dev))
        assert meta.update(new, slots_of(new, dev))
        graph.replay()
        close(out, q, views, new)
