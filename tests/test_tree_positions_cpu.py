"""RoPE positions of draft trees: what the planner refuses, ``tree_positions`` refuses too."""

from __future__ import annotations

import pytest

import miniserve_b200
from miniserve_b200 import SeqChunk, tree_positions
from miniserve_b200.attention import plan_tree_batch


def test_unused_positions() -> None:
    unused = miniserve_b200.UNUSED_DRAFT
    assert tree_positions(7, [-1, 0, unused, 1, -1, 3]) == [7, 8, 7, 9, 7, 10]
    assert tree_positions(7, []) == []


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 5], [-1, -3], [-1, -2, 1], [-2, 0]])
def test_bad_parents(parents: list[int]) -> None:
    with pytest.raises(ValueError, match="has parent"):
        tree_positions(7, parents)
    with pytest.raises(ValueError, match="has parent"):
        plan_tree_batch([SeqChunk(0, len(parents), 7, [0], parents=parents)], len(parents))
