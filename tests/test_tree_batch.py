"""Packing of draft trees next to prefill chunks and decode rows (no GPU)."""
from __future__ import annotations

import time

import numpy as np
import pytest

from railgun_amd.batch import _check_tree_blocks, DecodeSlot, DraftTree, PrefillChunk, pack_step


def test_rows_of_a_mixed_step():
    b = pack_step([PrefillChunk([1, 2, 3], 4, [7, 8])], [DecodeSlot(9, 6, [2, 3])], 4,
                  draft_trees=[DraftTree([20, 21, 22, 23], [-1, 0, 0, 2], 10, [5, 6, 1]), DraftTree([30], [-1], 1, [9]),
                               DraftTree([40, 41], [-1, 0], 7, [10, 11], position=50)])
    assert (b.num_prefill_tokens, b.num_decode, b.num_trees, b.num_tokens, b.num_requests) == (3, 1, 3, 11, 5)
    assert b.first_tree_row == 4 and b.max_tree_nodes == 4 and b.max_tree_depth == 3
    np.testing.assert_array_equal(b.tokens, [1, 2, 3, 9, 20, 21, 22, 23, 30, 40, 41])
    np.testing.assert_array_equal(b.positions, [4, 5, 6, 5, 6, 7, 7, 8, 0, 50, 51])
    np.testing.assert_array_equal(b.slot_mapping, [32, 33, 34, 13, 26, 27, 4, 5, 36, 45, 46])
    np.testing.assert_array_equal(b.context_lens, [7, 6, 10, 1, 7])
    np.testing.assert_array_equal(b.block_table[2:], [[5, 6, 1], [9, 0, 0], [10, 11, 0]])
    np.testing.assert_array_equal(b.last_rows, [2, 3, 4, 5, 6, 7, 8, 9, 10])
    np.testing.assert_array_equal(b.tree_cu, [0, 4, 5, 7])
    np.testing.assert_array_equal(b.tree_parents, [-1, 0, 0, 2, -1, -1, 0])
    np.testing.assert_array_equal(b.tree_places, [6, 0, 50])


def test_steps_without_trees_stay():
    b = pack_step([PrefillChunk([1, 2], 0, [7])], [DecodeSlot(9, 6, [2, 3])], 4)
    assert b.num_trees == 0 and b.num_decode == 1 and b.max_tree_nodes == 0
    np.testing.assert_array_equal(b.last_rows, [1, 2])


@pytest.mark.parametrize("tree,text", [
    (DraftTree([], [], 3, [1]), "draft tree of 0"), (DraftTree([1, 2], [-1], 3, [1]), "parents"),
    (DraftTree([1, 2], [0, 0], 3, [1]), "token 0"), (DraftTree([1, 2], [-1, 1], 3, [1]), "token 1"),
    (DraftTree([1, 2], [-1, -1], 3, [1]), "token 1"), (DraftTree([1, 2], [-1, 0], 1, [1]), "seq_len"),
    (DraftTree([1, 2], [-1, 0], 5, [1]), "needs more than 1 blocks"), (DraftTree([1, 2], [-1, 0], 4, [-1]), "block id"),
    (DraftTree([1, 2], [-1, 0], 4, [1], position=1), "position 1"),
    (DraftTree([0] * 1025, list(range(-1, 1024)), 1025, [1] * 300), "1025"),
])
def test_refused_trees(tree, text):
    with pytest.raises(ValueError, match=text):
        pack_step([], [], 4, draft_trees=[tree])


def test_blocks_of_a_tree_are_its_own():
    """Blocks in front of the trees may be shared, those that hold their tokens may not."""
    def step(a, b, slots=()):
        return pack_step([], list(slots), 4, draft_trees=[DraftTree([1, 2], [-1, 0], 10, a), DraftTree([1, 2], [-1, 0], 9, b)])

    step([1, 2, 3], [1, 4, 5])                      # the second tree begins in its second block
    for a, b, slots in (([1, 2, 3], [1, 2, 3], ()), ([1, 2, 3], [4, 5, 3], ()), ([1, 2, 3], [1, 3, 5], ()),
                        ([1, 2, 2], [4, 5, 6], ()), ([1, 2, 3], [4, 5, 6], [DecodeSlot(1, 9, [7, 8, 3])])):
        with pytest.raises(ValueError, match="appears twice"):
            step(a, b, slots)
    step([1, 2, 3], [4, 5, 6], [DecodeSlot(1, 8, [7, 8, 3])])   # an entry behind the slot's tokens


@pytest.mark.parametrize("table,nodes", [([5, 5], 20), ([7, 5, 5], 20), ([5, 6, 5], 40), ([4, 4, 6], 33)])
def test_a_block_twice_in_a_tree(table, nodes):
    """Two of the tree's own tokens would share a slot."""
    seq_len = 16 * len(table) - 7
    tree = DraftTree([1] * nodes, list(range(-1, nodes - 1)), seq_len, table)
    with pytest.raises(ValueError, match="appears twice"):
        pack_step([], [], 16, draft_trees=[tree])
    pack_step([], [], 16, draft_trees=[DraftTree([1] * nodes, tree.parents, seq_len, range(len(table)))])


def test_packing_many_trees():
    """The check of the trees' blocks costs less than the packing of as many decode rows: it looks at every table
    entry once, not once a tree.  (The least of five runs each; the margin is more than five times either way.)"""
    seqs, blocks = 1024, 256
    tables = [list(range(s * blocks, (s + 1) * blocks)) for s in range(seqs)]
    trees = [DraftTree([1] * 8, list(range(-1, 7)), 16 * blocks - 3, t) for t in tables]
    table, ctx = np.asarray(tables, np.int32), np.full(seqs, 16 * blocks - 3, np.int64)

    def least(call):
        took = []
        for _ in range(5):
            t0 = time.perf_counter()
            call()
            took.append(time.perf_counter() - t0)
        return min(took)

    check = least(lambda: _check_tree_blocks(trees, table, ctx, 16))
    assert check < least(lambda: pack_step([], [DecodeSlot(1, 16 * blocks - 3, t) for t in tables], 16))
