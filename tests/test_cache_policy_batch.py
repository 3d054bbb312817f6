"""Packing decode steps for a shared prefix, gathered scores and evicted caches."""
from __future__ import annotations

import pytest

from railgun_amd.batch import DecodeSlot, PrefillChunk, pack_step, shared_prefix_blocks


def slots(*rows):
    return [DecodeSlot(1, n, t) for n, t in rows]


@pytest.mark.parametrize("rows,want", [
    ([(9, [5, 6, 7]), (12, [5, 6, 8])], 2),
    ([(9, [5, 6, 7]), (8, [5, 6])], 1),            # the second writes its last token into block 6
    ([(9, [5, 6, 7])], 0),
    ([], 0),
    ([(9, [5, 6, 7]), (9, [6, 5, 7])], 0),
    ([(9, [5, 6, 7]), (9, [5, 9, 7])], 1),
    ([(9, [5, 6, 7]), (1, [8])], 0),
    ([(13, [5, 6, 7, 1]), (13, [5, 6, 7, 2]), (14, [5, 6, 3, 4])], 2),
])
def test_shared_blocks(rows, want):
    assert shared_prefix_blocks(slots(*rows), 4) == want
    assert pack_step([], slots(*rows), 4, share_prefix=True).shared_decode_blocks == want
    assert pack_step([], slots(*rows), 4).shared_decode_blocks == 0


def test_prefill_rows_do_not_count():
    st = pack_step([PrefillChunk([1, 2], 0, [11])], slots((9, [5, 6, 7]), (12, [5, 6, 8])), 4, share_prefix=True)
    assert st.shared_decode_blocks == 2 and st.scored_lens is None


def test_position_past_the_cached_length():
    st = pack_step([], [DecodeSlot(1, 9, [5, 6, 7], position=40), DecodeSlot(1, 5, [3, 4])], 4)
    assert st.positions.tolist() == [40, 4] and st.context_lens.tolist() == [9, 5]
    assert st.slot_mapping.tolist() == [7 * 4 + 0, 4 * 4 + 0]
    with pytest.raises(ValueError, match="position 7"):
        pack_step([], [DecodeSlot(1, 9, [5, 6, 7], position=7)], 4)


def test_scored_lens():
    rows = [DecodeSlot(1, 9, [5, 6, 7], scored_len=0), DecodeSlot(1, 10, [5, 6, 8], scored_len=9)]
    st = pack_step([], rows, 4, share_prefix=True, gather_scores=True)
    assert st.scored_lens.tolist() == [0, 9] and str(st.scored_lens.dtype) == "int32"
    with pytest.raises(ValueError, match="scored twice"):      # the prefix's blocks without share_prefix
        pack_step([], rows, 4, gather_scores=True)
    for bad in (None, 9, -1):
        with pytest.raises(ValueError, match="scored_len"):
            pack_step([], [DecodeSlot(1, 9, [5, 6, 7], scored_len=bad)], 4, gather_scores=True)
    three = rows + [DecodeSlot(1, 9, [5, 9, 7], scored_len=0)]  # one block shared by all, block 7 by two
    with pytest.raises(ValueError, match="block 7 is scored twice|block 6 is scored twice"):
        pack_step([], three, 4, share_prefix=True, gather_scores=True)
    # A block past a row's tokens is not scored.
    pack_step([], [DecodeSlot(1, 3, [5, 6], scored_len=0), DecodeSlot(1, 4, [6], scored_len=3)], 4, gather_scores=True)
