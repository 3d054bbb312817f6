"""Packing prompt chunks behind a cache that eviction has shortened."""
from __future__ import annotations

import pytest

from railgun_amd.batch import DecodeSlot, PrefillChunk, pack_step


def test_a_chunk_behind_an_evicted_cache():
    """Ten cached tokens of a text of 57: cells from the tenth on, rotations from the 57th."""
    st = pack_step([PrefillChunk([1, 2, 3], 10, [4, 5, 6, 7], position=57), PrefillChunk([8, 9], 2, [1])],
                   [DecodeSlot(1, 5, [2, 3], position=30)], 4)
    assert st.positions.tolist() == [57, 58, 59, 2, 3, 30]
    assert st.slot_mapping.tolist() == [6 * 4 + 2, 6 * 4 + 3, 7 * 4, 6, 7, 12]
    assert st.context_lens.tolist() == [13, 4, 5] and st.cu_seqlens.tolist() == [0, 3, 5]


def test_a_chunk_before_its_cached_tokens():
    with pytest.raises(ValueError, match="position 9"):
        pack_step([PrefillChunk([1], 10, [4, 5, 6], position=9)], [], 4)
