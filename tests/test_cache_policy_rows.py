"""Scored decode steps whose rows change: every cell that a row's scored length counts holds that row's
weights, or 0 where it never gathered any, and nothing of an earlier owner's.

The steps run over a pool of cells by the entry's contract (cell <- (t < scored ? cell : 0) + weight for
first <= t < length), with a weight of its own per step, row and position."""
from __future__ import annotations

import numpy as np
import pytest

from railgun_amd.batch import DecodeSlot, pack_step

BS = 4


class Cells:
    """The scores of a pool of blocks, left over from earlier owners: NaN."""

    def __init__(self, blocks):
        self.cell = np.full(blocks * BS, np.nan)
        self.rng = np.random.default_rng(0)

    def step(self, rows):
        """rows: [(table, length, scored)] with the new token counted; the weights that were added, per row."""
        st = pack_step([], [DecodeSlot(1, n, t, scored_len=s) for t, n, s in rows], BS, share_prefix=True,
                       gather_scores=True)
        self.cell[st.unscored_slots] = 0.0
        first, added = st.shared_decode_blocks * BS, []
        for (table, n, scored), told in zip(rows, st.scored_lens):
            assert told == scored
            w = self.rng.integers(1, 1000, n).astype(float)
            w[:first] = 0
            for t in range(first, n):
                at = table[t // BS] * BS + t % BS
                self.cell[at] = (self.cell[at] if t < scored else 0.0) + w[t]
            added.append(w)
        return added

    def of(self, table, n):
        t = np.arange(n)
        return self.cell[np.asarray(table)[t // BS] * BS + t % BS]


def grown(a, n):
    return np.concatenate([a, np.zeros(n - len(a))])


def test_a_row_leaves():
    c, prefix = Cells(16), [3, 9]
    a, b = prefix + [1, 2], prefix + [4, 5]
    want = np.zeros(0)
    for i in range(3):
        w, _ = c.step([(a, 9 + i, 0 if i == 0 else 8 + i), (b, 10 + i, 0 if i == 0 else 9 + i)])
        want = grown(want, 9 + i) + w
        np.testing.assert_array_equal(c.of(a, 9 + i), want)
    w, = c.step([(a, 12, 11)])                     # alone: its own tokens from the first on
    np.testing.assert_array_equal(c.of(a, 12), grown(want, 12) + w)
    assert w[0] > 0 and (want[:8] == 0).all()


def test_another_row_joins_and_the_prefix_gets_shorter():
    c = Cells(16)
    a, b, d = [3, 9, 1, 2], [3, 9, 4, 5], [3, 6, 7, 8]
    w0, _ = c.step([(a, 9, 0), (b, 9, 0)])
    c.cell[6 * BS:9 * BS] = 5e5                    # d's own blocks, used before
    # a and d: blocks 9 and 6 differ, so the prefix is block 3 alone, and block 9 is a's from now on.
    w1, w2 = c.step([(a, 10, 9), (d, 13, 0)])
    assert w1[4] > 0 and w1[3] == 0
    np.testing.assert_array_equal(c.of(a, 10), grown(w0, 10) + w1)
    np.testing.assert_array_equal(c.of(d, 13), w2)


def test_a_prefix_that_holds_scores_keeps_them():
    c = Cells(16)
    a, b = [3, 9, 1], [3, 9, 4]
    w0, = c.step([(a, 9, 0)])                      # alone, so its first two blocks gather too
    w1, w2 = c.step([(a, 10, 9), (b, 9, 0)])       # then another begins with them
    np.testing.assert_array_equal(c.of(a, 10), grown(w0, 10) + w1)
    np.testing.assert_array_equal(c.of(b, 9)[:8], w0[:8])
    np.testing.assert_array_equal(c.of(b, 9)[8:], w2[8:])


@pytest.mark.parametrize("scored,want", [((0, 0), range(0, 8)), ((5, 0), range(5, 8)), ((2, 7), range(7, 8)),
                                         ((8, 3), range(0)), ((0, 9), range(0))])
def test_the_slots_that_no_row_counts(scored, want):
    st = pack_step([], [DecodeSlot(1, 10, t, scored_len=s) for t, s in zip(([3, 9, 1], [3, 9, 4]), scored)], BS,
                   share_prefix=True, gather_scores=True)
    assert st.unscored_slots.dtype == np.int32
    assert st.unscored_slots.tolist() == [[3, 9][t // BS] * BS + t % BS for t in want]


def test_steps_without_scores_or_a_prefix():
    rows = [DecodeSlot(1, 10, [3, 9, 1], scored_len=0)]
    assert pack_step([], rows, BS, share_prefix=True).unscored_slots is None
    assert pack_step([], rows, BS, share_prefix=True, gather_scores=True).unscored_slots.size == 0
    assert pack_step([], [], BS, gather_scores=True).unscored_slots.size == 0
