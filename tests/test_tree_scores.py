"""Scores of slots that there may not be (no GPU)."""
from __future__ import annotations

import torch

from railgun_amd.kv_pool import GpuBlockPool


def test_cells_of_no_slot():
    """Slots below 0 are passed over; the cells of the others are cleared, in every layer, and no more."""
    pool = GpuBlockPool(2, 5, 2, 4, 8, "cpu", dtype=torch.float32)
    pool.scores.fill_(3.0)
    pool.clear_scores(torch.tensor([-1, 0, 7, -1, 19], dtype=torch.int32))
    want = torch.full((2, 5, 2, 4), 3.0)
    for block, at in ((0, 0), (1, 3), (4, 3)):
        want[:, block, :, at] = 0
    assert pool.scores.shape == want.shape and torch.equal(pool.scores, want)
    pool.scores.fill_(3.0)
    pool.clear_scores(torch.tensor([-1, -1], dtype=torch.int32))
    assert (pool.scores == 3).all()
