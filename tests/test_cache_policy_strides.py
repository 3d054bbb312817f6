"""Views of caches and scores that the bindings take and refuse (no GPU)."""
from __future__ import annotations

import pytest
import torch

from railgun_amd.ops import RailgunError, cache_geometry, check_scores

NB, HKV, BS, D = 6, 2, 16, 64


def test_blocks_that_are_one_block_expanded():
    one = torch.zeros(1, HKV, BS, D)
    with pytest.raises(RailgunError, match="apart"):
        cache_geometry(one.expand(NB, HKV, BS, D), one.expand(NB, HKV, BS, D))
    cache = torch.zeros(NB, HKV, BS, D)
    with pytest.raises(RailgunError, match="apart"):
        check_scores(torch.zeros(1, HKV, BS).expand(NB, HKV, BS), cache)
    with pytest.raises(RailgunError, match="apart"):
        check_scores(torch.zeros(3, 1, HKV, BS).expand(3, NB, HKV, BS), torch.zeros(3, NB, HKV, BS, D))


def test_blocks_apart_by_any_stride():
    pool = torch.zeros(NB, 2, HKV, BS, D)
    assert cache_geometry(pool[:, 0], pool[:, 1]) == (HKV, BS, D, 2 * HKV * BS * D)
    assert cache_geometry(pool[:1, 0], pool[:1, 1])[:3] == (HKV, BS, D)
    check_scores(torch.zeros(NB, 5 * HKV * BS)[:, :HKV * BS].view(NB, HKV, BS), pool[:, 0])
    check_scores(torch.zeros(1, HKV, BS).expand(1, HKV, BS), pool[:1, 0])
