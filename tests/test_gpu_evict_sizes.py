"""Evictions of unusual sizes: many chunks of the move, budgets far past what a table holds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import i32
from test_gpu_evict import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dst", ["apart", "in place"])
def test_more_chunks_than_a_grid_has_in_y(device, kernels, dst):
    """Rows of 1,000 bytes move in 2-byte pieces, a token a workgroup: 66,000 of them."""
    Case(device, [70100, 300], 66000, dtype="f32", hkv=1, d=250, dst=dst, seed=2).check(kernels, 50, 9)


@pytest.mark.parametrize("budget", [161, 100000, 2**31 - 1])
def test_budgets_past_the_table(device, kernels, budget):
    """Nothing is dropped, and nothing is asked for by the budget: the workspace holds what the table does."""
    pool = torch.randn((2, 12, 2, 2, 16, 64), device=device).bfloat16()
    scores = torch.rand((2, 12, 2, 16), device=device)
    before = pool.clone()
    table = i32(np.arange(10)[None], device)
    out = torch.zeros(1, dtype=torch.int32, device=device)
    guard = torch.full((256 + 4 * 160 * 4 + 64,), 77, dtype=torch.uint8, device=device)
    kernels.launch_evict(pool[:, :, 0], pool[:, :, 1], scores, table, None, i32([155], device), out, None, budget, 8, 4,
                         guard[:-64])
    assert out.tolist() == [155] and torch.equal(pool, before) and (guard[-64:] == 77).all()
    torch.cuda.reset_peak_memory_stats(device)
    held = torch.cuda.memory_allocated(device)
    kernels.launch_evict(pool[:, :, 0], pool[:, :, 1], scores, table, None, i32([155], device), out, None, budget, 8, 4)
    assert torch.cuda.max_memory_allocated(device) - held < 1 << 16


def test_a_list_of_kept_positions_as_long_as_32_bits_count(device, kernels):
    budget = 2**31 - 1
    pool = torch.randn((12, 2, 1, 16, 8), device=device).bfloat16()
    kept = torch.zeros(budget, dtype=torch.int32, device=device)
    kernels.launch_evict(pool[:, 0], pool[:, 1], torch.rand((12, 1, 16), device=device), i32(np.arange(12)[None], device),
                         None, i32([190], device), None, kept.view(1, 1, budget), budget, 8)
    assert kept[:190].tolist() == list(range(190))
    for part in kept[190:].split(1 << 28):
        assert int(part.min()) == int(part.max()) == -1
