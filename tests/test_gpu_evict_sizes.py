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
