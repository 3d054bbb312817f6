"""Gathered scores over tables too wide for the one-launch kernel: the stream-K worker and the finish kernel for
every type, head_dim and ratio of heads that the tiles take."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_scores import Batch

pytestmark = pytest.mark.gpu

RATIOS = [1, 2, 3, 4, 5, 6, 7, 8, 16]
# One launch takes tables of up to 1,024 tokens at the most; these have more.
WIDE = 100


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("g", RATIOS)
def test_every_ratio(device, kernels, dtype, d, g):
    """Lengths of zero and one, block ends and beside them; old scores kept, cut and absent."""
    b = Batch(device, [0, 1, 15, 16, 17, 250, 64, 640], dtype, 2 * g, 2, d, seed=100 * g + d, wide=WIDE)
    b.check(kernels, scored=np.array([0, 0, 7, 16, 16, 100, 70, 639]))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("g", RATIOS)
def test_workers_inside_and_across_segments(device, kernels, dtype, d, g):
    """A long sequence, whose segments are cut between workers, among many short ones, of which a worker
    takes several."""
    rng = np.random.default_rng(g)
    ctx = np.concatenate([rng.integers(1, 60, 150), [6000], rng.integers(1, 60, 150)])
    b = Batch(device, ctx, dtype, g, 1, d, seed=10 * g + d)
    b.check(kernels, scored=rng.integers(0, ctx + 1), first=5)


@pytest.mark.parametrize("g", RATIOS)
@pytest.mark.parametrize("bs", [32, 256])
def test_larger_blocks(device, kernels, g, bs):
    b = Batch(device, [700, 33, 1500, 16], "bf16", g, 1, 64, bs, seed=g + bs, fused=False)
    b.check(kernels, scored=np.array([0, 33, 777, 2]), first=16)
