"""The shared-prefix decode for every type, head_dim and ratio of heads of its product; the same bits from every
call of it and of the scored decode, whatever the workspace held."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import i32
from test_gpu_scores import Batch as Scored
from test_gpu_shared_prefix import Batch

pytestmark = pytest.mark.gpu

RATIOS = [1, 2, 3, 4, 5, 6, 7, 8, 16]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("g", RATIOS)
def test_every_ratio(device, kernels, dtype, d, g):
    """Rows of no token, of part of the prefix, of all of it and nothing else, and of a worker's several units."""
    ctx = [160 + 30, 0, 1, 160, 159, 161, 160 + 900, 33] + [160 + 7 * i for i in range(20)]
    Batch(device, ctx, 10, dtype, 2 * g, 2, d, seed=100 * g + d).check(kernels)


def garbage(n, device, i):
    return torch.randint(0, 256, (n,), dtype=torch.uint8, device=device,
                         generator=torch.Generator(device=device).manual_seed(i))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("ctx,shared,g", [([700, 330, 1000, 321] * 4, 20, 4), ([2100 + 31 * i for i in range(37)], 128, 7)])
def test_shared_prefix_repeats_itself(device, kernels, dtype, ctx, shared, g):
    b = Batch(device, ctx, shared, dtype, 2 * g, 2, 128, seed=g)
    n = kernels.shared_prefix_workspace_bytes(len(ctx), 2 * g, 2, 128, 16, b.table.shape[1], shared)
    outs = [b.run(kernels, workspace=garbage(n, device, i)) for i in range(8)]
    b.verify(outs[0])
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("ctx,g", [([9000, 40, 2600, 1], 4), ([300 + 100 * i for i in range(16)], 7), ([90, 33], 4)])
def test_scores_repeat_themselves(device, kernels, dtype, ctx, g):
    b = Scored(device, ctx, dtype, 2 * g, 2, 128, seed=g)
    n = kernels.v1_scores_workspace_bytes(len(ctx), 2 * g, 2, 128, 16, b.table.shape[1])
    table, lens, scored = i32(b.table, device), i32(b.ctx, device), i32(np.asarray(ctx) // 2, device)
    start, got = b.scores.clone(), []
    for i in range(8):
        b.scores.copy_(start)
        out = b.op(kernels).execute_with_scores(b.q, b.kc, b.vc, table, lens, b.scores, scored, 3,
                                                garbage(n, device, i))
        got.append((out, b.scores.clone()))
    for out, scores in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(scores, got[0][1])
