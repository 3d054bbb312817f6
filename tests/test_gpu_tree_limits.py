"""Attention of draft trees of more nodes than they are declared to have."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tree64 import TreeBatch, ancestors, random_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_nodes_past_the_declared_most(device, kernels, dtype, d):
    """Nodes from max_nodes on have no row and are not attended to, whatever the mask says of them."""
    rng = np.random.default_rng(d)
    b = TreeBatch(device, [70, 21, 0], [rng.random((60, 60)) < 0.5, rng.random((9, 9)) < 0.5, rng.random((41, 41)) < 0.5],
                  dtype, heads=4, hkv=1, d=d, seed=d, words=3)
    b.max_nodes = 40
    for s in (0, 2):
        b.sees[s][:, 40:] = False
    out = torch.full_like(b.q, 7.0)
    got = b.run(kernels, out=out)
    rows = np.concatenate([np.arange(c, c + min(n, 40)) for c, n in zip(b.cu, b.nodes)])
    want, tol = b.want()
    over = np.abs(got.float().cpu().numpy() - want) - tol
    assert (over[rows] <= 0).all()
    others = np.setdiff1d(np.arange(len(want)), rows)
    assert (got[torch.as_tensor(others, device=device)] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("prior", [4, 20])
def test_values_that_are_not_finite_in_a_tree_past_the_most(device, kernels, dtype, prior):
    """A tree of 1,100 nodes in a table that ends with it, of which 1,024 are declared: what is not finite reaches the
    nodes that see it and are declared, and no other."""
    rng = np.random.default_rng(prior)
    parents = random_tree(rng, 1100, depth=40)
    b = TreeBatch(device, [30, prior], [random_tree(rng, 5), parents], dtype, heads=2, hkv=1, d=64, seed=prior)
    assert int(b.ctx[1]) % 16 == 0 and b.table.shape[1] * 16 == b.ctx[1]
    b.max_nodes = 1024
    clean = b.run(kernels)
    sick = [5, 21, 300, 1010, 1023, 1030, 1061, 1072, 1080, 1098]
    for j in sick:
        at = prior + j
        b.kc[int(b.table[1, at // 16]), :, at % 16] = float("nan")
        b.vc[int(b.table[1, at // 16]), :, at % 16] = float("inf")
    got = b.run(kernels)
    seen_by = ancestors(parents)[:1024, sick].any(1)
    assert seen_by.any() and not seen_by.all()
    healthy = torch.as_tensor(np.concatenate([np.ones(5, bool), ~seen_by]), device=device)
    assert torch.isfinite(clean[:1029]).all() and torch.equal(got[:1029][healthy], clean[:1029][healthy])
    assert not torch.isfinite(got[:1029][~healthy]).all(-1).any()
    assert torch.isnan(got[1029:]).all()                               # (left as they were)
