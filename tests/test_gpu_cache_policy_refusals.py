"""Calls of the shared-prefix, scoring and eviction bindings that are refused before anything is launched, or taken."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from railgun_amd.ops import PagedAttentionOp, RailgunError

pytestmark = pytest.mark.gpu

BS = 16


class Call:
    """Two sequences over a pool of 12 blocks."""

    def __init__(self, device, heads=8, hkv=2, d=64, bs=BS):
        self.pool = torch.zeros((12, 2, hkv, bs, d), dtype=torch.bfloat16, device=device)
        self.kc, self.vc = self.pool[:, 0], self.pool[:, 1]
        self.scores = torch.zeros((12, hkv, bs), device=device)
        self.table = torch.arange(12, dtype=torch.int32, device=device).view(2, 6)
        self.table[:, 0] = 0
        self.lens = torch.tensor([40, 90], dtype=torch.int32, device=device)
        self.q = torch.zeros((2, heads, d), dtype=torch.bfloat16, device=device)
        self.shape = (heads, hkv, d, bs, 6, 2)
        self.ws = torch.empty(1 << 24, dtype=torch.uint8, device=device)

    def op(self, kernels):
        heads, hkv, d, bs, _, _ = self.shape
        return PagedAttentionOp(0.125, heads, hkv, d, bs, kernels)


@pytest.mark.parametrize("blocks", [2**32, 2**32 + 1, -2**32 + 1])
def test_shared_blocks_past_32_bits(device, kernels, blocks):
    c = Call(device)
    with pytest.raises(RailgunError, match="32 bits"):
        kernels.launch_shared_prefix(c.q, c.kc, c.vc, c.table, c.lens, torch.empty_like(c.q), 0.125, *c.shape, blocks,
                                     c.ws)


def test_one_block_expanded(device, kernels):
    """A block stride of 0 stands for dense blocks in the library, which would be read and written past the one."""
    c = Call(device)
    flat = c.scores[:1].expand_as(c.scores)
    k, v = c.kc[:1].expand_as(c.kc), c.vc[:1].expand_as(c.vc)
    out, op = torch.empty_like(c.q), c.op(kernels)
    for call in (lambda: op.execute_with_scores(c.q, c.kc, c.vc, c.table, c.lens, flat),
                 lambda: op.execute_with_scores(c.q, k, v, c.table, c.lens, c.scores),
                 lambda: op.execute_shared_prefix(c.q, k, v, c.table, c.lens, 1),
                 lambda: kernels.launch_v1_scores(c.q, k, v, c.table, c.lens, out, c.scores, None, 0, 0.125, *c.shape, c.ws),
                 lambda: kernels.launch_shared_prefix(c.q, k, v, c.table, c.lens, out, 0.125, *c.shape, 1, c.ws),
                 lambda: kernels.launch_evict(c.kc, c.vc, flat, c.table, None, c.lens, None, None, 32, 4),
                 lambda: kernels.launch_evict(k, v, c.scores, c.table, None, c.lens, None, None, 32, 4)):
        with pytest.raises(RailgunError, match="apart"):
            call()


@pytest.mark.parametrize("scale", [np.float32(0.125), torch.tensor(0.125), 0.125])
def test_scales_that_are_no_python_floats(device, kernels, scale):
    """Taken, as launch_v1 takes them."""
    c = Call(device)
    c.q.normal_()
    c.pool.normal_()
    outs = [torch.empty_like(c.q) for _ in range(4)]
    for out, x in zip(outs, (scale, 0.125)):
        kernels.launch_shared_prefix(c.q, c.kc, c.vc, c.table, c.lens, out, x, *c.shape, 1, c.ws)
    for out, x in zip(outs[2:], (scale, 0.125)):
        kernels.launch_v1_scores(c.q, c.kc, c.vc, c.table, c.lens, out, c.scores, None, BS, x, *c.shape, c.ws)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[3])
