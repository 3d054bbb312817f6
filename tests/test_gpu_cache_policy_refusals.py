"""Calls of the shared-prefix, scoring and eviction bindings that are refused before anything is launched."""
from __future__ import annotations

import pytest
import torch

from railgun_amd.ops import PagedAttentionOp, RailgunError

pytestmark = pytest.mark.gpu


class Call:
    """Two sequences over a pool of 12 blocks."""

    def __init__(self, device, heads=8, hkv=2, d=64, bs=16):
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
