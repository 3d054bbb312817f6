"""Block copies of a pool that has scores: a block's scores go where its K and V go."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from railgun_amd.kv_pool import CpuBlockPool, GpuBlockPool

pytestmark = pytest.mark.gpu


def pool_of(device, hkv, bs, layers=3, blocks=40, dtype=torch.bfloat16, scored=True):
    pool = GpuBlockPool(layers, blocks, hkv, bs, 16, device, dtype=dtype,
                        fill=torch.Generator(device=device).manual_seed(hkv))
    if scored:
        pool.scores.uniform_()
    return pool


@pytest.mark.parametrize("hkv,bs", [(8, 16), (2, 32), (1, 16), (3, 5), (1, 1), (2, 7)])
def test_copy_on_write(device, hkv, bs):
    pool = pool_of(device, hkv, bs, blocks=40, dtype=torch.float32)
    assert pool.scores.shape == (3, 40, hkv, bs)
    want, kv = pool.scores.cpu(), pool.storage.cpu()
    src, dst = [3, 17, 0, 39], [5, 2, 38, 11]
    want[:, dst] = want[:, src]
    kv[:, dst] = kv[:, src]
    pool.copy_blocks(src, dst)
    assert torch.equal(pool.scores.cpu(), want) and torch.equal(pool.storage.cpu(), kv)


@pytest.mark.parametrize("hkv,bs", [(8, 16), (3, 5)])
def test_swapped_out_and_in_elsewhere(device, hkv, bs):
    pool = pool_of(device, hkv, bs)
    host = CpuBlockPool(pool, 10)
    ids, there, back = [7, 30, 1], [0, 9, 4], [2, 33, 39]
    before = pool.scores.cpu()
    pool.swap_out(ids, host, there)
    torch.cuda.synchronize()
    pool.scores[:, ids] = -1.0                      # the blocks' next owners
    pool.swap_in(host, there, back)
    got = pool.scores.cpu()
    assert torch.equal(got[:, back], before[:, ids])
    rest = [i for i in range(40) if i not in ids + back]
    assert torch.equal(got[:, rest], before[:, rest])


def test_swapped_in_by_a_pool_without_scores_yet(device):
    pool, other = pool_of(device, 2, 16), pool_of(device, 2, 16, scored=False)
    host = CpuBlockPool(pool, 4)
    pool.swap_out([5], host, [1])
    other.swap_in(host, [1, 2], [8, 9])             # host block 2 was never scored: zeros
    assert torch.equal(other.scores[:, 8].cpu(), pool.scores[:, 5].cpu())
    assert float(other.scores[:, 9].abs().max()) == 0


def test_no_scores_no_copies_of_them(device):
    pool = pool_of(device, 2, 16, scored=False)
    host = CpuBlockPool(pool, 4)
    pool.copy_blocks([1], [2])
    pool.swap_out([1], host, [0])
    pool.swap_in(host, [0], [3])
    assert pool._scores is None and host.score_rows is None
    assert torch.equal(pool.storage[:, 3].cpu(), pool.storage[:, 1].cpu())


def test_eviction_of_a_pool_whose_score_rows_are_rounded_up(device):
    """15 cells to a block: the rows of the scores are 16 apart, and every cell is found."""
    pool = pool_of(device, 3, 5, layers=2, blocks=20, dtype=torch.float32)
    scores = pool.scores.cpu().numpy()
    table = torch.arange(8, dtype=torch.int32, device=device)[None]
    kept = torch.empty((2, 1, 3, 12), dtype=torch.int32, device=device)
    pool.evict(table, torch.tensor([37], dtype=torch.int32, device=device), 12, 2, 1, None, kept)
    t = np.arange(37)
    for layer in range(2):
        for h in range(3):
            s = scores[layer, t // 5, h, t % 5]
            best = 1 + np.argsort(-s[1:35], kind="stable")[:9]
            np.testing.assert_array_equal(kept[layer, 0, h].cpu().numpy(), np.sort(np.concatenate([[0, 35, 36], best])))
