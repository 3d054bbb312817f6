"""Eviction from the paged cache (rg_evict_cache) against a plain implementation.

The kept positions, the new lengths, K, V and scores are whole values or copies: every comparison
is bit for bit, and the comparisons cover the whole pools, so a cell written that should keep its
contents fails as well.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import TORCH_DT, i32
from railgun_amd.kv_pool import GpuBlockPool
from railgun_amd.ops import RailgunError


def keep_positions(scores, budget, recent, protected):
    """Positions kept of one segment with the given scores [n], in order."""
    n = len(scores)
    if n <= budget:
        return np.arange(n)
    middle = np.arange(protected, n - recent)
    s = scores[middle].astype(np.float64)
    s[np.isnan(s)] = -np.inf
    best = middle[np.argsort(-s, kind="stable")[:budget - protected - recent]]
    return np.sort(np.concatenate([np.arange(protected), best, np.arange(n - recent, n)])).astype(np.int64)


def bits(t):
    return t.contiguous().view(torch.int32 if t.element_size() == 4 else torch.int16).cpu().numpy()


class Case:
    """A pool of `layers` with shuffled blocks, tables for `lens` and destination rows."""

    def __init__(self, device, lens, budget, dtype="bf16", layers=1, hkv=2, bs=16, d=64, dst="apart", shared=0, seed=0,
                 scores=None, wide=0):
        rng = np.random.default_rng(seed)
        self.lens, self.budget, self.bs, self.layers, self.hkv = np.asarray(lens, np.int64), budget, bs, layers, hkv
        b = len(lens)
        need = -(-self.lens // bs)
        kept = -(-np.minimum(self.lens, budget) // bs)
        total = int(need.sum() + kept.sum()) + 3
        order = iter(rng.permutation(total).astype(np.int32))
        mb = max(1, int(need.max()) + wide)
        self.table = np.full((b, mb), -7, np.int32)        # entries past a row's blocks are never read
        prefix = [next(order) for _ in range(shared)]
        for s in range(b):
            for i in range(int(need[s])):
                self.table[s, i] = prefix[i] if i < shared else next(order)
        if dst == "in place":
            self.dst = None
        else:
            self.dst = np.full((b, max(1, int(kept.max()))), -9, np.int32)
            for s in range(b):
                for i in range(int(kept[s])):
                    same = dst == "same blocks" or i < shared or (dst == "mixed" and i % 2 == 0)
                    self.dst[s, i] = self.table[s, i] if same else next(order)
        g = torch.Generator(device=device).manual_seed(seed)
        pool = torch.randn((layers, total, 2, hkv, bs, d), generator=g, device=device).to(TORCH_DT[dtype])
        self.pool = pool
        self.scores = torch.rand((layers, total, hkv, bs), generator=g, device=device) ** 4
        if scores is not None:
            self.scores = scores(self.scores, g)
        self.new_lens = torch.full((b,), -3, device=device, dtype=torch.int32)
        self.kept = torch.full((layers, b, hkv, budget), -3, device=device, dtype=torch.int32)
        self.device = device

    def expected(self, recent, protected):
        pool, scores = bits(self.pool).copy(), bits(self.scores).copy()
        pool0, scores0 = pool.copy(), scores.copy()
        values = self.scores.cpu().numpy()
        kept = np.full(self.kept.shape, -1, np.int32)
        dst = self.table if self.dst is None else self.dst
        for layer in range(self.layers):
            for s, n in enumerate(self.lens):
                t = np.arange(n)
                for h in range(self.hkv):
                    p = keep_positions(values[layer, self.table[s, t // self.bs], h, t % self.bs], self.budget, recent,
                                       protected)
                    kept[layer, s, h, :len(p)] = p
                    j = np.arange(len(p))
                    to, src = dst[s, j // self.bs], self.table[s, p // self.bs]
                    pool[layer, to, :, h, j % self.bs] = pool0[layer, src, :, h, p % self.bs]
                    scores[layer, to, h, j % self.bs] = scores0[layer, src, h, p % self.bs]
        return pool, scores, kept, np.minimum(self.lens, self.budget)

    def run(self, kernels, recent, protected, k=None, v=None, workspace=None, give_kept=True):
        k = self.pool[:, :, 0] if k is None else k
        v = self.pool[:, :, 1] if v is None else v
        kernels.launch_evict(k, v, self.scores, i32(self.table, self.device),
                             None if self.dst is None else i32(self.dst, self.device), i32(self.lens, self.device),
                             self.new_lens, self.kept if give_kept else None, self.budget, recent, protected, workspace)

    def check(self, kernels, recent, protected, **kw):
        pool, scores, kept, lens = self.expected(recent, protected)
        self.run(kernels, recent, protected, **kw)
        torch.cuda.synchronize()
        if kw.get("give_kept", True):
            np.testing.assert_array_equal(self.kept.cpu().numpy(), kept)
        np.testing.assert_array_equal(self.new_lens.cpu().numpy(), lens)
        np.testing.assert_array_equal(bits(self.scores), scores)
        np.testing.assert_array_equal(bits(self.pool), pool)


pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dst", ["apart", "in place", "same blocks", "mixed"])
@pytest.mark.parametrize("budget,recent,protected", [(64, 16, 0), (50, 13, 7), (33, 0, 33), (40, 40, 0), (1, 0, 0),
                                                     (96, 8, 16)])
def test_budgets(device, kernels, dst, budget, recent, protected):
    c = Case(device, [0, 1, 17, 63, 64, 65, 100, 333], budget, dst=dst, seed=budget)
    c.check(kernels, recent, protected)


@pytest.mark.parametrize("dtype,hkv,bs,d", [("f32", 8, 16, 64), ("f16", 4, 32, 128), ("bf16", 1, 16, 256),
                                            ("bf16", 3, 8, 80), ("f16", 2, 5, 20), ("f32", 2, 1, 3), ("bf16", 2, 64, 1)])
@pytest.mark.parametrize("dst", ["apart", "in place"])
def test_shapes(device, kernels, dtype, hkv, bs, d, dst):
    c = Case(device, [200, 31, 90], 48, dtype=dtype, layers=2, hkv=hkv, bs=bs, d=d, dst=dst, seed=d)
    c.check(kernels, 10, 3)


@pytest.mark.parametrize("dtype,d", [("bf16", 8), ("f32", 4), ("f16", 1), ("bf16", 2)])
@pytest.mark.parametrize("dst", ["apart", "in place"])
def test_many_short_rows(device, kernels, dtype, d, dst):
    """Rows of one piece of the move: its workgroups take no more tokens than they have threads."""
    Case(device, [3000, 1200], 1100, dtype=dtype, d=d, dst=dst, seed=d).check(kernels, 40, 20)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 128)])
@pytest.mark.parametrize("dst", ["apart", "in place", "mixed"])
@pytest.mark.parametrize("lens,budget", [([1000, 640, 30], 600), ([3900, 1300, 999], 1200)])
def test_few_large_segments(device, kernels, dtype, d, dst, lens, budget):
    """Selection and move as two launches."""
    Case(device, lens, budget, dtype=dtype, d=d, dst=dst, seed=d).check(kernels, 77, 35)


@pytest.mark.parametrize("dst", ["apart", "in place", "mixed"])
def test_many_segments(device, kernels, dst):
    """More than four segments a CU, of several chunks each: one workgroup a segment."""
    lens = np.random.default_rng(1).integers(1, 700, 18)
    Case(device, lens, 300, layers=15, hkv=4, d=128, dst=dst).check(kernels, 50, 17)


def test_layers_and_shared_prefix(device, kernels):
    """Sequences that share their first blocks, protected: the shared blocks stay as they are."""
    c = Case(device, [700, 128, 90, 401], 128, layers=5, hkv=4, shared=2, seed=5)
    c.check(kernels, 31, 32)


@pytest.mark.parametrize("lens,budget", [([5000, 4097, 2500], 1024), ([40000], 9001), ([33000, 20], 32800)])
@pytest.mark.parametrize("dst", ["apart", "in place"])
def test_long(device, kernels, lens, budget, dst):
    """Tables past one strip of candidates, and past what LDS holds."""
    c = Case(device, lens, budget, hkv=2, d=64, dst=dst, seed=lens[0])
    c.check(kernels, 100, 16)


@pytest.mark.parametrize("bs,protected,recent", [(24, 5, 1), (6, 7, 33), (4, 1, 0), (2, 3, 2), (32, 30, 99)])
@pytest.mark.parametrize("lens", [[700, 90, 91], [3000, 41], [13001], [30000], [70001]])
def test_candidates_that_begin_anywhere(device, kernels, bs, protected, recent, lens):
    """First and last candidates inside a group of four, blocks that hold whole groups and blocks that do not, in
    each of the selection's forms."""
    c = Case(device, lens, max(40 + recent, lens[0] // 7), hkv=1, bs=bs, d=4, seed=lens[0] + bs)
    c.check(kernels, recent, protected)


@pytest.mark.parametrize("n", [500, 40000])
def test_scores_off_16_bytes(device, kernels, n):
    c = Case(device, [n], n // 3, d=8, seed=n)
    room = torch.zeros(c.scores.numel() + 1, device=device)
    room[1:] = c.scores.flatten()
    c.scores = room[1:].view(c.scores.shape)
    c.check(kernels, 9, 6)


@pytest.mark.parametrize("n", [900, 3900, 16000, 60000, 80000])
@pytest.mark.parametrize("values", [2, 40])
def test_few_distinct_scores(device, kernels, n, values):
    """Ties at the threshold, more of them than the later passes list."""
    c = Case(device, [n], n // 4, hkv=1, d=4, seed=n, scores=lambda s, g: torch.ceil(s * values))
    c.check(kernels, 20, 3)


def test_wide_table_of_short_contexts(device, kernels):
    c = Case(device, [70, 3, 200], 64, seed=11, wide=3000)
    c.check(kernels, 5, 0)


def special(s, g):
    """Scores with ties, zeros of both signs, infinities and NaN."""
    r = torch.rand(s.shape, generator=g, device=s.device)
    s = (s * 8).round() / 8
    s = torch.where(r < 0.10, torch.full_like(s, -0.0), s)
    s = torch.where((r >= 0.10) & (r < 0.15), torch.full_like(s, float("nan")), s)
    s = torch.where((r >= 0.15) & (r < 0.20), torch.full_like(s, -float("nan")), s)
    s = torch.where((r >= 0.20) & (r < 0.25), torch.full_like(s, float("inf")), s)
    s = torch.where((r >= 0.25) & (r < 0.30), torch.full_like(s, -float("inf")), s)
    s = torch.where((r >= 0.30) & (r < 0.35), -s, s)
    return torch.where((r >= 0.35) & (r < 0.40), torch.full_like(s, 1e-42), s)


@pytest.mark.parametrize("budget", [40, 200, 330, 480])
def test_special_scores(device, kernels, budget):
    c = Case(device, [500, 499], budget, hkv=3, scores=special, seed=budget)
    c.check(kernels, 9, 2)


@pytest.mark.parametrize("value", [0.0, 1.0, float("nan")])
def test_equal_scores_keep_the_lowest_positions(device, kernels, value):
    c = Case(device, [3000], 777, scores=lambda s, g: torch.full_like(s, value), seed=1)
    c.check(kernels, 10, 0)


def test_without_kept_and_with_a_kept_workspace(device, kernels):
    c = Case(device, [300, 100], 64, seed=3)
    ws = torch.full((kernels.evict_workspace_bytes(1, 2, 2, 64),), 255, dtype=torch.uint8, device=device)
    c.check(kernels, 5, 0, give_kept=False, workspace=ws)
    c = Case(device, [300, 100], 64, seed=4)
    c.check(kernels, 5, 0, give_kept=False)
    c = Case(device, [300, 100], 64, seed=4)
    c.new_lens = None
    c.run(kernels, 5, 0)


def test_unaligned_rows_move_in_small_pieces(device, kernels):
    """Caches whose base is not 16-byte aligned."""
    c = Case(device, [200, 64], 32, seed=8, d=64)
    flat = torch.zeros(c.pool.numel() + 1, dtype=c.pool.dtype, device=device)
    moved = flat[1:].view(c.pool.shape)
    moved.copy_(c.pool)
    c.pool = moved
    c.check(kernels, 4, 0)


def test_one_layer_cache_and_separate_pools(device, kernels):
    """[NB, H_kv, bs, D] caches that are two tensors, as a caller without layers holds them."""
    c = Case(device, [150, 90], 60, seed=9)
    pool, scores, kept, lens = c.expected(7, 0)
    k, v = c.pool[0, :, 0].contiguous(), c.pool[0, :, 1].contiguous()
    kernels.launch_evict(k, v, c.scores[0], i32(c.table, device), i32(c.dst, device), i32(c.lens, device), c.new_lens,
                         c.kept, 60, 7)
    np.testing.assert_array_equal(bits(k), pool[0, :, 0])
    np.testing.assert_array_equal(bits(v), pool[0, :, 1])
    np.testing.assert_array_equal(bits(c.scores), scores)


def test_replayed_graph(device, kernels):
    """Captured once, replayed on other contents; eager work between the replays."""
    c = Case(device, [400, 100, 250], 96, layers=2, seed=20)
    start, start_scores = c.pool.clone(), c.scores.clone()
    ws = torch.empty(kernels.evict_workspace_bytes(2, 3, 2, 96), dtype=torch.uint8, device=device)
    args = (i32(c.table, device), i32(c.dst, device), i32(c.lens, device))

    def step():
        kernels.launch_evict(c.pool[:, :, 0], c.pool[:, :, 1], c.scores, *args, c.new_lens, c.kept, 96, 20, 0, ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for seed in range(3):
        c.pool.copy_(start + seed)
        c.scores.copy_(start_scores.roll(seed, 1))
        pool, scores, kept, _ = c.expected(20, 0)
        g.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(c.kept.cpu().numpy(), kept)
        np.testing.assert_array_equal(bits(c.pool), pool)
        np.testing.assert_array_equal(bits(c.scores), scores)


def test_another_stream(device, kernels):
    c = Case(device, [400, 100], 96, seed=21)
    want = c.expected(20, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run(kernels, 20, 0)
    side.synchronize()
    np.testing.assert_array_equal(bits(c.pool), want[0])


def test_pool_far_past_32_bits(device, kernels):
    """Block offsets past 2^32 elements."""
    bs, d, hkv = 16, 64, 2
    stride = 2 * hkv * bs * d
    blocks = (1 << 32) // stride + 40
    pool = torch.zeros((1, blocks, 2, hkv, bs, d), dtype=torch.bfloat16, device=device)
    scores = torch.rand((1, blocks, hkv, bs), device=device)
    table = np.arange(blocks - 20, blocks, dtype=np.int32)[None]
    dst = np.arange(3, 8, dtype=np.int32)[None]
    pool[0, blocks - 20:].normal_()
    n, budget = 20 * bs - 3, 5 * bs
    t = np.arange(n)
    values = scores[0, blocks - 20:].cpu().numpy()
    kernels.launch_evict(pool[:, :, 0], pool[:, :, 1], scores, i32(table, device), i32(dst, device),
                         i32([n], device), None, None, budget, 8)
    src = bits(pool[0, blocks - 20:])
    got = bits(pool[0, 3:8])
    for h in range(hkv):
        p = keep_positions(values[t // bs, h, t % bs], budget, 8, 0)
        j = np.arange(budget)
        np.testing.assert_array_equal(got[j // bs, :, h, j % bs], src[p // bs, :, h, p % bs])


def test_refusals_of_the_binding(device, kernels):
    c = Case(device, [100], 32, seed=2)
    table, lens = i32(c.table, device), i32(c.lens, device)
    k, v = c.pool[:, :, 0], c.pool[:, :, 1]
    ok = dict(key_cache=k, value_cache=v, scores=c.scores, block_table=table, dst_block_table=None, context_lens=lens,
              new_context_lens=None, kept_positions=None, budget=32, recent=4)
    for change in (dict(scores=c.scores.double()), dict(scores=c.scores[:, :-1]), dict(value_cache=v.float()),
                   dict(block_table=table.long()), dict(block_table=table[0]), dict(budget=0), dict(recent=33),
                   dict(protected_len=29), dict(dst_block_table=table[:, :1].contiguous()),
                   dict(kept_positions=c.kept[..., :-1].contiguous()), dict(new_context_lens=lens.repeat(2)),
                   dict(key_cache=k.transpose(2, 3), value_cache=v.transpose(2, 3)),
                   dict(workspace=torch.empty(4, dtype=torch.uint8, device=device))):
        with pytest.raises(RailgunError):
            kernels.launch_evict(**{**ok, **change})
    with pytest.raises(RailgunError):
        kernels.launch_evict(**{**ok, "scores": c.scores.cpu()})


@pytest.mark.parametrize("name", ["budget", "recent", "protected_len"])
def test_counts_past_32_bits(device, name):
    pool = GpuBlockPool(1, 4, 2, 16, 64, device)
    counts = dict(budget=20, recent=4, protected_len=4)
    counts[name] += 2**32
    with pytest.raises(RailgunError, match="32 bits"):
        pool.evict(i32(np.arange(4).reshape(1, 4), device), i32([60], device), **counts)


def test_new_lengths_over_the_old_ones(device, kernels):
    c = Case(device, [90, 40], 32, seed=2)
    before = c.pool.clone()
    lens = i32(c.lens, device)
    with pytest.raises(RailgunError, match="overlaps"):
        kernels.launch_evict(c.pool[:, :, 0], c.pool[:, :, 1], c.scores, i32(c.table, device), i32(c.dst, device), lens,
                             lens, c.kept, 32, 4, 0)
    assert torch.equal(c.pool, before)


def test_pool_evicts_every_layer(device):
    """GpuBlockPool.evict: the pool's own storage and scores."""
    pool = GpuBlockPool(3, 40, 2, 16, 64, device, fill=torch.Generator(device=device).manual_seed(1))
    pool.scores.uniform_()
    table = np.arange(20, dtype=np.int32).reshape(2, 10)
    before, scores = bits(pool.storage), pool.scores.cpu().numpy()
    new_lens = pool.evict(i32(table, device), i32([150, 30], device), budget=48, recent=16)
    assert new_lens.tolist() == [48, 30]
    after = bits(pool.storage)
    t = np.arange(150)
    for layer in range(3):
        for h in range(2):
            p = keep_positions(scores[layer, table[0, t // 16], h, t % 16], 48, 16, 0)
            j = np.arange(48)
            np.testing.assert_array_equal(after[layer, table[0, j // 16], :, h, j % 16],
                                          before[layer, table[0, p // 16], :, h, p % 16])
    np.testing.assert_array_equal(after[:, 10:], before[:, 10:])
