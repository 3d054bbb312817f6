"""Decode attention that gathers attention weights (rg_paged_attention_v1_scores) against 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from attention64 import HALF_STEP, assert_within, attention64
from helpers import TORCH_DT, dev_f32, i32
from railgun_amd.ops import PagedAttentionOp, RailgunError

pytestmark = pytest.mark.gpu


class Batch:
    """A decode batch over a fused pool with shuffled blocks; cells no sequence uses hold NaN."""

    def __init__(self, device, ctx, dtype="bf16", heads=8, hkv=2, d=64, bs=16, seed=0, wide=0, fused=True):
        rng = np.random.default_rng(seed)
        self.ctx, self.dtype, self.device = np.asarray(ctx, np.int64), dtype, device
        need = -(-np.maximum(self.ctx, 0) // bs)
        b, total = len(ctx), int(need.sum()) + 3
        order = iter(rng.permutation(total))
        self.table = np.zeros((b, max(1, int(need.max()) + wide)), np.int32)
        for s in range(b):
            for i in range(int(need[s])):
                self.table[s, i] = next(order)
        g = torch.Generator(device=device).manual_seed(seed)
        dt = TORCH_DT[dtype]
        pool = torch.full((total, 2, hkv, bs, d), float("nan"), device=device, dtype=dt)
        used = torch.zeros((total, bs), dtype=torch.bool, device=device)
        for s in range(b):
            t = np.arange(max(int(self.ctx[s]), 0))
            used[torch.as_tensor(self.table[s, t // bs].astype(np.int64), device=device),
                 torch.as_tensor(t % bs, device=device)] = True
        fresh = torch.randn(pool.shape, generator=g, device=device).to(dt)
        self.pool = torch.where(used[:, None, None, :, None], fresh, pool)
        self.kc, self.vc = self.pool[:, 0], self.pool[:, 1]
        if not fused:
            self.kc, self.vc = self.kc.contiguous(), self.vc.contiguous()
        self.q = (2 * torch.randn((b, heads, d), generator=g, device=device)).to(dt)
        self.scores = torch.rand((total, hkv, bs), generator=g, device=device) * 3
        self.used = used
        self.hkv, self.bs, self.scale = hkv, bs, 1.0 / math.sqrt(d)
        self.heads, self.d = heads, d

    def op(self, kernels):
        return PagedAttentionOp(self.scale, self.heads, self.hkv, self.d, self.bs, kernels)

    def check(self, kernels, scored=None, first=0, workspace=None, lens=None):
        before = self.scores.clone()
        lens = self.ctx if lens is None else lens
        out = self.op(kernels).execute_with_scores(self.q, self.kc, self.vc, i32(self.table, self.device),
                                                   i32(lens, self.device), self.scores,
                                                   None if scored is None else i32(scored, self.device), first, workspace)
        self.verify(out, before, scored, first)

    def verify(self, out, before, scored, first):
        want, tol, weights, wtol = attention64(self.q, self.kc, self.vc, self.table, self.ctx, self.scale, self.dtype)
        assert_within(dev_f32(out), want, tol, "out")
        old = before.cpu().numpy().astype(np.float64)
        new, ntol = old.copy(), np.zeros_like(old)
        for s, n in enumerate(self.ctx):
            t = np.arange(first, max(int(n), first))
            blk, off = self.table[s, t // self.bs], t % self.bs
            keep = np.ones(len(t), bool) if scored is None else t < scored[s]
            new[blk, :, off] = np.where(keep[:, None], old[blk, :, off], 0) + weights[s].T[t]
            ntol[blk, :, off] = wtol[s].T[t] + HALF_STEP["f32"] * new[blk, :, off] + 1e-37
        got = self.scores.cpu().numpy()
        assert_within(got, new, ntol, "scores")
        untouched = ntol == 0
        np.testing.assert_array_equal(got[untouched], before.cpu().numpy()[untouched])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,hkv,d", [(4, 4, 64), (8, 4, 128), (6, 2, 64), (8, 2, 128), (10, 2, 64), (12, 2, 128),
                                         (14, 2, 128), (16, 2, 64), (32, 2, 128), (8, 2, 256), (2, 2, 256)])
def test_tiles(device, kernels, dtype, heads, hkv, d):
    """Every ratio of heads that the tiles take; lengths of zero and one, block ends and beside them."""
    b = Batch(device, [0, 1, 15, 16, 17, 250, 64], dtype, heads, hkv, d, seed=heads * d)
    b.check(kernels, scored=np.array([0, 0, 7, 16, 16, 100, 70]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,hkv,d,bs", [(4, 2, 80, 16), (6, 3, 20, 8), (2, 2, 4, 5), (18, 2, 64, 16), (9, 1, 128, 16),
                                            (4, 2, 128, 1), (6, 2, 256, 16), (4, 2, 64, 512)])
def test_other_shapes(device, kernels, dtype, heads, hkv, d, bs):
    b = Batch(device, [300, 0, 1, 77, 513], dtype, heads, hkv, d, bs, seed=d + bs)
    b.check(kernels, scored=np.array([299, 0, 0, 0, 256]), first=3)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("fused", [True, False])
def test_block_sizes(device, kernels, bs, fused):
    b = Batch(device, [700, 33, 1025], "bf16", bs=bs, fused=fused, seed=bs)
    b.check(kernels)


@pytest.mark.parametrize("ctx", [[70, 33], [2000, 900]])
@pytest.mark.parametrize("d", [64, 96])
def test_nothing_scored(device, kernels, ctx, d):
    """first_scored at and past the table's end, up to the largest: the output alone."""
    c = Batch(device, ctx, d=d, seed=d)
    before = c.scores.clone()
    for first in (max(ctx), 2048, 2**31 - 300, 2**31 - 1):
        c.check(kernels, first=first)
        assert torch.equal(c.scores, before)


@pytest.mark.parametrize("scale", [0.0, -0.4, 3.0])
@pytest.mark.parametrize("ctx", [[70, 33], [2000, 900]])
def test_scales(device, kernels, scale, ctx):
    c = Batch(device, ctx, seed=9)
    c.scale = scale
    c.check(kernels, scored=[20, 900])


@pytest.mark.parametrize("first", [0, 1, 16, 100, 299, 300, 5000])
def test_first_scored(device, kernels, first):
    Batch(device, [300, 120, 7], seed=first).check(kernels, scored=np.array([0, 120, 3]), first=first)


@pytest.mark.parametrize("ctx", [[9000], [5000, 1, 2600, 40], [1100] * 40])
def test_long_and_many(device, kernels, ctx):
    Batch(device, ctx, heads=16, hkv=4, d=128, seed=len(ctx)).check(kernels, scored=np.array(ctx) - 1)


def test_table_much_wider_than_the_contexts(device, kernels):
    Batch(device, [40, 700], wide=2000, seed=4).check(kernels)


def test_all_rows_empty(device, kernels):
    b = Batch(device, [0, 0, 0], seed=5)
    b.check(kernels)


def test_negative_length_counts_as_none(device, kernels):
    b = Batch(device, [0, 40], seed=6)
    b.check(kernels, lens=np.array([-7, 40]))


def test_large_scores_in_a_row(device, kernels):
    """One key that takes all the weight, others that get weights below the normal numbers."""
    b = Batch(device, [100], "f32", seed=7)
    b.kc[int(b.table[0, 0]), :, 3] *= 30
    b.check(kernels)


def test_two_calls_add_up(device, kernels):
    b = Batch(device, [90, 200], seed=8)
    b.check(kernels, scored=np.array([0, 0]))
    b.check(kernels)


def test_replayed_graph(device, kernels):
    """Captured once and replayed on other contents, with eager calls on the same stream between."""
    b = Batch(device, [400, 90, 0, 33], heads=16, hkv=4, d=128, seed=9)
    op, table, lens = b.op(kernels), i32(b.table, device), i32(b.ctx, device)
    scored = np.array([100, 0, 0, 33])
    scored_dev = i32(scored, device)
    ws = torch.empty(kernels.v1_scores_workspace_bytes(4, 16, 4, 128, 16, b.table.shape[1]), dtype=torch.uint8,
                     device=device)

    def step():
        return op.execute_with_scores(b.q, b.kc, b.vc, table, lens, b.scores, scored_dev, 5, ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        b.q.copy_(torch.randn_like(b.q))
        before = b.scores.clone()
        graph.replay()
        torch.cuda.synchronize()
        b.verify(out, before, scored, 5)
        step()


def test_workspace_contents_do_not_matter(device, kernels):
    b = Batch(device, [130, 500], seed=10)
    n = kernels.v1_scores_workspace_bytes(2, 8, 2, 64, 16, b.table.shape[1])
    b.check(kernels, workspace=torch.full((n,), 255, dtype=torch.uint8, device=device))


def test_pool_far_past_32_bits(device, kernels):
    """Block offsets past 2^32 elements, in the caches and (by a block stride) in the scores."""
    bs, d, hkv = 16, 64, 2
    blocks = (1 << 32) // (2 * hkv * bs * d) + 40
    pool = torch.zeros((blocks, 2, hkv, bs, d), dtype=torch.bfloat16, device=device)
    pool[blocks - 20:].normal_()
    wide = torch.zeros((blocks, 8192), device=device)  # 2^32 cells and more
    scores = wide[:, :hkv * bs].view(blocks, hkv, bs)
    b = Batch(device, [310], "bf16", seed=11)
    b.pool, b.kc, b.vc, b.scores = pool, pool[:, 0], pool[:, 1], scores
    b.table = np.arange(blocks - 20, blocks, dtype=np.int32)[None]
    before = scores[blocks - 20:].clone()
    out = b.op(kernels).execute_with_scores(b.q, b.kc, b.vc, i32(b.table, device), i32(b.ctx, device), scores)
    want, tol, weights, wtol = attention64(b.q, b.kc, b.vc, b.table, b.ctx, b.scale, "bf16")
    assert_within(dev_f32(out), want, tol)
    t = np.arange(310)
    got = scores[blocks - 20:].cpu().numpy()[t // bs, :, t % bs]
    assert_within(got, weights[0].T, wtol[0].T + 2 * HALF_STEP["f32"] * weights[0].T + 1e-37)
    assert float(before.abs().max()) == 0 and float(wide[:, hkv * bs:].abs().max()) == 0


def test_first_scored_past_32_bits(device, kernels):
    c = Batch(device, [70, 33], seed=3)
    with pytest.raises(RailgunError, match="32 bits"):
        c.op(kernels).execute_with_scores(c.q, c.kc, c.vc, i32(c.table, device), i32(c.ctx, device), c.scores,
                                          first_scored=2**32)


def test_refusals(device, kernels):
    b = Batch(device, [40, 30], seed=12)
    op, table, lens = b.op(kernels), i32(b.table, device), i32(b.ctx, device)
    good = dict(q=b.q, k_cache=b.kc, v_cache=b.vc, block_table=table, context_lens=lens, scores=b.scores)
    for change in (dict(scores=b.scores.double()), dict(scores=b.scores[:-1]), dict(scores=b.scores.transpose(1, 2)),
                   dict(scored_lens=lens.long()), dict(scored_lens=lens[:1]), dict(first_scored=-1), dict(q=b.q[0]),
                   dict(q=b.q.float()), dict(q=b.q[..., :32].contiguous()), dict(q=b.q[:1]), dict(block_table=table[:1]),
                   dict(q=b.q.transpose(0, 1)), dict(context_lens=lens[:1]), dict(scores=b.scores.cpu()),
                   dict(workspace=torch.empty(16, dtype=torch.uint8, device=device))):
        with pytest.raises(RailgunError):
            op.execute_with_scores(**{**good, **change})


def test_workers_with_more_tokens_than_they_gather_at_once(device, kernels):
    """16 heads to a kv-head at head_dim 64: a worker gathers the raw scores of 512 tokens, and has 586."""
    Batch(device, [150000], heads=64, hkv=4, d=64, seed=15).check(kernels, scored=np.array([149000]))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,hkv,d", [(4, 4, 64), (8, 4, 128), (6, 2, 64), (8, 2, 128), (10, 2, 64), (12, 2, 128),
                                         (14, 2, 128), (16, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("first", [0, 70])
def test_short_tables(device, kernels, dtype, heads, hkv, d, first):
    """Tables that one launch takes (and, fp32 with 8 heads of 128, the one it does not)."""
    b = Batch(device, [150, 0, 1, 16, 17, 129, 128], dtype, heads, hkv, d, bs=32 if d == 64 else 16, seed=heads + d)
    b.check(kernels, scored=np.array([149, 0, 0, 3, 17, 0, 500]), first=first)


def test_widest_short_tables(device, kernels):
    Batch(device, [890, 3, 512, 513], "bf16", 16, 2, 64, seed=16).check(kernels, scored=np.array([300, 0, 512, 9]))
