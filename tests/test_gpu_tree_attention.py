"""Attention of trees of drafted tokens (rg_paged_attention_tree) against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import i32
from railgun_amd.ops import PagedAttentionOp, RailgunError
from tree64 import TreeBatch, ancestors, random_tree

pytestmark = pytest.mark.gpu


def trees(rng, sizes, **kw):
    return [random_tree(rng, n, **kw) for n in sizes]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,hkv,d", [(4, 4, 64), (8, 4, 128), (6, 2, 64), (8, 2, 128), (10, 2, 64), (12, 2, 128),
                                         (14, 2, 128), (16, 2, 64), (32, 2, 128), (18, 2, 64), (40, 2, 64)])
def test_heads(device, kernels, dtype, heads, hkv, d):
    """Every ratio of heads; no tree, a root alone, nothing before the tree, edges of tiles and blocks."""
    rng = np.random.default_rng(heads * d)
    sizes = [5, 0, 1, 7, 12, 16, 33, 3]
    TreeBatch(device, [70, 0, 0, 0, 31, 32, 33, 300], trees(rng, sizes), dtype, heads, hkv, d, seed=heads + d,
              fused=d == 64).check(kernels)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,hkv,d,bs", [(4, 2, 80, 16), (6, 3, 20, 8), (2, 2, 4, 5), (4, 1, 128, 1), (4, 2, 64, 512),
                                            (4, 2, 256, 16), (3, 3, 252, 3), (4, 2, 64, 24)])
def test_other_shapes(device, kernels, dtype, heads, hkv, d, bs):
    rng = np.random.default_rng(d + bs)
    TreeBatch(device, [40, 0, 0, 1, 123], trees(rng, [9, 3, 0, 1, 34]), dtype, heads, hkv, d, bs,
              seed=d + bs).check(kernels)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_block_sizes(device, kernels, bs):
    rng = np.random.default_rng(bs)
    TreeBatch(device, [2 * bs - 1, bs, 3 * bs + 7, 0, 5 * bs - 9], trees(rng, [20, 4, 1, 2 * bs // 3, 9]), bs=bs,
              fused=bs != 64, seed=bs).check(kernels)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("nodes", [1, 2, 8, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
def test_tree_sizes(device, kernels, nodes, dtype):
    """Row tiles and mask words, their edges; where the tree begins inside a key tile and where it does not."""
    rng = np.random.default_rng(nodes)
    TreeBatch(device, [45, 64, 0], trees(rng, [nodes, max(1, nodes // 3), nodes]), dtype, heads=4, hkv=1,
              seed=nodes).check(kernels)


@pytest.mark.parametrize("d", [64, 128])
def test_largest_tree(device, kernels, d):
    rng = np.random.default_rng(d)
    TreeBatch(device, [77], [random_tree(rng, 1024, depth=40)], heads=2, hkv=1, d=d, seed=d).check(kernels)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("prior,nodes,batch", [(5000, 20, 1), (2500, 6, 3), (1024, 70, 5), (9000, 3, 2)])
def test_long_contexts(device, kernels, dtype, prior, nodes, batch):
    """Sequences split over many workgroups; a sequence of one token among long ones."""
    rng = np.random.default_rng(prior)
    TreeBatch(device, [prior + 13 * i for i in range(batch)] + [0], trees(rng, [nodes] * batch + [1]), dtype, heads=8,
              hkv=2, d=128, seed=prior).check(kernels)


@pytest.mark.parametrize("batch", [1, 2, 17, 65, 200, 300])
def test_batches(device, kernels, batch):
    """Ragged: long, short, padded and single rows, more sequences than a workgroup has threads."""
    rng = np.random.default_rng(batch)
    sizes = rng.integers(0, 12, batch)
    sizes[0] = 5
    prior = np.where(sizes > 0, rng.integers(0, 200, batch), 0)
    prior[0] = 900
    TreeBatch(device, prior, trees(rng, sizes), heads=4, hkv=2, seed=batch, wide=3).check(kernels)


@pytest.mark.parametrize("long,short,d", [(32, 38, 128), (48, 64, 64), (20, 75, 128)])
def test_segments_near_a_round(device, kernels, long, short, d):
    """Segments that are nearly as many as the workgroups that are at work together, some of them cut: more pieces
    than those."""
    rng = np.random.default_rng(long)
    prior = rng.permutation([20 * 32 - 3] * long + [12 * 32 - 3] * short)
    TreeBatch(device, prior, trees(rng, [3] * (long + short)), heads=8, hkv=8, d=d, seed=long).check(kernels)


@pytest.mark.parametrize("dtype,hkv,d,prior", [("bf16", 4, 128, [6000, 5500, 100, 6100]), ("f16", 8, 128, [27000]),
                                               ("f32", 2, 64, [5000, 4990]), ("f32", 2, 64, [9000, 8900]),
                                               ("bf16", 4, 64, [6000, 5500, 100, 6100])])
def test_few_segments(device, kernels, dtype, hkv, d, prior):
    """Few segments, cut into as many pieces as the chip has CUs and into more."""
    rng = np.random.default_rng(len(prior) + d)
    TreeBatch(device, prior, trees(rng, [3, 9, 1, 5][:len(prior)]), dtype, heads=2 * hkv, hkv=hkv, d=d,
              seed=len(prior) + d).check(kernels)


@pytest.mark.parametrize("d,nodes", [(64, 3), (128, 35)])
def test_parts_of_a_segment(device, kernels, d, nodes):
    """Segments in one to 66 parts, a key tile each, of one row tile and of two."""
    rng = np.random.default_rng(d)
    tiles = rng.permutation([1, 2, 3, 4, 5, 8, 9, 28, 29, 31, 32, 33, 36, 37, 64, 65] if nodes == 3 else [2, 3, 30, 33, 65])
    TreeBatch(device, 32 * tiles - 5, trees(rng, [nodes] * len(tiles)), "f32", heads=4, hkv=1, d=d, seed=d).check(kernels)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_any_mask(device, kernels, dtype):
    """Masks that are no tree's: dense, empty rows (zeros where nothing lies before), later nodes seen, oneself
    not; bits of nodes that are not there are not looked at."""
    rng = np.random.default_rng(5)
    masks = [rng.random((n, n)) < share for n, share in ((40, 0.5), (70, 0.05), (33, 0.0), (20, 1.0), (9, 0.3))]
    masks[1][3] = False
    b = TreeBatch(device, [0, 0, 0, 50, 64], masks, dtype, heads=6, hkv=2, seed=6, words=5)
    for s, n in enumerate(b.nodes):
        words = b.mask[b.cu[s]:b.cu[s + 1]].view(np.uint32)
        for i in range(int(n), 160):
            words[:, i // 32] |= np.uint32(1 << (i % 32))
    b.check(kernels)
    out = b.run(kernels)
    assert not out[b.cu[1] + 3].any() and not out[b.cu[2]:b.cu[3]].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_other_branches_do_not_matter(device, kernels, dtype, bad, d):
    """A node whose K and V are not finite reaches the nodes that see it, and no other."""
    rng = np.random.default_rng(d)
    parents = random_tree(rng, 50, depth=4)
    b = TreeBatch(device, [37, 0], [parents, random_tree(rng, 12)], dtype, d=d, seed=8)
    clean = b.run(kernels)
    sick = [21, 40, 44]
    seen_by = ancestors(parents)[:, sick].any(1)
    assert seen_by.any() and not seen_by.all()
    for j in sick:
        at = 37 + j
        b.kc[int(b.table[0, at // 16]), :, at % 16] = bad
        b.vc[int(b.table[0, at // 16]), :, at % 16, 3:] = bad
    got = b.run(kernels)
    healthy = torch.as_tensor(np.concatenate([~seen_by, np.ones(12, bool)]), device=device)
    # (The same sums, in the same order: to the bit.)
    assert torch.equal(got[healthy], clean[healthy])
    if bad != -float("inf"):
        assert not torch.isfinite(got[~healthy]).all(-1).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_values_that_are_not_finite_are_passed_on(device, kernels, dtype):
    """An infinite value of an ordinary key comes out as it does of a sum, in its dim alone."""
    b = TreeBatch(device, [10], [[-1, 0, 0, 1]], dtype, seed=9)
    at = 12                                                  # node 2
    b.vc[int(b.table[0, 0]), :, at, 5] = float("inf")
    got = b.run(kernels)
    assert torch.isinf(got[2, :, 5]).all() and torch.isfinite(got[[0, 1, 3]]).all()
    keep = [i for i in range(64) if i != 5]
    assert torch.isfinite(got[:, :, keep]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 80])
def test_rows_of_nobody_stay(device, kernels, dtype, d):
    """Nodes behind the last sequence, in a packed array of a fixed length."""
    rng = np.random.default_rng(2)
    b = TreeBatch(device, [40, 9, 0], trees(rng, [5, 3, 0]), dtype, d=d, extra_rows=70, seed=3)
    out = torch.full_like(b.q, 7.0)
    b.run(kernels, out=out)
    assert (out[8:] == 7).all()
    b.verify(out)


def test_contexts_shorter_than_the_tree(device, kernels):
    """Nodes that the length does not count are not attended to; a length of 0 gives zeros."""
    rng = np.random.default_rng(4)
    b = TreeBatch(device, [0, 20, 0], trees(rng, [10, 4, 6]), seed=4)
    out = b.run(kernels, lens=[7, 24, 0])
    assert not out[14:].any()
    b.sees[0] = b.sees[0] & (np.arange(10) < 7)
    want, tol = b.want()
    got = out.float().cpu().numpy()
    assert (np.abs(got - want) <= tol)[:14].all()


@pytest.mark.parametrize("scale", [0.0, -0.4, 30.0, 1e-3])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_scales(device, kernels, scale, dtype):
    rng = np.random.default_rng(7)
    TreeBatch(device, [50, 0], trees(rng, [20, 9]), dtype, seed=11, scale=scale).check(kernels)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_blocks(device, kernels, dtype):
    """Blocks whose elements lie past 2^32 in the pool."""
    rng = np.random.default_rng(8)
    b = TreeBatch(device, [100, 40], trees(rng, [12, 30]), dtype, heads=8, hkv=2, d=128, seed=12)
    es = b.pool.element_size()
    blocks = (1 << 32) // (2 * 2 * 16 * 128) + 40
    far = torch.empty((blocks, 2, 2, 16, 128), dtype=b.pool.dtype, device=device)
    assert far.numel() > 1 << 32 and far.numel() * es < 40 << 30
    n = b.pool.shape[0]
    far[-n:] = b.pool
    b.table = np.where(np.arange(b.table.shape[1]) < -(-b.ctx[:, None] // 16), b.table + blocks - n, 0).astype(np.int32)
    b.kc, b.vc = far[:, 0], far[:, 1]
    got = b.run(kernels)
    b.table = np.where(b.table > 0, b.table - (blocks - n), 0).astype(np.int32)
    b.kc, b.vc = b.pool[:, 0], b.pool[:, 1]
    b.verify(got)


def test_repeats_itself(device, kernels):
    rng = np.random.default_rng(13)
    b = TreeBatch(device, [3000, 10, 700], trees(rng, [40, 9, 17]), heads=8, hkv=2, d=128, seed=13)
    first = b.run(kernels)
    for _ in range(3):
        assert torch.equal(b.run(kernels), first)


def test_streams_at_once(device, kernels):
    """Calls on two streams, each with its own workspace."""
    rng = np.random.default_rng(14)
    batches = [TreeBatch(device, [900 + 300 * i, 50], trees(rng, [20, 30]), heads=8, hkv=2, d=128, seed=20 + i)
               for i in range(2)]
    want = [b.run(kernels) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    outs = [[], []]
    for _ in range(4):
        for i, (b, s) in enumerate(zip(batches, streams)):
            with torch.cuda.stream(s):
                outs[i].append(b.run(kernels))
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in got)


def test_captured(device, kernels):
    """A replayed graph sees new lengths, masks and queries."""
    rng = np.random.default_rng(15)
    b = TreeBatch(device, [500, 20, 0], trees(rng, [20, 30, 8]), heads=8, hkv=2, d=128, seed=30)
    table, ctx, cu, mask = b.arrays()
    op = PagedAttentionOp(b.scale, b.heads, b.hkv, b.d, b.bs, kernels)

    def step():
        return op.execute_tree(b.q, b.kc, b.vc, table, ctx, cu, mask, b.max_nodes)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for shift in (0, 3, 1):
        ctx.copy_(i32(np.maximum(b.ctx - shift, 1), device))
        mask.copy_(i32(np.roll(b.mask, shift, 0), device))
        b.q.mul_(1.25)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())
        torch.cuda.synchronize()


def test_refusals(device, kernels):
    b = TreeBatch(device, [20, 9], [[-1, 0, 0], [-1]], seed=1)
    table, ctx, cu, mask = b.arrays()
    out = torch.empty_like(b.q)
    good = dict(query=b.q, key_cache=b.kc, value_cache=b.vc, block_table=table, context_lens=ctx, cu_nodes=cu,
                tree_mask=mask, output=out, scale=b.scale, max_nodes=3)
    kernels.launch_tree(**good)
    bad = [dict(query=b.q[:, :, :32]), dict(query=b.q.float()), dict(output=out[:2]), dict(block_table=table[:1]),
           dict(context_lens=ctx.long()), dict(cu_nodes=cu[:0]), dict(cu_nodes=cu.long()), dict(tree_mask=mask[:2]),
           dict(max_nodes=33), dict(max_nodes=-1), dict(max_nodes=2**31), dict(key_cache=b.kc.float()),
           dict(query=b.q.cpu()), dict(tree_mask=mask.cpu()), dict(block_table=table[:, ::2]),
           dict(query=b.q[:, :7].contiguous(), output=out[:, :7].contiguous()),
           dict(tree_mask=i32(np.zeros((4, 40)), device), max_nodes=1025),
           dict(key_cache=b.kc[:1].expand(4, -1, -1, -1), value_cache=b.vc[:1].expand(4, -1, -1, -1))]
    for change in bad:
        with pytest.raises(RailgunError):
            kernels.launch_tree(**{**good, **change})
    n = kernels.tree_workspace_bytes(2, 3, b.heads, b.hkv, b.d, b.bs, table.shape[1])
    if n:
        with pytest.raises(RailgunError, match="workspace"):
            kernels.launch_tree(**good, workspace=torch.empty(n - 1, dtype=torch.uint8, device=device))
    op = PagedAttentionOp(b.scale, b.heads, b.hkv, b.d, 32, kernels)
    with pytest.raises(RailgunError):
        op.execute_tree(b.q, b.kc, b.vc, table, ctx, cu, mask, 3)


def test_nothing_to_do(device, kernels):
    b = TreeBatch(device, [20], [[-1, 0]], seed=1)
    table, ctx, cu, mask = b.arrays()
    out = torch.full_like(b.q, 5.0)
    none = torch.zeros(3, dtype=torch.int32, device=device)
    kernels.launch_tree(b.q, b.kc, b.vc, table[:0], ctx[:0], cu[:1], mask, out, b.scale, 2)
    kernels.launch_tree(b.q, b.kc, b.vc, table.expand(2, -1).contiguous(), ctx.expand(2).contiguous(), none, mask, out,
                        b.scale, 2)
    kernels.launch_tree(b.q[:0], b.kc, b.vc, table, ctx, cu * 0, mask[:0], out[:0], b.scale, 2)
    torch.cuda.synchronize()
    assert (out == 5).all()
