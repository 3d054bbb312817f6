"""Decode attention over a shared prefix (rg_paged_attention_shared_prefix) against 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from attention64 import assert_within, attention64
from helpers import TORCH_DT, dev_f32, i32
from railgun_amd.ops import PagedAttentionOp, RailgunError

pytestmark = pytest.mark.gpu


class Batch:
    """Sequences that begin with the same `shared` blocks; cells that no sequence uses hold NaN."""

    def __init__(self, device, ctx, shared, dtype="bf16", heads=8, hkv=2, d=64, bs=16, seed=0, wide=0, fused=True):
        rng = np.random.default_rng(seed)
        self.ctx, self.dtype, self.device, self.shared = np.asarray(ctx, np.int64), dtype, device, shared
        need = -(-np.maximum(self.ctx, 0) // bs)
        b = len(ctx)
        total = shared + int(np.maximum(need - shared, 0).sum()) + 3
        order = iter(rng.permutation(total))
        prefix = [next(order) for _ in range(shared)]
        self.table = np.zeros((b, max(1, shared, int(need.max())) + wide), np.int32)
        self.table[:, :shared] = prefix
        used = np.zeros((total, bs), bool)
        for s in range(b):
            for i in range(shared, int(need[s])):
                self.table[s, i] = next(order)
            t = np.arange(max(int(self.ctx[s]), 0))
            used[self.table[s, t // bs], t % bs] = True
        g = torch.Generator(device=device).manual_seed(seed)
        dt = TORCH_DT[dtype]
        fresh = torch.randn((total, 2, hkv, bs, d), generator=g, device=device).to(dt)
        mask = torch.as_tensor(used, device=device)[:, None, None, :, None]
        self.pool = torch.where(mask, fresh, torch.full_like(fresh, float("nan")))
        self.kc, self.vc = self.pool[:, 0], self.pool[:, 1]
        if not fused:
            self.kc, self.vc = self.kc.contiguous(), self.vc.contiguous()
        self.q = (2 * torch.randn((b, heads, d), generator=g, device=device)).to(dt)
        self.scale, self.heads, self.hkv, self.d, self.bs = 1.0 / math.sqrt(d), heads, hkv, d, bs

    def op(self, kernels):
        return PagedAttentionOp(self.scale, self.heads, self.hkv, self.d, self.bs, kernels)

    def run(self, kernels, workspace=None, lens=None):
        """launch_shared_prefix: the shared product wherever its shapes allow it."""
        out = torch.full_like(self.q, float("nan"))
        b, mb = self.table.shape
        shape = (b, self.heads, self.hkv, self.d, self.bs, mb)
        if workspace is None:
            n = kernels.shared_prefix_workspace_bytes(*shape, self.shared)
            workspace = torch.empty(n, dtype=torch.uint8, device=self.device)
        kernels.launch_shared_prefix(self.q, self.kc, self.vc, i32(self.table, self.device),
                                     i32(self.ctx if lens is None else lens, self.device), out, self.scale,
                                     self.heads, self.hkv, self.d, self.bs, mb, b, self.shared, workspace)
        return out

    def verify(self, out):
        want, tol, _, _ = attention64(self.q, self.kc, self.vc, self.table, self.ctx, self.scale, self.dtype,
                                      rounded_p=True)
        assert_within(dev_f32(out), want, tol)

    def check(self, kernels, **kw):
        self.verify(self.run(kernels, **kw))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,hkv,d", [(4, 4, 64), (8, 4, 128), (6, 2, 64), (8, 2, 128), (10, 2, 64), (12, 2, 128),
                                         (14, 2, 128), (16, 2, 64), (32, 2, 128), (8, 2, 256)])
def test_tiles(device, kernels, dtype, heads, hkv, d):
    """Every ratio of heads; rows of no token, of part of the prefix, of all of it and nothing else."""
    b = Batch(device, [48 + 30, 0, 1, 48, 47, 49, 48 + 300, 33], 3, dtype, heads, hkv, d, seed=heads * d)
    b.check(kernels)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,hkv,d,bs", [(4, 2, 80, 16), (6, 3, 20, 8), (2, 2, 4, 5), (18, 2, 64, 16), (9, 1, 128, 16),
                                            (4, 2, 128, 1), (4, 2, 64, 512)])
def test_other_shapes(device, kernels, dtype, heads, hkv, d, bs):
    p = 3 * bs
    Batch(device, [p + 40, 0, p, p + 1, p + 300], 3, dtype, heads, hkv, d, bs, seed=d + bs).check(kernels)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("shared", [1, 2, 5])
def test_block_sizes(device, kernels, bs, shared):
    """Prefixes of one sub-block, of an odd number of them, of several splits."""
    p = shared * bs
    Batch(device, [p + 9, p, p + 100, p + 33], shared, bs=bs, fused=bs != 64, seed=bs + shared).check(kernels)


@pytest.mark.parametrize("batch", [1, 2, 3, 8, 31, 32, 33, 65, 130])
def test_batches(device, kernels, batch):
    """One row tile, its edges, several of them."""
    rng = np.random.default_rng(batch)
    Batch(device, 112 + rng.integers(0, 60, batch), 7, heads=8, hkv=2, seed=batch).check(kernels)


@pytest.mark.parametrize("shared", [130, 257, 1100])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_long_prefix(device, kernels, shared, dtype):
    """Windows of 64 key tiles and more within one split."""
    p = shared * 16
    Batch(device, [p + 5] * 20 + [0, p - 1, p], shared, dtype, heads=32, hkv=8, d=128, seed=shared).check(kernels)


def test_many_rows_of_a_long_prefix(device, kernels):
    """Row tiles enough that a split holds more key tiles than a window."""
    p = 16 * 300
    Batch(device, [p + i % 7 for i in range(300)], 300, heads=64, hkv=16, d=64, seed=3).check(kernels)


def test_no_sequence_has_the_whole_prefix(device, kernels):
    Batch(device, [40, 100, 0, 7], 20, seed=4).check(kernels)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("ctx", [[0, 0, 700, 330, 0], [319, 40, 0, 320, 500], [0] * 150 + [400] + [0] * 70 + [321],
                                 [100, 0, 7]])
def test_shorter_rows_have_tables_of_their_own(device, kernels, dtype, ctx):
    """Rows that pad the batch, or end inside the prefix, hold other blocks and no valid entry behind their
    tokens; the prefix's blocks come from a row that has them all."""
    c = Batch(device, ctx, 20, dtype=dtype, seed=len(ctx), wide=2)
    spare = iter(range(len(c.pool), len(c.pool) + 64))
    own = []
    for s, n in enumerate(ctx):
        if n < 320:
            used = -(-n // 16)
            c.table[s] = -7
            for i in range(used):
                c.table[s, i] = next(spare)
                own.append(torch.randn(c.pool.shape[1:], device=device).to(c.pool.dtype))
    c.pool = torch.cat([c.pool, torch.stack(own)]) if own else c.pool
    c.kc, c.vc = c.pool[:, 0], c.pool[:, 1]
    c.check(kernels)


def test_all_rows_empty_and_nothing_shared(device, kernels):
    Batch(device, [0, 0, 0], 4, seed=5).check(kernels)
    Batch(device, [70, 0, 5], 0, seed=5).check(kernels)


def test_negative_length_counts_as_none(device, kernels):
    Batch(device, [0, 60, 33], 2, seed=6).check(kernels, lens=np.array([-9, 60, 33]))


def test_table_much_wider_than_the_contexts(device, kernels):
    Batch(device, [70, 700, 64], 4, wide=2000, seed=7).check(kernels)


@pytest.mark.parametrize("scale", [0.0, -0.4, 3.0])
def test_scales(device, kernels, scale):
    b = Batch(device, [200, 170, 161], 10, seed=8)
    b.scale = scale
    b.check(kernels)


def test_growing_scores_move_the_maximum(device, kernels):
    """Keys that get larger along the prefix: the running maximum moves at every tile."""
    b = Batch(device, [16 * 40 + 3] * 5, 40, d=128, seed=9)
    for i in range(40):
        b.pool[int(b.table[0, i]), 0] *= 0.05 * (i + 1)
    b.check(kernels)


def test_equals_the_plain_decode_of_the_same_tables(device, kernels):
    b = Batch(device, [330, 500, 321, 322], 20, heads=16, hkv=4, d=128, seed=10)
    table, lens = i32(b.table, device), i32(b.ctx, device)
    plain = b.op(kernels).execute(b.q, b.kc, b.vc, table, lens, None, 500)
    torch.testing.assert_close(b.run(kernels).float(), plain.float(), atol=2e-2, rtol=1e-2)


def test_replayed_graph(device, kernels):
    b = Batch(device, [400, 330, 0, 321], 20, heads=16, hkv=4, d=128, seed=11)
    table, lens, mb = i32(b.table, device), i32(b.ctx, device), b.table.shape[1]
    ws = torch.empty(kernels.shared_prefix_workspace_bytes(4, 16, 4, 128, 16, mb, 20), dtype=torch.uint8, device=device)
    out = torch.empty_like(b.q)

    def step():
        kernels.launch_shared_prefix(b.q, b.kc, b.vc, table, lens, out, b.scale, 16, 4, 128, 16, mb, 4, 20, ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        b.q.copy_(torch.randn_like(b.q))
        graph.replay()
        torch.cuda.synchronize()
        b.verify(out)
        step()


def test_workspace_contents_do_not_matter(device, kernels):
    b = Batch(device, [130, 500, 64, 3], 4, seed=12)
    n = kernels.shared_prefix_workspace_bytes(4, 8, 2, 64, 16, b.table.shape[1], 4)
    b.check(kernels, workspace=torch.full((n,), 255, dtype=torch.uint8, device=device))


def test_pool_far_past_32_bits(device, kernels):
    bs, d, hkv = 16, 64, 2
    blocks = (1 << 32) // (2 * hkv * bs * d) + 60
    pool = torch.zeros((blocks, 2, hkv, bs, d), dtype=torch.bfloat16, device=device)
    pool[blocks - 50:].normal_()
    b = Batch(device, [310, 320], 18, seed=13)
    b.pool, b.kc, b.vc = pool, pool[:, 0], pool[:, 1]
    b.table = np.stack([np.arange(20), np.concatenate([np.arange(18), [30, 31]])]).astype(np.int32) + blocks - 50
    b.check(kernels)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,shared,pays", [(3, 4, False), (150, 40, True)])
def test_op(device, kernels, dtype, batch, shared, pays):
    """The op takes the shared product where it pays, and is right on either side."""
    ctx = [shared * 16 + i % 50 for i in range(batch - 1)] + [0]
    b = Batch(device, ctx, shared, dtype, heads=16, hkv=4, d=128, seed=batch)
    mb = b.table.shape[1]
    assert kernels.shared_prefix_pays(batch, 16, 4, 128, 16, mb, shared, b.q.dtype) is pays
    table, lens = i32(b.table, device), i32(b.ctx, device)
    b.verify(b.op(kernels).execute_shared_prefix(b.q, b.kc, b.vc, table, lens, shared))
    ws = torch.empty(kernels.shared_prefix_workspace_bytes(batch, 16, 4, 128, 16, mb, shared), dtype=torch.uint8,
                     device=device)
    b.verify(b.op(kernels).execute_shared_prefix(b.q, b.kc, b.vc, table, lens, shared, ws))


def test_refusals(device, kernels):
    b = Batch(device, [40, 30], 1, seed=14)
    op, table, lens = b.op(kernels), i32(b.table, device), i32(b.ctx, device)
    good = dict(q=b.q, k_cache=b.kc, v_cache=b.vc, block_table=table, context_lens=lens, shared_blocks=1)
    for change in (dict(shared_blocks=-1), dict(shared_blocks=4), dict(q=b.q[0]), dict(q=b.q.float()), dict(q=b.q[:1]),
                   dict(q=b.q[..., :32].contiguous()), dict(q=b.q.transpose(0, 1)), dict(block_table=table[:1]),
                   dict(block_table=table.long()), dict(context_lens=lens[:1]), dict(q=b.q.cpu()),
                   dict(workspace=torch.empty(16, dtype=torch.uint8, device=device))):
        with pytest.raises(RailgunError):
            op.execute_shared_prefix(**{**good, **change})
    ws = torch.empty(kernels.shared_prefix_workspace_bytes(2, 8, 2, 64, 16, table.shape[1], 1), dtype=torch.uint8,
                     device=device)
    for t, n in ((table[:1], 2), (table, 3)):  # a row short, rows of another width than said
        with pytest.raises(RailgunError):
            kernels.launch_shared_prefix(b.q, b.kc, b.vc, t, lens, torch.empty_like(b.q), 0.1, 8, 2, 64, 16,
                                         table.shape[1] + (n == 3), 2, 1, ws)
