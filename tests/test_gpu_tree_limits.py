"""Attention of draft trees past its declared limits, at scores where fp32 runs out of steps, and at long contexts in the
form that takes any shape; lengths of accepted paths."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from attention64 import HALF_STEP, U
from test_gpu_tree import check_verify
from tree64 import TreeBatch, accept, ancestors, random_tree

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


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("first,step", [(2 ** 20 - 4000, 0), (2 ** 20 - 12, 0), (2 ** 20 - 6, 1), (2 ** 20 - 40, 4),
                                        (2 ** 20 + 5, 0), (3 * 2 ** 19, 0)])
def test_scores_around_two_to_the_twenty(device, kernels, dtype, d, first, step):
    """Scores (in log2 units) of ``first`` and a few more, ``step`` more every 300 tokens, so that the maximum passes
    2^20, where fp16's probabilities change their factor, in the middle of a piece, between the pieces of one
    sequence, or nowhere.

    The products are of whole numbers that every type holds: q is 1 in one dim, 2^4 in one and 2^7 in the others, K at
    most 2^8, so their sums are exact in fp32.  On the matrix cores a score is multiplied and its reference subtracted in
    one rounding, so its error is relative to the distance from the maximum; the form for other dims rounds the score
    first, by half a step of fp32 at its size.  In fp16 a probability below 2^-14 is off by 2^-25 at most, where the
    largest is 1 at least."""
    n, nodes = 1500, 6
    b = TreeBatch(device, [n, 40], [random_tree(np.random.default_rng(1), nodes), [-1]], dtype, heads=4, hkv=2, d=d, seed=3,
                  scale=math.log(2))
    g = torch.Generator(device=device).manual_seed(first)
    score = first + torch.randint(0, 7, (b.kc.shape[0], 16), generator=g, device=device)
    for s in range(2):
        t = np.arange(int(b.ctx[s]))
        score[b.table[s, t // 16], t % 16] += torch.as_tensor(t // 300 * step, device=device)
    # score = 2^7 high + 2^4 k_(d - 2) + k_(d - 1), high spread over the other dims.
    high = score // 128
    k = (high // (d - 2))[..., None] + (torch.arange(d, device=device) < (high % (d - 2))[..., None]).long()
    k[..., d - 2], k[..., d - 1] = score // 16 % 8, score % 16
    q = torch.full((d,), 128, dtype=torch.int64, device=device)
    q[d - 2], q[d - 1] = 16, 1
    assert torch.equal((k * q).sum(-1), score)
    assert all(torch.equal(x.to(b.kc.dtype).to(torch.int64), x) for x in (k, q))
    used = ~torch.isnan(b.kc[:, 0, :, 0])
    b.kc.copy_(torch.where(used[:, None, :, None], k[:, None].to(b.kc.dtype), b.kc))
    b.q.copy_(q.to(b.q.dtype).expand_as(b.q))
    got = b.run(kernels).float().cpu().numpy().astype(np.float64)
    half = HALF_STEP[dtype]
    at, vc = score.cpu().numpy().astype(np.float64), b.vc.float().cpu().numpy().astype(np.float64)
    scale = float(np.float32(b.scale))
    for s, sees in enumerate(b.sees):
        t = np.arange(int(b.ctx[s]))
        blocks = b.table[s, t // 16]
        x = scale * at[blocks, t % 16]
        for j in range(len(sees)):
            see = np.concatenate([np.ones(int(b.prior[s]), bool), sees[j]])
            away = x[see] - x[see].max()
            p = np.exp(away)
            # Weights of e^-100 and less count for nothing; the others' relative error: the scale's, the product's and the
            # difference's rounding (3 U of the distance), the exponential's, and the sum's.
            dx = 3 * U * min(100.0, float(-away.min())) + 2 * U + (U / 2 * float(np.abs(x).max()) if d == 80 else 0)
            rel = 2 * (dx + len(t) * U)
            p /= p.sum()
            for h in range(b.heads):
                v = vc[blocks, h // 2, t % 16][see]
                o, pv = p @ v, p @ np.abs(v)
                tol = rel * pv * (1 + half) + half * np.abs(o) + 1e-30 + (2 * half * pv if dtype != "f32" else 0)
                tol = tol + (len(t) * 2.0 ** -25 * np.abs(v).max() if dtype == "f16" else 0)
                off = np.abs(got[int(b.cu[s]) + j, h] - o)
                assert (off <= tol).all(), f"sequence {s} node {j} head {h}: {off.max():.3g}, {(off - tol).max():.3g} over"


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,hkv,d,bs", [(4, 2, 256, 16), (6, 2, 80, 16), (4, 4, 96, 8)])
def test_other_shapes_at_long_contexts(device, kernels, dtype, heads, hkv, d, bs):
    rng = np.random.default_rng(d + heads)
    TreeBatch(device, [4096, 0, 1777], [random_tree(rng, 24), [-1], random_tree(rng, 7)], dtype, heads, hkv, d, bs,
              seed=d).check(kernels)


@pytest.mark.parametrize("most", [1, 2, 12])
def test_lengths_of_accepted_paths(device, kernels, most):
    """Those of the plain walk without a limit, or the limit."""
    rng = np.random.default_rng(most)
    sizes = [0, 1, 2, 40, 200, 1024, 33] * 20
    trees = [random_tree(rng, n, 9, roots=1 + n % 3) for n in sizes]
    given = dict(agree=0.9, seed=most, sampled=rng.integers(0, 3, sum(sizes)))
    lengths = check_verify(kernels, device, trees, None, most=most, **given)
    whole = check_verify(kernels, device, trees, None, most=1024, **given)
    assert lengths == [min(n, most) for n in whole] and max(whole) >= 9
    assert accept([-1, 0, 1], [5, 1, 2], [1, 2, 9], 9) == ([0, 1, 2], 9)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_as_many_sequences_as_there_may_be(device, kernels, dtype):
    """65,535, most of them a root alone, which takes its own value; some padded, some long."""
    rng = np.random.default_rng(4)
    seqs, some = 65535, [0, 300, 40000, 65534]
    trees = [[-1] if i % 7 else [] for i in range(seqs)]
    prior = np.zeros(seqs, np.int64)
    for s in some:
        trees[s], prior[s] = random_tree(rng, 9), 500 + s % 100
    b = TreeBatch(device, prior, trees, dtype, heads=4, hkv=2, d=64, seed=4)
    got = b.run(kernels)
    alone = np.asarray([s for s in range(seqs) if len(trees[s]) == 1])
    rows = torch.as_tensor(b.cu[alone], device=device)
    values = b.vc[torch.as_tensor(b.table[alone, 0].astype(np.int64), device=device), :, 0]
    values = values.repeat_interleave(2, 1)
    # p v / p: in 16 bits p is a power of two.  In fp32 it is 1 but for the rounding of its score, so the product (which
    # may truncate, U), the quotient 1 / p and the product with that (U / 2 each) are rounded.
    off = (got[rows].double() - values.double()).abs()
    assert (off <= (2 * U if dtype == "f32" else 0) * values.double().abs()).all()
    few = TreeBatch(device, prior[some], [trees[s] for s in some], dtype, heads=4, hkv=2, d=64)
    few.kc, few.vc, few.table = b.kc, b.vc, b.table[some]
    few.q = torch.cat([b.q[b.cu[s]:b.cu[s + 1]] for s in some])
    few.verify(torch.cat([got[b.cu[s]:b.cu[s + 1]] for s in some]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_are_not_on_16_bytes(device, kernels, dtype):
    """Queries, output or caches off the 16 bytes that the matrix cores' form reads: the other form."""
    rng = np.random.default_rng(6)
    b = TreeBatch(device, [50, 0, 7], [random_tree(rng, 12), [-1], random_tree(rng, 40)], dtype, seed=6)

    def off(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape)
        return flat.copy_(t)

    q, kc, vc = b.q, b.kc.contiguous(), b.vc.contiguous()
    for what in ("q", "out", "k", "v"):
        b.q, b.kc, b.vc = off(q) if what == "q" else q, off(kc) if what == "k" else kc, off(vc) if what == "v" else vc
        b.check(kernels, out=off(torch.full_like(q, float("nan"))) if what == "out" else None)
