"""Trees of drafted tokens: plain layout, verification and compaction, and attention in 64 bits with the
bounds of attention64."""
from __future__ import annotations

import math

import numpy as np
import torch

from attention64 import HALF_STEP, U, rows64
from helpers import TORCH_DT, i32


def random_tree(rng, n, depth=6, roots=1):
    """Parents of n nodes, none deeper than ``depth``; the first ``roots`` nodes have none."""
    parents, level = [], []
    for j in range(n):
        fits = [i for i in range(j) if level[i] < depth]
        p = -1 if j < roots or not fits else int(rng.choice(fits[-8:] if rng.random() < 0.5 else fits))
        parents.append(p)
        level.append(0 if p < 0 else level[p] + 1)
    return parents


def ancestors(parents):
    """bool [n, n]: row j has set j and its ancestors."""
    sees = np.zeros((len(parents), len(parents)), bool)
    for j, p in enumerate(parents):
        if 0 <= p < j:
            sees[j] = sees[p]
        sees[j, j] = True
    return sees


def words_of(sees, words):
    """The bits of bool [n, m] as int32 [n, words]."""
    n, m = sees.shape
    bits = np.zeros((n, 32 * words), np.uint64)
    bits[:, :m] = sees
    return (bits.reshape(n, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


def first_largest(row):
    """Lowest index of the largest value, NaN as -inf."""
    row = np.where(np.isnan(row), -np.inf, row)
    return int(np.flatnonzero(row == row.max())[0])


def accept(parents, draft, target, most):
    """(path, next token) of one tree, plainly."""
    if not len(parents):
        return [], -1
    path = [0]
    while len(path) < most:
        fits = [j for j, p in enumerate(parents) if p == path[-1] and j > p and draft[j] == target[p]]
        if not fits:
            break
        path.append(fits[0])
    return path, int(target[path[-1]])


class TreeBatch:
    """Sequences of ``prior`` cached tokens and a tree each (its parents, or a bool mask); cells that no
    sequence uses hold NaN."""

    def __init__(self, device, prior, trees, dtype="bf16", heads=8, hkv=2, d=64, bs=16, seed=0, wide=0, fused=True,
                 extra_rows=0, words=None, scale=None):
        rng = np.random.default_rng(seed)
        self.device, self.dtype, self.heads, self.hkv, self.d, self.bs = device, dtype, heads, hkv, d, bs
        self.sees = [t if isinstance(t, np.ndarray) else ancestors(t) for t in trees]
        self.nodes = np.array([len(t) for t in self.sees], np.int64)
        self.prior = np.asarray(prior, np.int64)
        self.ctx = self.prior + self.nodes
        self.cu = np.concatenate([[0], np.cumsum(self.nodes)])
        self.max_nodes = int(self.nodes.max())
        need = -(-self.ctx // bs)
        total = int(need.sum()) + 3
        order = iter(rng.permutation(total))
        self.table = np.zeros((len(need), max(1, int(need.max())) + wide), np.int32)
        used = np.zeros((total, bs), bool)
        for s, n in enumerate(need):
            self.table[s, :n] = [next(order) for _ in range(int(n))]
            t = np.arange(int(self.ctx[s]))
            used[self.table[s, t // bs], t % bs] = True
        g = torch.Generator(device=device).manual_seed(seed)
        dt = TORCH_DT[dtype]
        fresh = torch.randn((total, 2, hkv, bs, d), generator=g, device=device).to(dt)
        keep = torch.as_tensor(used, device=device)[:, None, None, :, None]
        self.pool = torch.where(keep, fresh, torch.full_like(fresh, float("nan")))
        self.kc, self.vc = self.pool[:, 0], self.pool[:, 1]
        if not fused:
            self.kc, self.vc = self.kc.contiguous(), self.vc.contiguous()
        rows = int(self.cu[-1]) + extra_rows
        self.q = (2 * torch.randn((rows, heads, d), generator=g, device=device)).to(dt)
        words = words or max(1, -(-self.max_nodes // 32))
        self.mask = np.full((rows, words), -1, np.int32)
        for s, sees in enumerate(self.sees):
            self.mask[self.cu[s]:self.cu[s + 1]] = words_of(sees, words)
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale

    def arrays(self):
        return tuple(i32(a, self.device) for a in (self.table, self.ctx, self.cu, self.mask))

    def run(self, kernels, workspace=None, out=None, lens=None):
        table, ctx, cu, mask = self.arrays()
        if lens is not None:
            ctx = i32(lens, self.device)
        out = torch.full_like(self.q, float("nan")) if out is None else out
        if workspace is None:
            n = kernels.tree_workspace_bytes(len(self.nodes), self.max_nodes, self.heads, self.hkv, self.d, self.bs,
                                             self.table.shape[1])
            workspace = torch.full((n,), 0xFF, dtype=torch.uint8, device=self.device)  # NaN wherever it is read
        kernels.launch_tree(self.q, self.kc, self.vc, table, ctx, cu, mask, out, self.scale, self.max_nodes, workspace)
        return out

    def want(self, rounded_p=True):
        """(out, bound on it), float64 [rows, H, D]; zeros in rows of nobody."""
        qn = self.q.float().cpu().numpy().astype(np.float64)
        out, tol = np.zeros_like(qn), np.zeros_like(qn)
        half, g, d = HALF_STEP[self.dtype], self.heads // self.hkv, self.d
        for s, sees in enumerate(self.sees):
            n, count, first = int(self.ctx[s]), int(self.nodes[s]), int(self.cu[s])
            if not count:
                continue
            blocks = self.table[s, :-(-n // self.bs)]
            k, v = rows64(self.kc, blocks, n), rows64(self.vc, blocks, n)
            seen = np.concatenate([np.ones((count, int(self.prior[s])), bool), sees], 1)
            for h in range(self.heads):
                kh, vh, x3 = k[h // g], v[h // g], qn[first:first + count, h]
                for j in range(count):
                    t = np.flatnonzero(seen[j])
                    if not len(t):
                        continue
                    x = self.scale * (kh[t] @ x3[j])
                    mass = abs(self.scale) * (np.abs(kh[t]) @ np.abs(x3[j]))
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    dx = ((d + 2) * U * mass + 2 * U * np.abs(x - x.max())).max() + 2 * U
                    rel = 2 * (dx + n * U)
                    o, pv = p @ vh[t], p @ np.abs(vh[t])
                    out[first + j, h] = o
                    tol[first + j, h] = (rel * pv * (1 + half) + half * np.abs(o) + 1e-30
                                         + (2 * half * pv if rounded_p and self.dtype != "f32" else 0))
        return out, tol

    def verify(self, out):
        want, tol = self.want()
        got = out.float().cpu().numpy().astype(np.float64)[:int(self.cu[-1])]
        want, tol = want[:len(got)], tol[:len(got)]
        assert np.isfinite(got).all(), f"not finite in rows {np.unique(np.nonzero(~np.isfinite(got))[0])[:10]}"
        over = np.abs(got - want) - tol
        row = int(over.max((1, 2)).argmax())
        assert (over <= 0).all(), f"row {row} off by {np.abs(got - want)[row].max():.3g}, {over.max():.3g} over the bound"

    def check(self, kernels, **kw):
        self.verify(self.run(kernels, **kw))
