"""Paged decode attention in 64 bits, with the error bounds its kernels are held to.

Bounds (u = 2^-23 per fp32 operation: the matrix instructions may truncate).  A raw score is a sum of D
products, so it is off by at most (D + 2) u sum|q||k|; times the scale that is the relative error of
e^x, to which rounding x - max (u |x - max|) and the exponential (2 u) add.  A weight is a quotient of
such terms, the sum over T tokens adding T u: relative error 2 (dx + T u).  An output is sum p v:
off by that times sum p |v|, plus its own rounding, half a step of the output's type.  Where the
probabilities are rounded to the storage type before the product with V, that adds half a step of it
to each term of the sum.
"""
from __future__ import annotations

import numpy as np
import torch

U = 2.0 ** -23
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def rows64(cache: torch.Tensor, blocks, n: int) -> np.ndarray:
    """The first n rows behind a list of blocks of a [NB, H_kv, bs, D] cache: float64 [H_kv, n, D]."""
    ids = torch.as_tensor(np.asarray(blocks, np.int64), device=cache.device)
    x = cache[ids].float().cpu().numpy().astype(np.float64)
    nb, hkv, bs, d = x.shape
    return x.transpose(1, 0, 2, 3).reshape(hkv, nb * bs, d)[:, :n]


def attention64(q, kc, vc, table, ctx, scale, dtype, rounded_p=False):
    """(out, bound on it, weights, bound on them): out [B, H, D]; weights a list of [H_kv, ctx] sums over
    the query heads of a kv-head.  table [B, MB] and ctx [B] on the host."""
    qn = q.float().cpu().numpy().astype(np.float64)
    b, heads, d = qn.shape
    hkv, bs = int(kc.shape[1]), int(kc.shape[2])
    g = heads // hkv
    out, tol = np.zeros_like(qn), np.zeros_like(qn)
    weights, wtol = [], []
    half = HALF_STEP[dtype]
    for s in range(b):
        n = int(ctx[s])
        if n <= 0:
            weights.append(np.zeros((hkv, 0)))
            wtol.append(np.zeros((hkv, 0)))
            continue
        blocks = table[s, :-(-n // bs)]
        k, v = rows64(kc, blocks, n), rows64(vc, blocks, n)
        x3 = qn[s].reshape(hkv, g, d)
        x = scale * np.einsum("hgd,htd->hgt", x3, k)
        mass = abs(scale) * np.einsum("hgd,htd->hgt", np.abs(x3), np.abs(k))
        top = x.max(-1, keepdims=True)
        p = np.exp(x - top)
        p /= p.sum(-1, keepdims=True)
        dx = ((d + 2) * U * mass + 2 * U * np.abs(x - top)).max(-1, keepdims=True) + 2 * U
        rel = 2 * (dx + n * U)
        o = np.einsum("hgt,htd->hgd", p, v)
        pv = np.einsum("hgt,htd->hgd", p, np.abs(v))
        out[s] = o.reshape(heads, d)
        tol[s] = (rel * pv * (1 + half) + (2 * half * pv if rounded_p and dtype != "f32" else 0)
                  + half * np.abs(o) + 1e-30).reshape(heads, d)
        weights.append(p.sum(1))
        wtol.append((rel * p).sum(1))
    return out, tol, weights, wtol


def assert_within(got, want, tol, what=""):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - tol
    assert (over <= 0).all(), f"{what}: off by {np.abs(got - want).max():.3g}, {over.max():.3g} over the bound"
