"""Draft trees beside decode rows that share a prefix or gather scores, and behind an evicted cache."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import i32
from railgun_amd.batch import DecodeSlot, DraftTree, PrefillChunk, pack_step
from railgun_amd.llama import DeviceStep
from test_gpu_cache_policy import _EvictedReference
from test_gpu_tree_model import BS, TreeReference, make
from tree64 import accept, first_largest, random_tree

pytestmark = pytest.mark.gpu


class Reference(TreeReference, _EvictedReference):
    """The CPU model with trees, over evicted caches too."""


class Steps:
    """A model and its two references; every step's logits stay within twice the drift that rounding the activations
    explains (plus 1e-3), as the model's other steps do."""

    def __init__(self, device, kernels, dtype, kv_heads, hidden):
        self.device, (self.cfg, sd, self.model) = device, make(device, kernels, dtype, kv_heads, hidden)
        self.refs = [Reference(self.cfg, sd, self.model.pool.num_blocks, BS, act_dtype=t) for t in (torch.float32, dtype)]

    def run(self, step, what):
        st = DeviceStep.from_host(step, self.device)
        logits = self.model.forward(st)
        ref32, ref16 = (r.forward(step) for r in self.refs)
        self.drift = float((ref16 - ref32).abs().max())
        err = float((logits.float().cpu() - ref32).abs().max())
        assert logits.shape == ref32.shape and err <= 2 * self.drift + 1e-3, f"{what}: {err:.4g}, drift {self.drift:.4g}"
        return st, logits

    def keep(self, st, logits, trees):
        """Verifies and compacts; trees: (DraftTree, first cached position); returns the new lengths."""
        rows = logits[st.host.num_requests - st.host.num_trees:].float().cpu().numpy()
        target = [first_largest(row) for row in rows]
        verdict = self.model.verify_trees(logits, st)
        new = self.model.keep_accepted(st, verdict).tolist()
        for s, (d, prior) in enumerate(trees):
            a, e = st.host.tree_cu[s:s + 2]
            path, following = accept(d.parents, d.token_ids, target[a:e], st.host.max_tree_depth)
            assert verdict.accepted[s].tolist() == path + [-1] * (st.host.max_tree_depth - len(path))
            assert int(verdict.next_tokens[s]) == following and new[s] == prior + len(path)
            for r in self.refs:
                r.keep(d.block_table, prior, path)
        return new


@pytest.mark.parametrize("kv_heads,hidden,dtype", [(2, 512, torch.bfloat16), (1, 1024, torch.float16)])
def test_beside_rows_that_share_a_prefix(device, kernels, kv_heads, hidden, dtype):
    """Decode rows over common blocks, read once, with their scores gathered and without, a prompt chunk, and trees,
    one of them behind the same common blocks."""
    t = Steps(device, kernels, dtype, kv_heads, hidden)
    model, pool, rng = t.model, t.model.pool, np.random.default_rng(9)
    order = iter(rng.permutation(pool.num_blocks).tolist())
    prefix = [next(order) for _ in range(6)]
    own = [7, 30, 16, 3]                                               # behind the common blocks; the last checks drafts
    tables = [prefix + [next(order) for _ in range(8)] for _ in own] + [[next(order) for _ in range(8)]]
    lens = [6 * BS + n for n in own] + [21]
    text = rng.integers(t.cfg.vocab_size, size=6 * BS).tolist()
    t.run(pack_step([PrefillChunk(text, 0, prefix)], [], BS), "common prompt")
    t.run(pack_step([PrefillChunk(rng.integers(t.cfg.vocab_size, size=n).tolist(), 6 * BS, table)
                     for n, table in zip(own, tables)]
                    + [PrefillChunk(rng.integers(t.cfg.vocab_size, size=21).tolist(), 0, tables[4])], [], BS), "prompts")
    pool.scores.fill_(5.0)
    used, real = [], model.kernels.launch_shared_prefix
    model.kernels.launch_shared_prefix = lambda *a: (used.append(a[-2]), real(*a))[1]
    model.kernels.shared_prefix_pays = lambda *a: True
    chunk_table = [next(order) for _ in range(4)]
    chunk = 0
    try:
        for i, gather in enumerate((False, True, True, False)):
            sizes = [17 + i, 9]
            trees = [DraftTree(rng.integers(t.cfg.vocab_size, size=n).tolist(), random_tree(rng, n, 5), lens[s] + n, tables[s])
                     for s, n in zip((3, 4), sizes)]
            rows = [DecodeSlot(int(rng.integers(t.cfg.vocab_size)), lens[s] + 1, tables[s],
                               scored_len=(0 if i == 1 else lens[s]) if gather else None) for s in range(3)]
            beside = [PrefillChunk(rng.integers(t.cfg.vocab_size, size=11).tolist(), chunk, chunk_table)]
            chunk += 11
            step = pack_step(beside, rows, BS, share_prefix=True, gather_scores=gather, draft_trees=trees)
            assert step.shared_decode_blocks == 6 and step.num_decode == 3
            before = pool.scores.clone()
            st, logits = t.run(step, f"step {i}")
            for s in range(3):
                lens[s] += 1
            if gather:                                                 # each row's cells behind the prefix, and no others
                cells = torch.zeros_like(pool.scores, dtype=torch.bool)
                for s in range(3):
                    at = np.arange(6 * BS, lens[s])
                    cells[:, np.asarray(tables[s])[at // BS], :, at % BS] = True
                assert (pool.scores[cells] > 0).all() and (pool.scores[cells] != 5).all()
                at = np.arange(6 * BS)                                 # (the prefix: cleared where no row counts it)
                cells[:, np.asarray(prefix)[at // BS], :, at % BS] = True
                for d in trees:
                    at = np.arange(d.seq_len - len(d.token_ids), d.seq_len)
                    cells[:, np.asarray(d.block_table)[at // BS], :, at % BS] = True
                assert torch.equal(pool.scores[~cells], before[~cells])
            lens[3:] = t.keep(st, logits, [(d, lens[s]) for d, s in zip(trees, (3, 4))])
    finally:
        del model.kernels.launch_shared_prefix, model.kernels.shared_prefix_pays
    assert len(used) == 2 * t.cfg.num_hidden_layers                    # the steps that did not gather


@pytest.mark.parametrize("kv_heads,hidden,dtype", [(2, 512, torch.bfloat16), (1, 512, torch.float16)])
def test_behind_an_evicted_cache(device, kernels, kv_heads, hidden, dtype):
    """Trees whose place in the text lies past what is cached, and the steps behind them."""
    t = Steps(device, kernels, dtype, kv_heads, hidden)
    pool, rng = t.model.pool, np.random.default_rng(10)
    lens, budget = [150, 90], 64
    tables = [list(range(20 * s, 20 * s + 14)) for s in range(2)]
    t.run(pack_step([PrefillChunk(rng.integers(t.cfg.vocab_size, size=n).tolist(), 0, table)
                     for n, table in zip(lens, tables)], [], BS), "prompts")
    pool.scores.copy_(torch.rand(pool.scores.shape, generator=torch.Generator().manual_seed(2)))
    kept = torch.empty((t.cfg.num_hidden_layers, 2, kv_heads, budget), device=device, dtype=torch.int32)
    new = pool.evict(i32(tables, device), i32(lens, device), budget, 8, 4, None, kept).tolist()
    assert new == [budget] * 2
    for r in t.refs:
        r.evict(tables, lens, kept.cpu().numpy(), new)
    place, lens = list(lens), new
    for i in range(2):
        trees = [DraftTree(rng.integers(t.cfg.vocab_size, size=n).tolist(), random_tree(rng, n, 4), lens[s] + n, tables[s],
                           position=place[s]) for s, n in enumerate((20, 33 + i))]
        step = pack_step([], [], BS, draft_trees=trees)
        st, logits = t.run(step, f"trees {i}")
        np.testing.assert_array_equal(st.positions.cpu().numpy(), step.positions)
        wrong = pack_step([], [], BS, draft_trees=[DraftTree(d.token_ids, d.parents, d.seq_len, d.block_table)
                                                   for d in trees])
        off = t.model.forward(DeviceStep.from_host(wrong, device)).float().cpu()
        assert float((off - t.refs[0].forward(step)).abs().max()) > 2 * t.drift + 1e-3
        st, logits = t.run(step, f"trees {i} again")                   # (the caches hold this step's tokens)
        after = t.keep(st, logits, [(d, n) for d, n in zip(trees, lens)])
        place = [p + a - n for p, a, n in zip(place, after, lens)]
        lens = after
    t.run(pack_step([], [DecodeSlot(3 + s, lens[s] + 1, tables[s], position=place[s]) for s in range(2)], BS), "decode")
