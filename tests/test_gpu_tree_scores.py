"""Steps over drafted tokens in a pool with scores: accepted tokens hold a score of no weight, whatever their blocks
held before, and decode steps that gather and evictions go on from there."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from railgun_amd.batch import DecodeSlot, DraftTree, pack_step
from railgun_amd.llama import DeviceStep
from test_gpu_cache_policy_rows import BS, GROUP, SLACK, gathered, prefill, small_model, step
from test_gpu_evict import keep_positions

pytestmark = pytest.mark.gpu
PARENTS = [-1, 0, 0, 2, 2, 4, 3, 5]


def tree_step(model, device, rows, agree=3):
    """A step of a tree of eight tokens behind each of the rows (table, cached tokens), whose drafts agree with the
    model for ``agree`` levels; returns (step, new lengths)."""
    draft = [[3 + s] + [0] * (len(PARENTS) - 1) for s in range(len(rows))]
    for _ in range(agree + 1):
        st = DeviceStep.from_host(pack_step([], [], BS, draft_trees=[
            DraftTree(d, PARENTS, n + len(PARENTS), t) for d, (t, n) in zip(draft, rows)]), device)
        verdict = model.verify_trees(model.forward(st), st)
        target = verdict.target_tokens.view(len(rows), -1).tolist()
        for d, told in zip(draft, target):
            for j in (2, 4, 5)[:agree]:
                d[j] = told[PARENTS[j]]
    return st, model.keep_accepted(st, verdict).tolist()


def test_accepted_tokens_hold_no_weight(device, kernels):
    """Behind a decode step that gathered: the cells before the tree stay, those of the accepted tokens are 0; the next
    gathering step may count them or not, and eviction goes by the sums."""
    model, pool = small_model(device, kernels)
    tables, lens = [[20, 21, 22, 23, 24], [30, 31, 32, 33, 34]], [40, 47]
    prefill(model, device, tables, lens)
    pool.scores.fill_(7.0)                                             # left over from earlier owners
    lens = [n + 1 for n in lens]
    step(model, device, [(t, n, 0) for t, n in zip(tables, lens)])
    before = [gathered(pool, t, n) for t, n in zip(tables, lens)]
    _, new = tree_step(model, device, list(zip(tables, lens)))
    assert all(n > o + 2 for n, o in zip(new, lens))
    for t, n, o, was in zip(tables, new, lens, before):
        now = gathered(pool, t, n)
        np.testing.assert_array_equal(now[:, :, :o], was)
        assert (now[:, :, o:] == 0).all()
    cells = pool.scores.clone()
    after = []
    for counted in (new, lens):
        pool.scores.copy_(cells)
        step(model, device, [(t, n + 1, s) for t, n, s in zip(tables, new, counted)])
        after.append([gathered(pool, t, n + 1) for t, n in zip(tables, new)])
    for with_them, without, was, o in zip(*after, before, lens):
        np.testing.assert_array_equal(with_them, without)
        added = with_them.copy()
        added[:, :, :o] -= was
        np.testing.assert_allclose(added.sum(-1), GROUP, atol=SLACK)
    budget, recent = 30, 4
    kept = torch.empty((2, 2, 2, budget), dtype=torch.int32, device=device)
    table = torch.tensor(tables, dtype=torch.int32, device=device)
    pool.evict(table, torch.tensor([n + 1 for n in new], dtype=torch.int32, device=device), budget, recent, 2, None, kept)
    for layer in range(2):
        for s in range(2):
            for h in range(2):
                want = keep_positions(after[1][s][layer, h], budget, recent, 2)
                np.testing.assert_array_equal(kept[layer, s, h].cpu().numpy(), want)


def test_a_step_without_a_tree_clears_nothing(device, kernels):
    model, pool = small_model(device, kernels)
    prefill(model, device, [[20, 21, 22]], [40])
    assert pool._scores is None
    tree_step(model, device, [([20, 21, 22, 23], 40)])
    assert pool._scores is None                                        # nobody asked for scores
    pool.scores.fill_(7.0)
    model.forward(DeviceStep.from_host(pack_step([], [DecodeSlot(1, 41, [20, 21, 22])], BS), device))
    assert (pool.scores == 7).all()
    tree_step(model, device, [([20, 21, 22, 23], 40)])
    t = np.arange(40, 40 + len(PARENTS))
    cleared = torch.zeros_like(pool.scores, dtype=torch.bool)
    cleared[:, np.asarray([20, 21, 22, 23])[t // BS], :, t % BS] = True
    assert (pool.scores[cleared] == 0).all() and (pool.scores[~cleared] == 7).all()


def test_captured(device, kernels):
    """A replayed tree step clears its tokens' cells each time; a tree that a replay's lengths leave without a slot
    touches no cell."""
    model, pool = small_model(device, kernels)
    tables, lens = [[20, 21, 22, 23], [30, 31, 32, 33]], [40, 33]
    prefill(model, device, tables, lens)
    pool.scores.fill_(7.0)
    st, _ = tree_step(model, device, list(zip(tables, lens)))
    first = DeviceStep.from_host(st.host, device)
    model.forward(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.forward(first)
    whole = first.context_lens.clone()
    for shorter in (False, True, False):
        pool.scores.fill_(7.0)
        first.context_lens.copy_(whole)
        if shorter:
            first.context_lens[1] = 0
        graph.replay()
        torch.cuda.synchronize()
        for i, (t, n) in enumerate(zip(tables, lens)):
            got = gathered(pool, t, n + len(PARENTS))
            assert (got[:, :, :n] == 7).all() and (got[:, :, n:] == (7 if shorter and i == 1 else 0)).all()
        touched = int((pool.scores != 7).sum())
        assert touched == 2 * 2 * len(PARENTS) * (1 if shorter else 2)
        torch.cuda.synchronize()
        tree_step(model, device, list(zip(tables, lens)))
