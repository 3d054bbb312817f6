"""Model steps over drafted tokens: the four operators as a serving loop uses them, one after the other."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from helpers import i32
from oracle import llama_ref
from railgun_amd.batch import DecodeSlot, DraftTree, PrefillChunk, pack_step
from railgun_amd.kv_pool import GpuBlockPool
from railgun_amd.llama import DeviceStep, LlamaConfig, LlamaWeights, RailgunLlama
from tree64 import accept, ancestors, first_largest, random_tree

pytestmark = pytest.mark.gpu
BS = 16


class TreeReference(llama_ref.ReferenceLlama):
    """The CPU model, whose attention also takes the rows of draft trees."""

    def attention(self, layer, q, k, v, batch):
        out = super().attention(layer, q, k, v, batch)
        cfg, first = self.cfg, batch.first_tree_row
        group, scale = cfg.num_attention_heads // cfg.num_key_value_heads, 1 / math.sqrt(cfg.head_dim)
        for s in range(batch.num_trees):
            a, e = (int(x) for x in batch.tree_cu[s:s + 2])
            r = batch.num_requests - batch.num_trees + s
            n = int(batch.context_lens[r])
            blocks = torch.as_tensor(batch.block_table[r, :-(-n // BS)].astype("int64"))
            keys, vals = (c[blocks].permute(1, 0, 2, 3).flatten(1, 2)[:, :n] for c in (self.k[layer], self.v[layer]))
            sees = np.concatenate([np.ones((e - a, n - e + a), bool), ancestors(batch.tree_parents[a:e].tolist())], 1)
            hides = torch.as_tensor(~sees)
            for h in range(cfg.num_attention_heads):
                x = (q[first + a:first + e, h] @ keys[h // group].T * scale).masked_fill(hides, -math.inf)
                out[first + a:first + e, h] = torch.softmax(x, 1) @ vals[h // group]
        return out

    def keep(self, table, prior, path):
        t = np.asarray(table, np.int64)
        src, dst = prior + np.asarray(path), prior + np.arange(len(path))
        for cache in (*self.k, *self.v):
            cache[t[dst // BS], :, dst % BS] = cache[t[src // BS], :, src % BS].clone()


def make(device, kernels, dtype, kv_heads=2, hidden=512, vocab=500, nb=300, seed=3):
    cfg = LlamaConfig(hidden_size=hidden, intermediate_size=2 * hidden, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=kv_heads, vocab_size=vocab)
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, sd=0.06):
        return (sd * torch.randn(shape, generator=g)).to(dtype).float()

    d = cfg.head_dim
    sd = {"model.embed_tokens.weight": normal(vocab, hidden, sd=1.0), "lm_head.weight": normal(vocab, hidden),
          "model.norm.weight": (1 + normal(hidden)).to(dtype).float()}
    for i in range(cfg.num_hidden_layers):
        p = f"model.layers.{i}."
        for name in ("input_layernorm", "post_attention_layernorm"):
            sd[p + name + ".weight"] = (1 + normal(hidden)).to(dtype).float()
        for name, rows in (("q", 8 * d), ("k", kv_heads * d), ("v", kv_heads * d)):
            sd[p + f"self_attn.{name}_proj.weight"] = normal(rows, hidden)
        sd[p + "self_attn.o_proj.weight"] = normal(hidden, 8 * d)
        sd[p + "mlp.gate_proj.weight"], sd[p + "mlp.up_proj.weight"] = normal(2 * hidden, hidden), normal(2 * hidden, hidden)
        sd[p + "mlp.down_proj.weight"] = normal(hidden, 2 * hidden)
    pool = GpuBlockPool.for_model(cfg, nb, BS, device, dtype=dtype)
    model = RailgunLlama(cfg, LlamaWeights.from_state_dict(cfg, sd, device, dtype=dtype), pool, kernels, max_position=4096)
    return cfg, sd, model


@pytest.mark.parametrize("kv_heads,hidden,dtype", [(2, 512, torch.bfloat16), (1, 1024, torch.float16)])
def test_steps(device, kernels, kv_heads, hidden, dtype):
    """Prefill, a step of trees beside a prefill chunk and decode rows, verification, compaction, and the steps behind
    them.  The logits stay within twice the drift that rounding the activations explains (plus 1e-3), the verdict is
    that of the model's own logits, the cached tokens are the accepted ones to the bit."""
    cfg, sd, model = make(device, kernels, dtype, kv_heads, hidden)
    refs = [TreeReference(cfg, sd, model.pool.num_blocks, BS, act_dtype=t) for t in (torch.float32, dtype)]
    rng = np.random.default_rng(6)
    order = iter(rng.permutation(model.pool.num_blocks).tolist())
    lens = [70, 5, 33, 130, 1, 64]
    tables = [[next(order) for _ in range(-(-(n + 120) // BS))] for n in lens]
    scores = model.pool.scores
    scores.copy_(torch.rand(scores.shape, generator=torch.Generator(device).manual_seed(1), device=device))

    def run(step, what):
        st = DeviceStep.from_host(step, device)
        logits = model.forward(st)
        ref32, ref16 = (r.forward(step) for r in refs)
        drift, err = float((ref16 - ref32).abs().max()), float((logits.float().cpu() - ref32).abs().max())
        assert logits.shape == ref32.shape and err <= 2 * drift + 1e-3, f"{what}: {err:.4g} against a drift of {drift:.4g}"
        return st, logits

    text = [rng.integers(cfg.vocab_size, size=n).tolist() for n in lens]
    run(pack_step([PrefillChunk(t, 0, table) for t, table in zip(text, tables)], [], BS), "prompts")
    more = [next(order) for _ in range(3)]
    sizes = [40, 1, 64, 17]                                          # trees of the first four; the others decode
    trees = [random_tree(rng, n, 7) for n in sizes]
    draft = [rng.integers(0, 4, n).tolist() for n in sizes]

    def tree_step(*beside):
        return pack_step(*beside, BS, draft_trees=[DraftTree(d, t, lens[s] + len(t), tables[s])
                                                   for s, (d, t) in enumerate(zip(draft, trees))])

    beside = ([PrefillChunk([5, 6, 7], 0, more)], [DecodeSlot(3, lens[s] + 1, tables[s]) for s in (4, 5)])
    st, logits = run(tree_step(*beside), "trees")
    # Drafts that the model agrees with here and there, told by its own logits for the tokens above them.
    cu = st.host.tree_cu
    for _ in range(7):
        target = [first_largest(row) for row in logits[3:].float().cpu().numpy()]
        for s, t in enumerate(trees):
            for j, p in enumerate(t):
                if p >= 0 and j % 3:
                    draft[s][j] = target[cu[s] + p]
        st, logits = run(tree_step(*beside), "trees again")
    target = [first_largest(row) for row in logits[3:].float().cpu().numpy()]
    verdict = model.verify_trees(logits, st)
    paths = []
    for s, t in enumerate(trees):
        path, following = accept(t, draft[s], target[cu[s]:cu[s + 1]], st.host.max_tree_depth)
        paths.append(path)
        assert verdict.accepted[s].tolist() == path + [-1] * (st.host.max_tree_depth - len(path))
        assert int(verdict.num_accepted[s]) == len(path) and int(verdict.next_tokens[s]) == following
    assert verdict.target_tokens.tolist() == target and max(map(len, paths)) > 2
    again = model.verify_trees(logits, st, verdict.target_tokens)
    assert torch.equal(again.accepted, verdict.accepted) and torch.equal(again.next_tokens, verdict.next_tokens)
    before, cells = model.pool.storage.clone(), scores.clone()
    new = model.keep_accepted(st, verdict).tolist()
    for s, path in enumerate(paths):
        table = np.asarray(tables[s])
        src, dst = lens[s] + np.asarray(path), lens[s] + np.arange(len(path))
        before[:, table[dst // BS], :, :, dst % BS] = before[:, table[src // BS], :, :, src % BS].clone()
        cells[:, table[dst // BS], :, dst % BS] = cells[:, table[src // BS], :, src % BS].clone()
        for r in refs:
            r.keep(tables[s], lens[s], path)
        assert new[s] == lens[s] + len(path)
        lens[s] = new[s]
    assert torch.equal(model.pool.storage, before) and torch.equal(scores, cells)
    lens[4] += 1
    lens[5] += 1
    following = verdict.next_tokens.tolist() + [1, 2]
    run(pack_step([], [DecodeSlot(t, n + 1, table) for t, n, table in zip(following, lens, tables)], BS), "decode behind")
    for s in range(6):
        lens[s] += 1
    trees = [random_tree(rng, n, 4) for n in (9, 30)]
    draft = [rng.integers(0, cfg.vocab_size, len(t)).tolist() for t in trees]
    run(pack_step([], [], BS, draft_trees=[DraftTree(d, t, lens[s] + len(t), tables[s])
                                           for s, (d, t) in enumerate(zip(draft, trees))]), "trees behind")


def test_generates_what_greedy_decoding_does(device, kernels):
    """In fp32: many tokens a step through trees whose drafts are partly right, against one token a step on the
    CPU, as long as no two logits of the latter are within 1e-3 of each other."""
    cfg, sd, model = make(device, kernels, torch.float32, nb=60)
    ref = llama_ref.ReferenceLlama(cfg, sd, 60, BS)
    rng = np.random.default_rng(1)
    prompt, table = rng.integers(cfg.vocab_size, size=21).tolist(), list(range(20))
    truth, clear, logits = [], 0, ref.forward(pack_step([PrefillChunk(prompt, 0, table)], [], BS))
    for i in range(40):
        top = torch.topk(logits[0], 2).values
        clear += int(clear == i and float(top[0] - top[1]) > 1e-3)
        truth.append(int(logits[0].argmax()))
        logits = ref.forward(pack_step([], [DecodeSlot(truth[-1], len(prompt) + i + 1, table)], BS))
    assert clear >= 20
    gpu_table = [25 + i for i in range(20)]
    logits = model.forward(DeviceStep.from_host(pack_step([PrefillChunk(prompt, 0, gpu_table)], [], BS), device))
    out, n, steps = [int(logits[0].argmax())], len(prompt), 0
    while len(out) < clear:
        # A tree whose path to node 7 is right up to a place that differs from step to step.
        parents = [-1, 0, 0, 2, 2, 4, 4, 6]
        tokens = [out[-1]] + [int(x) for x in rng.integers(cfg.vocab_size, size=7)]
        for i, j in enumerate((2, 4, 6, 7)):
            if i < steps % 5 and len(out) + i < len(truth):
                tokens[j] = truth[len(out) + i]
        st = DeviceStep.from_host(pack_step([], [], BS, draft_trees=[DraftTree(tokens, parents, n + 8, gpu_table)]), device)
        verdict = model.verify_trees(model.forward(st), st)
        n = int(model.keep_accepted(st, verdict)[0])
        path = [j for j in verdict.accepted[0].tolist() if j >= 0]
        out += [tokens[j] for j in path[1:]] + [int(verdict.next_tokens[0])]
        assert n == len(prompt) + len(out) - 1
        steps += 1
    assert out[:clear] == truth[:clear] and steps < clear


def test_captured_step(device, kernels):
    """Layout, model, verification and compaction in one graph, replayed on other trees; a decode step captured before
    it, on the model's own workspace, still gives its results."""
    cfg, _, model = make(device, kernels, torch.bfloat16)
    rng = np.random.default_rng(2)
    tables = [list(range(20 * s, 20 * s + 20)) for s in range(3)]
    lens = [100, 37, 250]
    prompts = [PrefillChunk(rng.integers(cfg.vocab_size, size=n).tolist(), 0, t) for n, t in zip(lens, tables)]
    model.forward(DeviceStep.from_host(pack_step(prompts, [], BS), device))
    filled = model.pool.storage.clone()
    decode = DeviceStep.from_host(pack_step([], [DecodeSlot(4, n + 1, t) for n, t in zip(lens, tables)], BS), device)
    model.forward(decode)
    g0 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g0):
        plain = model.forward(decode)
    g0.replay()
    torch.cuda.synchronize()
    want_plain = plain.clone()
    trees = [random_tree(rng, n, 5) for n in (20, 6, 33)]
    st = DeviceStep.from_host(pack_step([], [], BS, draft_trees=[
        DraftTree(rng.integers(cfg.vocab_size, size=len(t)).tolist(), t, n + len(t), table)
        for t, n, table in zip(trees, lens, tables)]), device)

    def step():
        logits = model.forward(st)
        verdict = model.verify_trees(logits, st)
        return logits, verdict.accepted, verdict.next_tokens, model.keep_accepted(st, verdict)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for seed in range(3):
        r = np.random.default_rng(seed)
        st.tree_parents.copy_(i32(sum((random_tree(r, len(t), 5) for t in trees), []), device))
        st.draft_tokens.copy_(i32(r.integers(0, 5, 59), device))
        st.tokens.copy_(st.draft_tokens)
        model.pool.storage.copy_(filled)
        g.replay()
        torch.cuda.synchronize()
        got, pool = [t.clone() for t in outs], model.pool.storage.clone()
        model.pool.storage.copy_(filled)
        assert all(torch.equal(a, b) for a, b in zip(got, step())) and torch.equal(pool, model.pool.storage)
        model.pool.storage.copy_(filled)
        g0.replay()
        torch.cuda.synchronize()
        assert torch.equal(plain, want_plain)
