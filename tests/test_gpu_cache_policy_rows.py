"""Model steps that gather attention weights while the rows of the batch change."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from railgun_amd.batch import DecodeSlot, PrefillChunk, pack_step
from railgun_amd.kv_pool import GpuBlockPool
from railgun_amd.llama import DeviceStep, LlamaConfig, LlamaWeights, RailgunLlama

pytestmark = pytest.mark.gpu

BS = 16
CFG = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=8,
                  num_key_value_heads=2, vocab_size=300)
GROUP = CFG.num_attention_heads // CFG.num_key_value_heads


def small_model(device, kernels, blocks=64, dtype=torch.bfloat16, seed=3):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, sd=0.08):
        return sd * torch.randn(shape, generator=g)

    hid, inter, d = CFG.hidden_size, CFG.intermediate_size, CFG.head_dim
    sd = {"model.embed_tokens.weight": normal(CFG.vocab_size, hid, sd=1.0), "model.norm.weight": 1 + normal(hid),
          "lm_head.weight": normal(CFG.vocab_size, hid)}
    for i in range(CFG.num_hidden_layers):
        p = f"model.layers.{i}."
        sd[p + "input_layernorm.weight"] = 1 + normal(hid)
        sd[p + "post_attention_layernorm.weight"] = 1 + normal(hid)
        for name, rows in (("q", CFG.num_attention_heads * d), ("k", CFG.num_key_value_heads * d),
                           ("v", CFG.num_key_value_heads * d)):
            sd[p + f"self_attn.{name}_proj.weight"] = normal(rows, hid)
        sd[p + "self_attn.o_proj.weight"] = normal(hid, CFG.num_attention_heads * d)
        sd[p + "mlp.gate_proj.weight"] = normal(inter, hid)
        sd[p + "mlp.up_proj.weight"] = normal(inter, hid)
        sd[p + "mlp.down_proj.weight"] = normal(hid, inter)
    sd = {k: v.bfloat16().float() for k, v in sd.items()}  # (in float16 the same but for the smallest)
    pool = GpuBlockPool.for_model(CFG, blocks, BS, device, dtype=dtype)
    model = RailgunLlama(CFG, LlamaWeights.from_state_dict(CFG, sd, device, dtype=dtype), pool, kernels,
                         max_position=2048, choices="rg")
    return model, pool


def prefill(model, device, tables, lens, seed=0):
    rng = np.random.default_rng(seed)
    chunks = [PrefillChunk(rng.integers(CFG.vocab_size, size=n).tolist(), 0, t) for n, t in zip(lens, tables)]
    model.forward(DeviceStep.from_host(pack_step(chunks, [], BS), device))


def gathered(pool, table, n):
    """float64 [layers, H_kv, n]: the scores of a row's tokens."""
    t = np.arange(n)
    s = pool.scores.cpu().numpy().astype(np.float64)
    return s[:, np.asarray(table)[t // BS], :, t % BS].transpose(1, 2, 0)


def step(model, device, rows):
    st = pack_step([], [DecodeSlot(7 + i, n, t, scored_len=s) for i, (t, n, s) in enumerate(rows)], BS,
                   share_prefix=True, gather_scores=True)
    dev = DeviceStep.from_host(st, device)
    model.forward(dev)
    return dev


# A step gives each kv-head of a row its group's weights, which sum to the group's size: fp32 weights of
# relative error some 2^-13 at most at these lengths (128 steps of 2^-23 in a score of magnitude 10, twice).
SLACK = GROUP * 2.0 ** -12


def test_a_row_that_outlives_the_others_of_its_prefix(device, kernels):
    """Two rows over eight common blocks gather, one leaves, the other goes on alone: its cells hold the weights
    of its own steps, whatever the blocks held before, and eviction goes by those."""
    model, pool = small_model(device, kernels)
    prefix = list(range(20, 28))
    a, b = prefix + [1, 2], prefix + [5, 6]
    start = 8 * BS + 9
    prefill(model, device, [a], [start])
    prefill(model, device, [b], [start])
    pool.scores.fill_(float("nan"))
    n = start
    for i in range(3):
        n += 1
        step(model, device, [(a, n, 0 if i == 0 else n - 1), (b, n, 0 if i == 0 else n - 1)])
    own = gathered(pool, a, n)
    assert np.isfinite(own).all() and (own[:, :, :8 * BS] == 0).all() and (own[:, :, 8 * BS:] > 0).all()
    n += 1
    step(model, device, [(a, n, n - 1)])
    after = gathered(pool, a, n)
    added = after.copy()
    added[:, :, :n - 1] -= own
    assert (after[:, :, :8 * BS] > 0).all()
    np.testing.assert_allclose(added.sum(-1), GROUP, atol=SLACK)
    # What stays is what gathered the most.
    table = torch.tensor([a], dtype=torch.int32, device=device)
    lens = torch.tensor([n], dtype=torch.int32, device=device)
    kept = torch.empty((2, 1, 2, 64), dtype=torch.int32, device=device)
    pool.evict(table, lens, 64, 4, 0, None, kept)
    for layer in range(2):
        for h in range(2):
            best = np.argsort(-after[layer, h, :n - 4], kind="stable")[:60]
            want = np.sort(np.concatenate([best, np.arange(n - 4, n)]))
            np.testing.assert_array_equal(kept[layer, 0, h].cpu().numpy(), want)


def test_a_row_that_joins_shortens_the_prefix(device, kernels):
    model, pool = small_model(device, kernels)
    a, b, c = [20, 21, 22, 1, 2], [20, 21, 22, 5, 6], [20, 30, 31, 8, 9]
    prefill(model, device, [a], [60])
    prefill(model, device, [b], [60])
    prefill(model, device, [c], [70])
    pool.scores.fill_(float("nan"))
    step(model, device, [(a, 61, 0), (b, 61, 0)])
    old = gathered(pool, a, 61)
    step(model, device, [(a, 62, 61), (c, 71, 0)])
    new, other = gathered(pool, a, 62), gathered(pool, c, 71)
    new[:, :, :61] -= old
    assert (new[:, :, :BS] == 0).all() and (new[:, :, BS:] > 0).all()
    assert (other[:, :, :BS] == 0).all() and (other[:, :, BS:] > 0).all()


def test_a_captured_step_clears_the_same_cells_each_time(device, kernels):
    """Captured with a prefix that no row counts, replayed with eager steps between."""
    model, pool = small_model(device, kernels)
    a, b = [20, 21, 1, 2], [20, 21, 5, 6]
    prefill(model, device, [a], [40])
    prefill(model, device, [b], [40])
    pool.scores.fill_(float("nan"))
    dev = step(model, device, [(a, 41, 0), (b, 41, 0)])
    want = gathered(pool, a, 41), gathered(pool, b, 41)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.forward(dev)
    for _ in range(3):
        pool.scores.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip((a, b), want):
            np.testing.assert_array_equal(gathered(pool, t, 41), w)
        step(model, device, [(a, 41, 0), (b, 41, 0)])


def test_the_next_prompt_of_a_trimmed_chat(device, kernels):
    """A chunk behind an evicted cache, at its place in the text: the logits of the same tokens fed one at a
    time as decode steps, whose positions are given too.  Both round their activations to bf16 in an order of
    their own, so they differ by the drift of that rounding: measured here as the difference between those
    decode steps and the same ones in float16, which rounds eight times finer (twice it, plus 1e-3)."""
    n, budget, text = 150, 64, 150
    table = list(range(30, 42))
    tokens = np.random.default_rng(1).integers(CFG.vocab_size, size=9).tolist()

    def trimmed(dtype):
        model, pool = small_model(device, kernels, dtype=dtype)
        prefill(model, device, [table], [n])
        pool.scores.copy_(torch.rand(pool.scores.shape, generator=torch.Generator().manual_seed(1)))
        lens = pool.evict(torch.tensor([table], dtype=torch.int32, device=device),
                          torch.tensor([n], dtype=torch.int32, device=device), budget, 8, 4)
        assert lens.tolist() == [budget]
        return model

    def forward(model, st):
        return model.forward(DeviceStep.from_host(st, device)).float().cpu()

    def one_at_a_time(dtype):
        model = trimmed(dtype)
        for i, t in enumerate(tokens):
            out = forward(model, pack_step([], [DecodeSlot(t, budget + i + 1, table, position=text + i)], BS))
        return out

    steps = one_at_a_time(torch.bfloat16)
    drift = float((steps - one_at_a_time(torch.float16)).abs().max())
    chunk = forward(trimmed(torch.bfloat16), pack_step([PrefillChunk(tokens, budget, table, position=text)], [], BS))
    assert float((chunk - steps).abs().max()) <= 2 * drift + 1e-3
    wrong = forward(trimmed(torch.bfloat16), pack_step([PrefillChunk(tokens, budget, table)], [], BS))
    assert float((wrong - steps).abs().max()) > 2 * drift + 1e-3
