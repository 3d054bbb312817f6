"""Shared-prefix decode, gathered scores and eviction run together, as a long chat uses them.

Rows that begin with the same blocks decode for some steps while their attention weights are gathered,
are trimmed to a budget (the shared prefix protected), and decode on over the trimmed caches: on the
op's entry points against 64 bits, and through the model against the CPU model.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from attention64 import HALF_STEP, assert_within, attention64
from helpers import TORCH_DT, dev_f32, i32
from oracle import llama_ref
from railgun_amd.batch import DecodeSlot, PrefillChunk, pack_step
from railgun_amd.kv_pool import GpuBlockPool
from railgun_amd.llama import DeviceStep, LlamaConfig, LlamaWeights, RailgunLlama
from railgun_amd.ops import PagedAttentionOp
from test_gpu_evict import keep_positions

pytestmark = pytest.mark.gpu
LAYERS, BS = 2, 16


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype,heads,hkv,d", [("bf16", 8, 2, 128), ("f16", 7, 1, 64), ("f32", 8, 2, 64),
                                               ("bf16", 4, 4, 96)])
def test_decode_score_evict_decode(device, kernels, dtype, heads, hkv, d, in_place):
    shared, budget, recent, steps = 33, 600, 24, 3
    first = shared * BS
    start = np.asarray([first, first + 1, 700, 590, 1100, 641])        # cached tokens before the first step
    b = len(start)
    need = -(-(start + 2 * steps) // BS) - shared
    rng = np.random.default_rng(d)
    total = shared + int(need.sum()) + b * (budget // BS + 1 - shared + 1)
    order = iter(rng.permutation(total).astype(np.int32))
    prefix = [next(order) for _ in range(shared)]
    rows = [prefix + [next(order) for _ in range(int(n))] for n in need]
    table = np.zeros((b, max(map(len, rows))), np.int32)
    for s, r in enumerate(rows):
        table[s, :len(r)] = r
    pool = GpuBlockPool(LAYERS, total, hkv, BS, d, device, dtype=TORCH_DT[dtype])
    g = torch.Generator(device=device).manual_seed(d)
    pool.storage.copy_(torch.randn(pool.storage.shape, generator=g, device=device))
    pool.scores.fill_(7.0)                                             # left over from earlier owners
    op = PagedAttentionOp(1 / math.sqrt(d), heads, hkv, d, BS, kernels)
    lens, scored = start.copy(), np.full(b, 0)
    expected = [[np.zeros((hkv, 0)) for _ in range(b)] for _ in range(LAYERS)]
    slack = [[np.zeros((hkv, 0)) for _ in range(b)] for _ in range(LAYERS)]

    def step():
        nonlocal lens, scored
        slots = torch.as_tensor([table[s, n // BS] * BS + n % BS for s, n in enumerate(lens)], device=device,
                                dtype=torch.int32)
        lens = lens + 1
        for layer in range(LAYERS):
            kc, vc = pool.k_cache(layer), pool.v_cache(layer)
            k, v = (torch.randn((b, hkv, d), generator=g, device=device).to(pool.storage.dtype) for _ in range(2))
            op.reshape_and_cache(k, v, kc, vc, slots, None, False)
            q = (2 * torch.randn((b, heads, d), generator=g, device=device)).to(pool.storage.dtype)
            dt, dl = i32(table, device), i32(lens, device)
            out = op.execute_with_scores(q, kc, vc, dt, dl, pool.scores[layer], i32(scored, device), first)
            alike = op.execute_shared_prefix(q, kc, vc, dt, dl, shared)
            want, tol, weights, wtol = attention64(q, kc, vc, table, lens, op.scale, dtype)
            assert_within(dev_f32(out), want, tol, "with scores")
            want, tol, _, _ = attention64(q, kc, vc, table, lens, op.scale, dtype, rounded_p=True)
            assert_within(dev_f32(alike), want, tol, "shared prefix")
            for s in range(b):
                n = lens[s] - first
                grown = np.zeros((hkv, n)), np.zeros((hkv, n))
                for old, new in zip((expected[layer][s], slack[layer][s]), grown):
                    new[:, :old.shape[1]] = old
                expected[layer][s] = grown[0] + weights[s][:, first:]
                slack[layer][s] = grown[1] + wtol[s][:, first:] + HALF_STEP["f32"] * expected[layer][s]
        scored = lens.copy()
        check_scores()

    def gathered(layer, s):
        t = np.arange(first, lens[s])
        return pool.scores[layer].cpu().numpy()[table[s, t // BS], :, t % BS].T

    def check_scores():
        for layer in range(LAYERS):
            for s in range(b):
                assert_within(gathered(layer, s), expected[layer][s], slack[layer][s] + 1e-37, f"scores {layer} {s}")
            prefix_scores = pool.scores[layer][torch.as_tensor(prefix, device=device).long()]
            assert (prefix_scores == 7.0).all()

    for _ in range(steps):
        step()
    # Trim; what stays follows from the gathered scores exactly.
    before = pool.storage.clone()
    dst = None
    if not in_place:
        fresh = np.zeros((b, -(-(budget + steps) // BS)), np.int32)
        for s in range(b):
            fresh[s, :shared] = prefix
            for i in range(shared, fresh.shape[1]):
                fresh[s, i] = next(order)
        dst = fresh
    kept = torch.empty((LAYERS, b, hkv, budget), device=device, dtype=torch.int32)
    want_kept = [[[np.concatenate([np.arange(first), first + rel]) for rel in
                   (keep_positions(gathered(layer, s)[h], budget - first, recent, 0) for h in range(hkv))]
                  for s in range(b)] for layer in range(LAYERS)]
    new_lens = pool.evict(i32(table, device), i32(lens, device), budget, recent, first,
                          None if dst is None else i32(dst, device), kept)
    new_lens = new_lens.cpu().numpy()
    np.testing.assert_array_equal(new_lens, np.minimum(lens, budget))
    kept = kept.cpu().numpy()
    to = table if dst is None else dst
    for layer in range(LAYERS):
        for s in range(b):
            n = int(new_lens[s])
            for h in range(hkv):
                p = want_kept[layer][s][h]
                np.testing.assert_array_equal(kept[layer, s, h, :n], p)
                j = np.arange(n)
                assert torch.equal(pool.storage[layer, to[s, j // BS].astype(np.int64), :, h, j % BS],
                                   before[layer, table[s, p // BS].astype(np.int64), :, h, p % BS])
            keep = [want_kept[layer][s][h][first:] - first for h in range(hkv)]
            expected[layer][s] = np.stack([expected[layer][s][h][keep[h]] for h in range(hkv)])
            slack[layer][s] = np.stack([slack[layer][s][h][keep[h]] for h in range(hkv)])
    table, lens, scored = to, new_lens.astype(np.int64), new_lens.astype(np.int64)
    for _ in range(steps):
        step()


def test_two_streams_at_once(device, kernels):
    """A shared-prefix decode and a scored decode of one pool, and an eviction of another, on streams of their
    own: the results of the calls one after the other, bit for bit."""
    g = torch.Generator(device=device).manual_seed(4)
    b, shared, hkv, heads, d = 24, 40, 2, 8, 128
    table = np.zeros((b, 80), np.int32)
    order = iter(np.random.default_rng(4).permutation(40 + 40 * b).astype(np.int32))
    table[:, :shared] = [next(order) for _ in range(shared)]
    for s in range(b):
        table[s, shared:] = [next(order) for _ in range(40)]
    lens = np.random.default_rng(5).integers(640, 1280, b)
    pool, other = (GpuBlockPool(1, 40 + 40 * b, hkv, BS, d, device) for _ in range(2))
    for x in (pool, other):
        x.storage.copy_(torch.randn(x.storage.shape, generator=g, device=device))
        x.scores.copy_(torch.rand(x.scores.shape, generator=g, device=device))
    q = torch.randn((b, heads, d), generator=g, device=device).to(torch.bfloat16)
    op = PagedAttentionOp(1 / math.sqrt(d), heads, hkv, d, BS, kernels)
    dt, dl = i32(table, device), i32(lens, device)
    kc, vc = pool.k_cache(0), pool.v_cache(0)
    shape = (b, heads, hkv, d, BS, 80)
    start = pool.scores.clone(), other.storage.clone(), other.scores.clone()

    def prefix():
        out = torch.empty_like(q)
        ws = torch.empty(kernels.shared_prefix_workspace_bytes(*shape, shared), dtype=torch.uint8, device=device)
        kernels.launch_shared_prefix(q, kc, vc, dt, dl, out, op.scale, *shape[1:], b, shared, ws)
        return out

    calls = [prefix, lambda: op.execute_with_scores(q, kc, vc, dt, dl, pool.scores[0], None, shared * BS),
             lambda: other.evict(dt, dl, 800, 100, shared * BS)]

    def reset():
        pool.scores.copy_(start[0])
        other.storage.copy_(start[1])
        other.scores.copy_(start[2])
        torch.cuda.synchronize()

    def results(outs):
        torch.cuda.synchronize()
        return [x.clone() for x in (*outs, pool.scores, other.storage, other.scores)]

    reset()
    want = results([f() for f in calls])
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        reset()
        outs = []
        for f, st in zip(calls, streams):
            with torch.cuda.stream(st):
                outs.append(f())
        for got, w in zip(results(outs), want):
            assert torch.equal(got, w)


class _EvictedReference(llama_ref.ReferenceLlama):
    """The CPU model where a decode token sees all cached tokens, fewer than its position says."""

    @staticmethod
    def keys_seen(pos, ctx):
        return min(pos + 1, ctx)

    def evict(self, tables, lens, kept, new_lens):
        bs = self.block_size
        for layer, (kc, vc) in enumerate(zip(self.k, self.v)):
            for cache in (kc, vc):
                old = cache.clone()
                for s, t in enumerate(tables):
                    t = np.asarray(t, np.int64)
                    for h in range(cache.shape[1]):
                        j = np.arange(new_lens[s])
                        p = kept[layer, s, h, :new_lens[s]]
                        cache[t[j // bs], h, j % bs] = old[t[p // bs], h, p % bs]


@pytest.mark.parametrize("kv_heads,hidden,dtype", [(2, 512, torch.bfloat16), (1, 512, torch.float16)])
def test_model_steps(device, kernels, kv_heads, hidden, dtype):
    """Prefill of a common prompt and of every row's own, scored decode steps, shared-prefix decode steps,
    eviction and both kinds of decode again.  The logits stay within twice the drift that rounding the
    activations explains, as the model's other steps do (plus 1e-3)."""
    cfg = LlamaConfig(hidden_size=hidden, intermediate_size=2 * hidden, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=kv_heads, vocab_size=500)
    bs, nb, shared = 16, 700, 64
    g = torch.Generator().manual_seed(3)

    def normal(*shape, sd=0.06):
        return (sd * torch.randn(shape, generator=g)).to(dtype).float()

    D = cfg.head_dim
    sd = {"model.embed_tokens.weight": normal(cfg.vocab_size, hidden, sd=1.0),
          "model.norm.weight": 1 + normal(hidden), "lm_head.weight": normal(cfg.vocab_size, hidden)}
    for i in range(cfg.num_hidden_layers):
        p = f"model.layers.{i}."
        sd[p + "input_layernorm.weight"] = (1 + normal(hidden)).to(dtype).float()
        sd[p + "post_attention_layernorm.weight"] = (1 + normal(hidden)).to(dtype).float()
        for name, rows in (("q", 8 * D), ("k", kv_heads * D), ("v", kv_heads * D)):
            sd[p + f"self_attn.{name}_proj.weight"] = normal(rows, hidden)
        sd[p + "self_attn.o_proj.weight"] = normal(hidden, 8 * D)
        sd[p + "mlp.gate_proj.weight"] = normal(2 * hidden, hidden)
        sd[p + "mlp.up_proj.weight"] = normal(2 * hidden, hidden)
        sd[p + "mlp.down_proj.weight"] = normal(hidden, 2 * hidden)
    sd["model.norm.weight"] = sd["model.norm.weight"].to(dtype).float()
    pool = GpuBlockPool.for_model(cfg, nb, bs, device, dtype=dtype)
    model = RailgunLlama(cfg, LlamaWeights.from_state_dict(cfg, sd, device, dtype=dtype), pool, kernels,
                         max_position=4096)
    refs = [_EvictedReference(cfg, sd, nb, bs, act_dtype=t) for t in (torch.float32, dtype)]
    rng = np.random.default_rng(5)
    order = iter(rng.permutation(nb).tolist())
    prefix = [next(order) for _ in range(shared)]
    own = [10, 30, 77, 1, 120, 64, 33, 50, 95, 18, 111, 40]            # tokens behind the common ones
    tables = [prefix + [next(order) for _ in range(-(-(n + 12) // bs))] for n in own]
    lens = [shared * bs + n for n in own]
    position = list(lens)
    used = []
    real = model.kernels.launch_shared_prefix

    def run(step, what):
        got = model.forward(DeviceStep.from_host(step, device)).float().cpu()
        ref32, ref16 = (r.forward(step) for r in refs)
        drift = float((ref16 - ref32).abs().max())
        err = float((got - ref32).abs().max())
        assert err <= 2 * drift + 1e-3, f"{what}: |gpu - fp32 oracle| {err:.4g} vs drift {drift:.4g}"

    def decode(what, scored=None):
        rows = [DecodeSlot(int(rng.integers(cfg.vocab_size)), n + 1, t, position=p,
                           scored_len=None if scored is None else (n if scored else 0))
                for n, t, p in zip(lens, tables, position)]
        run(pack_step([], rows, bs, share_prefix=True, gather_scores=scored is not None), what)
        for s in range(len(lens)):
            lens[s] += 1
            position[s] += 1

    text = rng.integers(cfg.vocab_size, size=shared * bs).tolist()
    run(pack_step([PrefillChunk(text, 0, prefix)], [], bs), "common prompt")
    run(pack_step([PrefillChunk(rng.integers(cfg.vocab_size, size=n).tolist(), shared * bs, t)
                   for n, t in zip(own, tables)], [], bs), "own prompts")
    model.kernels.launch_shared_prefix = lambda *a: (used.append(1), real(*a))[1]
    try:
        decode("plain")                                    # too small to pay
        assert not used
        model.kernels.shared_prefix_pays = lambda *a: True
        decode("shared prefix")
        assert len(used) == cfg.num_hidden_layers
        decode("first scored", scored=False)
        decode("scored", scored=True)
        assert len(used) == cfg.num_hidden_layers
        budget, recent = shared * bs + 40, 8
        table = np.zeros((len(tables), max(map(len, tables))), np.int32)
        for s, t in enumerate(tables):
            table[s, :len(t)] = t
        kept = torch.empty((cfg.num_hidden_layers, len(lens), kv_heads, budget), device=device, dtype=torch.int32)
        new = pool.evict(i32(table, device), i32(lens, device), budget, recent, shared * bs, None, kept).tolist()
        assert new == [min(n, budget) for n in lens] and any(n < o for n, o in zip(new, lens))
        for r in refs:
            r.evict(tables, lens, kept.cpu().numpy(), new)
        lens[:] = new
        decode("after eviction")
        assert len(used) == 2 * cfg.num_hidden_layers
    finally:
        del model.kernels.launch_shared_prefix, model.kernels.shared_prefix_pays
    decode("scored after eviction", scored=False)


def test_scores_are_not_made_in_a_capture(device):
    pool = GpuBlockPool(1, 4, 2, 16, 64, device)
    x = torch.zeros(4, device=device)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x += 1
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="before it"):
            pool.scores
    assert pool.scores.shape == (1, 4, 2, 16)
