"""Operators on a paged KV cache that many sequences share or that has outgrown its budget.

A case is a dict of plain values; sequence lengths belong to the case (``lengths`` seeds them), tensor
contents come from the seed given to :func:`prepare`.  Kinds:

``prefix``  one decode step's attention for a batch whose sequences begin with the same cached blocks
            (a system prompt, few-shot examples): those blocks are attended to once for all rows.
``scores``  one decode step's attention that also adds to every cached token's score the softmax weight
            that the step's queries gave it, summed over the query heads of a kv-head.
``evict``   trimming sequences to a budget of tokens in every layer and kv-head: the first ``protected``
            and the last ``recent`` tokens stay, and of the others those with the highest scores; what
            stays is written, in order, to the destination blocks.

Where ``own`` is false, :func:`run` computes the same in elementary torch operations in 32 bits.
"""
from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ELEMENT = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # The reference's element type and CPU-runnable head shape: three short chats under one
        # instruction.  The smallest attention call: launches and latency count.
        dict(name="prefix_f32_small", kind="prefix", dtype="f32", heads=32, kv_heads=8, head_dim=64, block_size=16,
             fused=False, batch=3, shared=96, own_lo=1, own_hi=40, padded=0, lengths=1),
        # An assistant's system prompt and tool descriptions: sixteen chats of an 8B-shaped model.
        dict(name="prefix_chat_b16", kind="prefix", dtype="bf16", heads=32, kv_heads=8, head_dim=128, block_size=16,
             fused=True, batch=16, shared=2048, own_lo=1, own_hi=700, padded=0, lengths=2),
        # An odd batch in fp16 with seven query heads to a kv-head, blocks of 32, over a prefix that
        # ends nowhere special; three rows pad the batch to a captured graph's size.
        dict(name="prefix_f16_gqa7", kind="prefix", dtype="f16", heads=28, kv_heads=4, head_dim=128, block_size=32,
             fused=True, batch=37, shared=4960, own_lo=5, own_hi=900, padded=3, lengths=3),
        # Many short answers to questions about one long document: the largest attention call.
        dict(name="prefix_document_b256", kind="prefix", dtype="bf16", heads=32, kv_heads=8, head_dim=128,
             block_size=16, fused=True, batch=256, shared=16384, own_lo=64, own_hi=1024, padded=0, lengths=4),
        # Two fp32 chats, the first scoring call after their prompts.
        dict(name="scores_f32_small", kind="scores", dtype="f32", heads=32, kv_heads=8, head_dim=64, block_size=16,
             fused=False, batch=2, ctx_lo=9, ctx_hi=77, first=0, scored="none", lengths=5),
        # The headline serving load, one layer: 64 sequences of 512 to 4096 tokens, scored at every step.
        dict(name="scores_b64", kind="scores", dtype="bf16", heads=32, kv_heads=8, head_dim=128, block_size=16,
             fused=True, batch=64, ctx_lo=512, ctx_hi=4096, first=0, scored="step", lengths=6),
        # Long documents whose first blocks are shared and not scored.
        dict(name="scores_long_b4", kind="scores", dtype="bf16", heads=32, kv_heads=8, head_dim=128, block_size=16,
             fused=True, batch=4, ctx_lo=30001, ctx_hi=32768, first=512, scored="step", lengths=7),
        # An odd-sized batch in fp16, seven query heads to a kv-head, blocks of 32, some cells scored before.
        dict(name="scores_f16_gqa7", kind="scores", dtype="f16", heads=28, kv_heads=4, head_dim=128, block_size=32,
             fused=True, batch=17, ctx_lo=90, ctx_hi=3900, first=32, scored="some", lengths=8),
        # Three fp32 chats of two layers, one of them within its budget.  The smallest call of all.
        dict(name="evict_f32_small", kind="evict", dtype="f32", kv_heads=8, head_dim=64, block_size=16, layers=2,
             batch=3, ctx_lo=40, ctx_hi=600, budget=128, recent=64, protected=0, lengths=9),
        # Every layer of a 1B-shaped model at once: sixteen sequences down to 1024 tokens.
        dict(name="evict_16_layers", kind="evict", dtype="bf16", kv_heads=8, head_dim=64, block_size=16, layers=16,
             batch=16, ctx_lo=1500, ctx_hi=4096, budget=1024, recent=256, protected=64, lengths=10),
        # One layer of two long documents after their prefill, an eighth to a quarter kept.
        dict(name="evict_long_b2", kind="evict", dtype="bf16", kv_heads=8, head_dim=128, block_size=16, layers=1,
             batch=2, ctx_lo=32771, ctx_hi=65001, budget=8192, recent=1024, protected=16, lengths=11),
        # A trim of a serving batch in fp16, some sequences within the budget.
        dict(name="evict_f16_b17", kind="evict", dtype="f16", kv_heads=4, head_dim=128, block_size=32, layers=4,
             batch=17, ctx_lo=600, ctx_hi=2100, budget=1500, recent=500, protected=128, lengths=12),
    ]


# (heads, kv_heads, head_dim) of the drawn cases.
HEADS = [(32, 8, 64), (32, 8, 128), (28, 4, 128), (40, 8, 128), (16, 16, 64)]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prefix", "scores", "evict"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    case = dict(kind=kind, dtype=dtype, kv_heads=kv_heads, head_dim=head_dim, block_size=rng.choice([16, 16, 32]),
                lengths=rng.randrange(1 << 30))
    # A token's K and V in bytes, against the 4 KB of the large listed cases.
    weight = kv_heads * head_dim * 2 * ELEMENT[dtype] / 4096
    if kind == "evict":
        layers, batch = _log_int(rng, 1, 16), _log_int(rng, 1, 17)
        hi = _log_int(rng, 20, max(20, min(65001, int(120000 / (layers * batch * weight)))))
        budget = rng.randint(2, hi)
        recent = rng.randint(0, budget)
        protected = rng.choice([0, 0, rng.randint(0, budget - recent)])
        return dict(case, layers=layers, batch=batch, ctx_lo=rng.randint(1, hi), ctx_hi=hi, budget=budget,
                    recent=recent, protected=protected)
    case.update(heads=heads, fused=rng.random() < 0.5)
    if kind == "scores":
        batch = _log_int(rng, 1, 64)
        hi = _log_int(rng, 17, max(17, min(32768, int(131072 / (batch * weight)))))
        return dict(case, batch=batch, ctx_lo=rng.randint(1, hi), ctx_hi=hi, first=rng.choice([0, 0, rng.randint(0, hi)]),
                    scored=rng.choice(["none", "step", "some"]))
    batch = _log_int(rng, 1, 256)
    # Rows times prefix tokens held to a fifth of the largest listed case's in fp32, and to all of it in 16 bits.
    limit = (256 * 16384) * (32 * 128) / (heads * head_dim) / (5 if dtype == "f32" else 1)
    shared = _log_int(rng, 32, max(32, min(16384, int(limit / batch)))) // 32 * 32
    hi = _log_int(rng, 1, max(1, min(4096, int(120000 / (batch * weight)))))
    return dict(case, batch=batch, shared=shared, own_lo=rng.randint(0, hi), own_hi=hi,
                padded=rng.choice([0, 0, min(3, batch - 1)]))


# ---------------------------------------------------------------- inputs ----


def _lengths(case):
    """Context length of each sequence, int64."""
    rng = np.random.default_rng(case["lengths"])
    if case["kind"] == "prefix":
        ctx = case["shared"] + rng.integers(case["own_lo"], case["own_hi"], size=case["batch"], endpoint=True)
        ctx[case["batch"] - case["padded"]:] = 0
        return ctx
    return rng.integers(case["ctx_lo"], case["ctx_hi"], size=case["batch"], endpoint=True)


def _blocks(tokens, case):
    return (tokens + case["block_size"] - 1) // case["block_size"]


def _tables(need, shared, spare, seed):
    """Block tables [sequences, longest] over a shuffled pool: the first ``shared`` entries of the rows
    that have any are the same blocks, the others their own; and the pool's size with ``spare`` blocks more."""
    total = shared + int(np.maximum(need - shared, 0).sum()) + spare
    order = np.random.default_rng(seed).permutation(total).astype(np.int32)
    table = np.zeros((len(need), max(1, int(need.max()), shared)), np.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for s, n in enumerate(need):
        table[s, shared:n] = order[at:at + max(n - shared, 0)]
        at += max(n - shared, 0)
    return table, total, order[at:]


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)


def _weights(g, shape):
    """Scores as many steps leave them: most cells small, few large, some never looked at."""
    s = torch.empty(shape, device=DEVICE, dtype=torch.float32).exponential_(1.0, generator=g).square_()
    return s.masked_fill_(torch.rand(shape, device=DEVICE, generator=g) < 0.1, 0.0)


def _normal(g, shape, dtype):
    return torch.empty(shape, device=DEVICE, dtype=dtype).normal_(0.0, 1.0, generator=g)


def prepare(case, seed):
    ctx = _lengths(case)
    g, dt = torch.Generator(device=DEVICE).manual_seed(seed), DTYPES[case["dtype"]]
    hkv, d, bs, batch = case["kv_heads"], case["head_dim"], case["block_size"], case["batch"]
    state = dict(case=case, ctx=_i32(ctx), positions=int(ctx.max()))
    if case["kind"] == "evict":
        kept = np.minimum(ctx, case["budget"])
        spare = int(_blocks(kept, case).sum())
        table, blocks, free = _tables(_blocks(ctx, case), 0, spare + 1, seed)
        dst = np.zeros((batch, int(_blocks(kept, case).max())), np.int32)
        at = 0
        for s, n in enumerate(_blocks(kept, case)):
            dst[s, :n] = free[at:at + n]
            at += n
        layers = case["layers"]
        pool = torch.empty((layers, blocks, 2, hkv, bs, d), device=DEVICE, dtype=dt)
        for layer in range(layers):
            pool[layer].copy_(_normal(g, (blocks, 2, hkv, bs, d), dt))
        state.update(table=_i32(table), dst=_i32(dst), pool=pool, k=pool[:, :, 0], v=pool[:, :, 1],
                     scores=_weights(g, (layers, blocks, hkv, bs)),
                     new_lens=torch.zeros(batch, device=DEVICE, dtype=torch.int32),
                     kept=torch.zeros((layers, batch, hkv, case["budget"]), device=DEVICE, dtype=torch.int32))
        return state
    shared = case["shared"] // bs if case["kind"] == "prefix" else 0
    table, blocks, _ = _tables(_blocks(ctx, case), shared, 7, seed)
    heads = case["heads"]
    if case["fused"]:
        pool = _normal(g, (blocks, 2, hkv, bs, d), dt)
        kc, vc = pool[:, 0], pool[:, 1]
    else:
        kc, vc = _normal(g, (blocks, hkv, bs, d), dt), _normal(g, (blocks, hkv, bs, d), dt)
    # Queries that look at a few keys more than at the others, as a trained model's do.
    state.update(q=(2.0 * _normal(g, (batch, heads, d), torch.float32)).to(dt), k=kc, v=vc, table=_i32(table),
                 scale=1.0 / math.sqrt(d))
    if case["kind"] == "scores":
        rng = np.random.default_rng(seed)
        done = {"none": 0 * ctx, "step": ctx - 1, "some": rng.integers(0, ctx, endpoint=True)}[case["scored"]]
        state.update(scores=50.0 * _weights(g, (blocks, hkv, bs)), scored=_i32(done))
    return state


# ------------------------------------------------------- the plain forms ----


def _gather(cache, table, positions, block_size):
    """Rows of a paged cache [blocks, H_kv, bs, D] at ``positions`` of each sequence, fp32 [B, H_kv, T, D]."""
    block = table[:, positions // block_size].long()
    return cache[block, :, positions % block_size].permute(0, 2, 1, 3).float().contiguous()


def _softmax(logits, valid):
    """exp(x - max) / sum over the last dimension where ``valid``, zeros in a row without any."""
    top = logits.masked_fill(~valid, -math.inf).amax(-1, keepdim=True)
    e = torch.where(valid, torch.exp(logits - torch.where(top.isinf(), torch.zeros_like(top), top)),
                    torch.zeros_like(logits))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _plain_prefix(state):
    case, q, table, ctx = state["case"], state["q"], state["table"], state["ctx"]
    batch, hkv, d, bs = case["batch"], case["kv_heads"], case["head_dim"], case["block_size"]
    group, n = case["heads"] // hkv, case["shared"]
    first = torch.arange(n, device=DEVICE)
    rest = torch.arange(n, max(n + 1, state["positions"]), device=DEVICE)
    valid_rest = (rest < ctx[:, None])[:, None, None]                         # [B, 1, 1, R]
    rest = rest.clamp(max=table.shape[1] * bs - 1)
    x = q.float().view(batch, hkv, group, d)
    rows = x.permute(1, 0, 2, 3).reshape(hkv, batch * group, d).contiguous()  # the batch as rows of one product
    k0, v0 = (_gather(c, table[:1], first, bs)[0] for c in (state["k"], state["v"]))
    k1, v1 = (_gather(c, table, rest, bs) for c in (state["k"], state["v"]))
    a0 = torch.bmm(rows, k0.transpose(1, 2).contiguous()).view(hkv, batch, group, n).permute(1, 0, 2, 3)
    a1 = torch.matmul(x, k1.transpose(2, 3).contiguous())
    valid = torch.cat([(first < ctx[:, None])[:, None, None].expand(a0.shape), valid_rest.expand(a1.shape)], -1)
    p = _softmax(torch.cat([a0, a1], -1) * state["scale"], valid)
    o = torch.bmm(p[..., :n].permute(1, 0, 2, 3).reshape(hkv, batch * group, n).contiguous(), v0)
    v1 = torch.where(valid_rest.transpose(2, 3), v1, torch.zeros_like(v1))
    o = o.view(hkv, batch, group, d).permute(1, 0, 2, 3) + torch.matmul(p[..., n:].contiguous(), v1)
    return o.reshape(q.shape).to(q.dtype)


def _plain_scores(state):
    case, q, table, ctx = state["case"], state["q"], state["table"], state["ctx"]
    batch, hkv, d, bs = case["batch"], case["kv_heads"], case["head_dim"], case["block_size"]
    t = torch.arange(state["positions"], device=DEVICE)
    inside = t < ctx[:, None]                                                 # [B, T]
    x = q.float().view(batch, hkv, case["heads"] // hkv, d)
    k, v = (_gather(c, table, t, bs) for c in (state["k"], state["v"]))
    p = _softmax(torch.matmul(x, k.transpose(2, 3).contiguous()) * state["scale"], inside[:, None, None])
    o = torch.matmul(p, torch.where(inside[:, None, :, None], v, torch.zeros_like(v)))
    # [B, T, H_kv] weights into the cells of the scored positions.
    block, offset = table[:, t // bs].long(), (t % bs).expand(batch, -1)
    at = inside & (t >= case["first"])
    new = p.sum(2).transpose(1, 2)
    old = state["scores"][block, :, offset]
    new = torch.where((t < state["scored"][:, None])[..., None], old + new, new)
    state["scores"][block[at], :, offset[at]] = new[at]
    return {"out": o.reshape(q.shape).to(q.dtype), "scores": state["scores"]}


def _plain_evict(state):
    case, table, dst, ctx = state["case"], state["table"].long(), state["dst"].long(), state["ctx"].long()
    layers, batch, hkv, bs = case["layers"], case["batch"], case["kv_heads"], case["block_size"]
    budget, n = case["budget"], state["positions"]
    t = torch.arange(n, device=DEVICE)
    scores = state["scores"][:, table[:, t // bs], :, (t % bs).expand(batch, -1)]  # [B, T, L, H_kv]
    rank = torch.nan_to_num(scores.permute(2, 0, 3, 1), nan=-math.inf, posinf=3.4e38).double()
    forced = (ctx[:, None] <= budget) | (t < case["protected"]) | (t >= ctx[:, None] - case["recent"])
    rank = rank.clamp(min=-1e300).masked_fill(forced[:, None], math.inf)
    rank = rank.masked_fill((t >= ctx[:, None])[:, None], -math.inf)
    room = max(budget, 1)
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :room]
    # In the order of their positions, behind them those that are no token.
    lens = ctx.clamp(max=budget)                                              # [B]
    j = torch.arange(first.shape[-1], device=DEVICE)
    real = (j < lens[:, None])[:, None].expand(layers, batch, hkv, -1)
    first = torch.where(real, first, torch.full_like(first, n)).sort(-1).values
    old = first.clamp(max=n - 1)
    lane = torch.arange(layers, device=DEVICE)[:, None, None, None].expand_as(old)
    row = torch.arange(batch, device=DEVICE)[:, None, None].expand_as(old)
    head = torch.arange(hkv, device=DEVICE)[:, None].expand_as(old)
    block, offset = table[row, old // bs][real], (old % bs)[real]
    to = dst[:, (j // bs).clamp(max=dst.shape[1] - 1)][:, None].expand_as(old)[real]
    into, lane, head = (j % bs).expand_as(old)[real], lane[real], head[real]
    state["k"][lane, to, head, into] = state["k"][lane, block, head, offset]
    state["v"][lane, to, head, into] = state["v"][lane, block, head, offset]
    state["scores"][lane, to, head, into] = state["scores"][lane, block, head, offset]
    state["new_lens"].copy_(lens)
    state["kept"].fill_(-1)[..., :first.shape[-1]] = torch.where(real, first, torch.full_like(first, -1)).int()
    return {"pool": state["pool"], "scores": state["scores"], "new_lens": state["new_lens"], "kept": state["kept"]}


@functools.lru_cache(maxsize=None)
def _kernels():
    from railgun_amd.ops import PagedAttentionKernels

    return PagedAttentionKernels(0)


def _own(state):
    case, q, k, v, table, ctx = (state.get(n) for n in ("case", "q", "k", "v", "table", "ctx"))
    if case["kind"] == "evict":
        _kernels().launch_evict(k, v, state["scores"], table, state["dst"], ctx, state["new_lens"], state["kept"],
                                case["budget"], case["recent"], case["protected"])
        return {"pool": state["pool"], "scores": state["scores"], "new_lens": state["new_lens"], "kept": state["kept"]}
    from railgun_amd.ops import PagedAttentionOp

    op = PagedAttentionOp(state["scale"], case["heads"], case["kv_heads"], case["head_dim"], case["block_size"],
                          _kernels())
    if case["kind"] == "prefix":
        return op.execute_shared_prefix(q, k, v, table, ctx, case["shared"] // case["block_size"])
    out = op.execute_with_scores(q, k, v, table, ctx, state["scores"], state["scored"], case["first"])
    return {"out": out, "scores": state["scores"]}


def run(state):
    if own:
        return _own(state)
    return {"prefix": _plain_prefix, "scores": _plain_scores, "evict": _plain_evict}[state["case"]["kind"]](state)


# -------------------------------------------------- floors and 64 bits ----


def work(case):
    ctx = _lengths(case).astype(np.float64)
    row = case["kv_heads"] * case["head_dim"] * ELEMENT[case["dtype"]]
    if case["kind"] == "evict":
        kept = np.minimum(ctx, case["budget"])
        cells = case["layers"] * case["kv_heads"] * 4
        # K and V of what is kept, read and written; every score read; those kept and their positions written.
        return {"bytes": float(case["layers"] * kept.sum() * row * 4 + cells * (ctx.sum() + 2 * kept.sum())),
                "flops": 0.0}
    rows = case["batch"] * case["heads"] * case["head_dim"] * ELEMENT[case["dtype"]] * 2
    flops = 4.0 * case["heads"] * case["head_dim"] * ctx.sum()
    if case["kind"] == "prefix":
        tokens = case["shared"] + np.maximum(ctx - case["shared"], 0).sum()
        return {"bytes": float(tokens * row * 2 + rows), "flops": float(flops)}
    scored = np.maximum(ctx - case["first"], 0).sum() * case["kv_heads"] * (4 if case["scored"] == "none" else 8)
    return {"bytes": float(ctx.sum() * row * 2 + rows + scored), "flops": float(flops)}


def _rows64(cache, table_row, n, block_size):
    """The first n rows of one sequence, float64 [H_kv, n, D]."""
    blocks = table_row[:(n + block_size - 1) // block_size].long()
    return cache[blocks].double().transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_evict(case, s):
    k, v, scores, kept = s["k"], s["v"], s["scores"], s["kept"]
    all_scores = scores.cpu().numpy()
    table, dst, ctx = (s[name].cpu().numpy() for name in ("table", "dst", "ctx"))
    bs, hkv, layers = case["block_size"], case["kv_heads"], case["layers"]
    kept.fill_(-1)
    for b, n in enumerate(ctx):
        t = np.arange(n)
        seen = all_scores[:, table[b, t // bs], :, t % bs].transpose(1, 2, 0)  # [L, H_kv, n]
        m = min(int(n), case["budget"])
        middle = np.arange(case["protected"], n - case["recent"])
        take = case["budget"] - case["protected"] - case["recent"]
        where = np.zeros((layers, hkv, m), np.int64)
        for layer in range(layers):
            for h in range(hkv):
                if n <= m:
                    where[layer, h] = t
                else:
                    best = middle[np.argsort(-seen[layer, h, middle], kind="stable")[:take]]
                    where[layer, h] = np.sort(np.concatenate([t[:case["protected"]], best, t[n - case["recent"]:]]))
        j = np.arange(m)
        at = torch.from_numpy(where).to(DEVICE)
        source = torch.from_numpy(table[b].astype(np.int64)).to(DEVICE)[at // bs]
        lane = torch.arange(layers, device=DEVICE)[:, None, None]
        head = torch.arange(hkv, device=DEVICE)[None, :, None]
        to = torch.from_numpy(dst[b, j // bs].astype(np.int64)).to(DEVICE)
        into = torch.from_numpy(j % bs).to(DEVICE)
        for x in (k, v, scores):
            x[lane, to, head, into] = x[lane, source, head, at % bs]
        kept[:, b, :, :m] = at.int()
    return {"pool": s["pool"], "scores": scores, "kept": kept,
            "new_lens": torch.from_numpy(np.minimum(ctx, case["budget"]).astype(np.int32))}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(case, s)
    q, bs, hkv = s["q"].double(), case["block_size"], case["kv_heads"]
    out = torch.zeros_like(q)
    scores = s["scores"].double() if case["kind"] == "scores" else None
    for b, n in enumerate(s["ctx"].tolist()):
        if n == 0:
            continue
        k, v = (_rows64(c, s["table"][b], n, bs) for c in (s["k"], s["v"]))
        group = case["heads"] // hkv
        weights = []
        for h in range(hkv):
            a = (q[b, h * group:(h + 1) * group] @ k[h].t().contiguous()) * s["scale"]
            a = torch.exp(a - a.max(1, keepdim=True).values)
            a /= a.sum(1, keepdim=True)
            out[b, h * group:(h + 1) * group] = a @ v[h]
            weights.append(a.sum(0))
        if scores is not None and case["first"] < n:
            t = torch.arange(case["first"], n, device=DEVICE)
            block, offset = s["table"][b].long()[t // bs], t % bs
            w = torch.stack(weights, 1)[t]
            before = torch.where((t < s["scored"][b])[:, None], scores[block, :, offset], torch.zeros_like(w))
            scores[block, :, offset] = before + w
    return out if scores is None else {"out": out, "scores": scores}
