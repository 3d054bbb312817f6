"""Operators of a step over drafted tokens: every sequence brings a tree of them behind its cached ones, the
model looks at all of them at once, and the path that it agrees with stays.

A case is a dict of plain values; lengths and trees belong to the case (``lengths`` seeds them), tensor contents
come from the seed given to :func:`prepare`.  A sequence's tokens in the cache are its ``ctx``, of which the last
``L`` are the nodes of its tree, node 0 the token that was decided last.  Kinds:

``layout``   from the nodes' parents: the bits of each node's ancestors and itself, its position in the text (the
             root's plus its depth) and its slot in the paged cache.
``tree``     attention of all nodes over the paged cache: a node sees every token before the tree, and of the
             tree its ancestors and itself.
``verify``   which nodes the model agrees with: each node's target token is the argmax of its logits (or, with
             ``sampled``, comes from a sampler); from the root on, the lowest child that drafted the target of the
             last accepted node is accepted; the target of the last one is the next token.
``compact``  the accepted nodes' K, V and scores move down to directly behind the tokens before the tree, in
             every layer.

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
        # One user's drafts of 64 tokens: the smallest call, all latency.
        dict(name="layout_b1", kind="layout", block_size=16, batch=1, padded=0, ctx_lo=900, ctx_hi=1400, nodes_lo=64,
             nodes_hi=64, depth=6, moved=False, lengths=1),
        # A large serving batch with trees of up to 256 drafted tokens, some sequences' caches evicted before.
        dict(name="layout_b256", kind="layout", block_size=16, batch=256, padded=0, ctx_lo=300, ctx_hi=4096,
             nodes_lo=33, nodes_hi=256, depth=12, moved=True, lengths=2),
        # The reference's element type and CPU-runnable head shape: three short chats, a few drafts each.
        dict(name="tree_f32_small", kind="tree", dtype="f32", heads=32, kv_heads=8, head_dim=64, block_size=16,
             fused=False, batch=3, padded=0, ctx_lo=40, ctx_hi=300, nodes_lo=4, nodes_hi=12, depth=4, lengths=3),
        # One chat of an 8B-shaped model, 64 drafted tokens.
        dict(name="tree_b1", kind="tree", dtype="bf16", heads=32, kv_heads=8, head_dim=128, block_size=16, fused=True,
             batch=1, padded=0, ctx_lo=4001, ctx_hi=4096, nodes_lo=64, nodes_hi=64, depth=6, lengths=4),
        # The headline serving load, one layer: 64 sequences of 512 to 4096 tokens, trees of 8 to 32 tokens.
        dict(name="tree_b64", kind="tree", dtype="bf16", heads=32, kv_heads=8, head_dim=128, block_size=16,
             fused=True, batch=64, padded=0, ctx_lo=512, ctx_hi=4096, nodes_lo=8, nodes_hi=32, depth=5, lengths=5),
        # An odd batch in fp16, seven query heads to a kv-head, blocks of 32, two rows that pad a captured
        # graph's batch, some trees of the root alone.
        dict(name="tree_f16_gqa7", kind="tree", dtype="f16", heads=28, kv_heads=4, head_dim=128, block_size=32,
             fused=True, batch=17, padded=2, ctx_lo=90, ctx_hi=3900, nodes_lo=1, nodes_hi=37, depth=7, lengths=6),
        # Long documents with wide trees: the largest attention call.
        dict(name="tree_long_b4", kind="tree", dtype="bf16", heads=32, kv_heads=8, head_dim=128, block_size=16,
             fused=True, batch=4, padded=0, ctx_lo=30001, ctx_hi=32768, nodes_lo=101, nodes_hi=128, depth=10,
             lengths=7),
        # One user's 64 drafts under the headline model's vocabulary.
        dict(name="verify_b1", kind="verify", dtype="bf16", sampled=False, vocab=128256, batch=1, padded=0,
             nodes_lo=64, nodes_hi=64, depth=6, agree=0.8, lengths=8),
        # The headline serving load's drafts.
        dict(name="verify_b64", kind="verify", dtype="bf16", sampled=False, vocab=128256, batch=64, padded=0,
             nodes_lo=8, nodes_hi=32, depth=5, agree=0.7, lengths=9),
        # Tokens that a sampler drew, a large batch.
        dict(name="verify_sampled_b256", kind="verify", dtype="bf16", sampled=True, vocab=128256, batch=256, padded=3,
             nodes_lo=1, nodes_hi=64, depth=8, agree=0.7, lengths=10),
        # Two fp32 layers of three chats.
        dict(name="compact_f32_small", kind="compact", dtype="f32", kv_heads=8, head_dim=64, block_size=16, layers=2,
             batch=3, padded=0, ctx_lo=40, ctx_hi=300, nodes_lo=4, nodes_hi=12, depth=4, scores=False, lengths=11),
        # Every layer of a 1B-shaped model at once, 64 sequences, with the attention weights that eviction goes by.
        dict(name="compact_16_layers", kind="compact", dtype="bf16", kv_heads=8, head_dim=64, block_size=16,
             layers=16, batch=64, padded=0, ctx_lo=200, ctx_hi=700, nodes_lo=16, nodes_hi=64, depth=8, scores=True,
             lengths=12),
    ]


# (heads, kv_heads, head_dim) of the drawn cases.
HEADS = [(32, 8, 64), (32, 8, 128), (28, 4, 128), (40, 8, 128), (16, 16, 64)]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["layout", "tree", "tree", "verify", "compact"])
    batch = _log_int(rng, 1, {"layout": 256, "tree": 64, "verify": 256, "compact": 64}[kind])
    case = dict(kind=kind, batch=batch, padded=rng.choice([0, 0, min(3, batch - 1)]), depth=_log_int(rng, 1, 12),
                lengths=rng.randrange(1 << 30))
    if kind == "layout":
        hi = _log_int(rng, 1, 256)
        return dict(case, block_size=rng.choice([16, 16, 32]), nodes_lo=rng.randint(1, hi), nodes_hi=hi,
                    ctx_lo=hi, ctx_hi=_log_int(rng, hi, 32768), moved=rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "verify":
        sampled, vocab = rng.random() < 0.3, rng.choice([128256, 32000, 49999])
        # Logits held to those of the large listed case.
        most = 64 * 32 * 128256 * 2 // (vocab * ELEMENT[dtype] * batch)
        hi = _log_int(rng, 1, max(1, min(128, 128 if sampled else most)))
        return dict(case, dtype=dtype, sampled=sampled, vocab=vocab, nodes_lo=rng.randint(1, hi), nodes_hi=hi,
                    agree=rng.choice([0.0, 0.5, 0.8, 1.0]))
    heads, kv_heads, head_dim = rng.choice(HEADS)
    case.update(dtype=dtype, kv_heads=kv_heads, head_dim=head_dim, block_size=rng.choice([16, 16, 32]))
    # A token's K and V in bytes, against the 4 KB of the large listed cases.
    weight = kv_heads * head_dim * 2 * ELEMENT[dtype] / 4096
    nodes = _log_int(rng, 1, 128)
    case.update(nodes_lo=rng.randint(1, nodes), nodes_hi=nodes)
    if kind == "compact":
        layers = _log_int(rng, 1, 16)
        hi = _log_int(rng, nodes, max(nodes, min(4096, int(400000 / (layers * batch * weight)))))
        return dict(case, layers=layers, ctx_lo=rng.randint(nodes, hi), ctx_hi=hi, scores=rng.random() < 0.5)
    # Cached tokens held to the large listed cases', and rows times tokens to the largest's (a tenth in fp32).
    tokens = min(200000 / weight, 4 * 30000 * 110 / nodes * 4096 / (heads * head_dim) / (10 if dtype == "f32" else 1))
    hi = _log_int(rng, nodes, max(nodes, min(32768, int(tokens / batch))))
    return dict(case, heads=heads, fused=rng.random() < 0.5, ctx_lo=rng.randint(nodes, hi), ctx_hi=hi)


# ---------------------------------------------------------------- inputs ----


def _tree(rng, n, depth):
    """Parents of a tree of n nodes: a chain of the likeliest drafts first, then its side branches."""
    main = min(depth, n - 1)
    parents, level = [-1] + list(range(main)), list(range(main + 1))
    for _ in range(main + 1, n):
        p = int(rng.integers(0, len(parents)))
        p = parents[p] if level[p] >= depth else p
        parents.append(p)
        level.append(level[p] + 1)
    return parents


@functools.lru_cache(maxsize=8)
def _forest_of(batch, padded, lo, hi, depth, lengths):
    rng = np.random.default_rng(lengths)
    count = rng.integers(lo, hi, size=batch, endpoint=True)
    count[batch - padded:] = 0
    trees = [_tree(rng, int(n), depth) if n else [] for n in count]
    return np.concatenate([[0], np.cumsum(count)]), np.asarray(sum(trees, []), np.int64)


def _forest(case):
    """(first node of each sequence and their number, int64 [B + 1]; parents, int64 [N])."""
    return _forest_of(*(case[k] for k in ("batch", "padded", "nodes_lo", "nodes_hi", "depth", "lengths")))


def _ancestors(cu, parents):
    """Per node the nodes it sees, itself among them, as lists of places in its tree."""
    seen = []
    for s in range(len(cu) - 1):
        own_tree = []
        for j, p in enumerate(parents[cu[s]:cu[s + 1]]):
            own_tree.append((own_tree[p] if p >= 0 else []) + [j])
        seen += own_tree
    return seen


def _mask_words(case):
    return (case["nodes_hi"] + 31) // 32


def _mask(case):
    """The bits of _ancestors, int32 [N, words]."""
    seen = _ancestors(*_forest(case))
    words = np.zeros((len(seen), _mask_words(case)), np.uint32)
    for n, nodes in enumerate(seen):
        for i in nodes:
            words[n, i // 32] |= np.uint32(1 << (i % 32))
    return words.view(np.int32)


def _lengths(case):
    """Tokens in the cache of each sequence, its tree's among them, int64; none where it has no tree."""
    rng = np.random.default_rng(case["lengths"] + 1)
    ctx = rng.integers(case["ctx_lo"], case["ctx_hi"], size=case["batch"], endpoint=True)
    nodes = np.diff(_forest(case)[0])
    return np.where(nodes > 0, np.maximum(ctx, nodes), 0)


def _tables(ctx, block_size, spare, seed):
    """A block table over a shuffled pool, and the pool's size with ``spare`` blocks more."""
    need = (ctx + block_size - 1) // block_size
    total = int(need.sum()) + spare
    order = np.random.default_rng(seed).permutation(total).astype(np.int32)
    table = np.zeros((len(need), max(1, int(need.max()))), np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)


def _empty(*shape, dtype=torch.int32):
    return torch.zeros(shape, device=DEVICE, dtype=dtype)


def _normal(g, shape, dtype):
    return torch.empty(shape, device=DEVICE, dtype=dtype).normal_(0.0, 1.0, generator=g)


def _prepare_verify(case, seed, state, cu, parents):
    g, rng = torch.Generator(device=DEVICE).manual_seed(seed), np.random.default_rng(seed)
    n, width = len(parents), case["depth"] + 1
    if case["sampled"]:
        target = rng.integers(0, case["vocab"], size=n)
        state["target"] = _i32(target)
    else:
        # Logits as a trained model's: most of them small, a few far above.
        logits = _normal(g, (n, case["vocab"]), DTYPES[case["dtype"]])
        peak = torch.randint(0, case["vocab"], (n, 4), device=DEVICE, generator=g)
        logits.scatter_add_(1, peak, (8.0 + _normal(g, (n, 4), torch.float32)).to(logits.dtype))
        target = _first_largest(logits).cpu().numpy()
        state.update(logits=logits, target=_empty(n))
    # Drafts: mostly what the model says behind the parent, or something else.
    up = np.repeat(cu[:-1], np.diff(cu)) + np.maximum(parents, 0)
    draft = np.where(rng.random(n) < case["agree"], target[up], rng.integers(0, case["vocab"], size=n))
    state.update(draft=_i32(draft), accepted=_empty(case["batch"], width), count=_empty(case["batch"]),
                 next=_empty(case["batch"]))
    return state


def prepare(case, seed):
    cu, parents = _forest(case)
    state = dict(case=case, cu=_i32(cu), parents=_i32(parents), nodes=case["nodes_hi"])
    if case["kind"] == "verify":
        return _prepare_verify(case, seed, state, cu, parents)
    ctx, bs, batch = _lengths(case), case["block_size"], case["batch"]
    table, blocks = _tables(ctx, bs, 7, seed)
    state.update(table=_i32(table), ctx=_i32(ctx), longest=int(ctx.max()))
    if case["kind"] == "layout":
        n = len(parents)
        place = ctx - np.diff(cu) + np.random.default_rng(seed).integers(0, 1000, size=batch)
        state.update(place=_i32(place) if case["moved"] else None, mask=_empty(n, _mask_words(case)),
                     positions=_empty(n), slots=_empty(n))
        return state
    g, dt, hkv, d = (torch.Generator(device=DEVICE).manual_seed(seed), DTYPES[case["dtype"]], case["kv_heads"],
                     case["head_dim"])
    if case["kind"] == "compact":
        layers = case["layers"]
        pool = torch.empty((layers, blocks, 2, hkv, bs, d), device=DEVICE, dtype=dt)
        for layer in range(layers):
            pool[layer].copy_(_normal(g, (blocks, 2, hkv, bs, d), dt))
        # The path to any of a tree's nodes.
        rng = np.random.default_rng(seed)
        seen = _ancestors(cu, parents)
        accepted, count = np.full((batch, case["depth"] + 1), -1), np.zeros(batch, np.int64)
        for s in range(batch):
            if cu[s + 1] > cu[s]:
                path = seen[rng.integers(cu[s], cu[s + 1])]
                accepted[s, :len(path)], count[s] = path, len(path)
        scores = torch.empty((layers, blocks, hkv, bs), device=DEVICE).exponential_(1.0, generator=g)
        state.update(pool=pool, k=pool[:, :, 0], v=pool[:, :, 1], scores=scores if case["scores"] else None,
                     accepted=_i32(accepted), count=_i32(count), new_lens=_empty(batch))
        return state
    heads = case["heads"]
    if case["fused"]:
        pool = _normal(g, (blocks, 2, hkv, bs, d), dt)
        kc, vc = pool[:, 0], pool[:, 1]
    else:
        kc, vc = _normal(g, (blocks, hkv, bs, d), dt), _normal(g, (blocks, hkv, bs, d), dt)
    # Queries that look at a few keys more than at the others, as a trained model's do.
    state.update(q=(2.0 * _normal(g, (len(parents), heads, d), torch.float32)).to(dt), k=kc, v=vc,
                 mask=_i32(_mask(case)), scale=1.0 / math.sqrt(d))
    return state


# ------------------------------------------------------- the plain forms ----


def _rows(cu, n):
    """(sequence, place in its tree) of each of n nodes."""
    row = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(cu.long(), row, right=True) - 1
    return seq, row - cu.long()[seq]


def _prior(state):
    """Tokens before each sequence's tree."""
    return state["ctx"].long() - torch.diff(state["cu"].long())


def _plain_layout(state):
    case, table, parents = state["case"], state["table"], state["parents"].long()
    n, words, bs = len(parents), state["mask"].shape[1], case["block_size"]
    seq, place = _rows(state["cu"], n)
    up = torch.where(parents >= 0, state["cu"].long()[seq] + parents, torch.full_like(parents, n))
    bits = torch.nn.functional.one_hot(place, 32 * words).bool()
    seen = bits
    for _ in range(case["depth"]):
        seen = bits | torch.cat([seen, torch.zeros_like(seen[:1])])[up]
    word = (seen.view(n, words, 32).long() << torch.arange(32, device=DEVICE)).sum(-1)
    prior = _prior(state)
    root = prior if state["place"] is None else state["place"].long()
    at = prior[seq] + place
    state["mask"].copy_(torch.where(word >= 1 << 31, word - (1 << 32), word))
    state["positions"].copy_(root[seq] + seen.sum(-1) - 1)
    state["slots"].copy_(table[seq, at // bs].long() * bs + at % bs)
    return {"mask": state["mask"], "positions": state["positions"], "slots": state["slots"]}


def _gather(cache, table, positions, block_size):
    """Rows of a paged cache [blocks, H_kv, bs, D] at ``positions`` of each sequence, fp32 [B, H_kv, T, D]."""
    block = table[:, positions // block_size].long()
    return cache[block, :, positions % block_size].permute(0, 2, 1, 3).float().contiguous()


def _softmax_(logits, valid):
    """exp(x - max) / sum over the last dimension where ``valid``, zeros in a row without any, in place."""
    logits.masked_fill_(~valid, -math.inf)
    top = logits.amax(-1, keepdim=True)
    e = logits.sub_(torch.where(top.isinf(), torch.zeros_like(top), top)).exp_()
    total = e.sum(-1, keepdim=True)
    return e.div_(torch.where(total > 0, total, torch.ones_like(total)))


def _plain_tree(state):
    case, q, table, cu, ctx = state["case"], state["q"], state["table"], state["cu"].long(), state["ctx"].long()
    batch, hkv, d, bs, most = case["batch"], case["kv_heads"], case["head_dim"], case["block_size"], state["nodes"]
    group, n = case["heads"] // hkv, len(q)
    seq, place = _rows(cu, n)
    t, j = torch.arange(state["longest"], device=DEVICE), torch.arange(most, device=DEVICE)
    row = (cu[:-1, None] + j).clamp(max=n - 1)                                 # [B, L], padded
    prior = _prior(state)
    bit = (state["mask"][:, j // 32] >> (j % 32)) & 1                          # [N, L]
    node = (t - prior[:, None]).clamp(0, most - 1)                             # [B, T]
    sees = bit[row].gather(2, node[:, None].expand(-1, most, -1)).bool()       # [B, L, T]
    valid = ((t < prior[:, None])[:, None] | sees) & (t < ctx[:, None])[:, None]
    x = q[row].float().view(batch, most, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * most, d)
    k, v = (_gather(c, table, t, bs) for c in (state["k"], state["v"]))
    a = torch.matmul(x, k.transpose(2, 3).contiguous()).mul_(state["scale"]).view(batch, hkv, group, most, -1)
    p = _softmax_(a, valid[:, None, None]).view(batch, hkv, group * most, -1)
    o = torch.matmul(p, torch.where((t < ctx[:, None])[:, None, :, None], v, torch.zeros_like(v)))
    o = o.view(batch, hkv, group, most, d).permute(0, 3, 1, 2, 4).reshape(batch, most, case["heads"], d)
    return o[seq, place].to(q.dtype)


def _first_largest(logits):
    """Lowest index of the largest value of each row, NaN counted as the least."""
    x = torch.nan_to_num(logits.float(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    at = torch.arange(x.shape[1], device=x.device, dtype=torch.int32)
    return torch.where(x == x.amax(1, keepdim=True), at, x.shape[1]).amin(1)


def _plain_verify(state):
    case, cu, parents, draft = state["case"], state["cu"].long(), state["parents"].long(), state["draft"]
    n = len(draft)
    if not case["sampled"]:
        state["target"].copy_(_first_largest(state["logits"]))
    target = state["target"]
    seq, place = _rows(cu, n)
    up = cu[seq] + parents.clamp(min=0)
    agrees = (parents >= 0) & (target[up] == draft)
    child = torch.full((n + 1,), n, device=DEVICE).scatter_reduce(
        0, torch.where(agrees, up, torch.full_like(up, n)), torch.where(agrees, cu[seq] + place, n), "amin")
    child[n] = n
    has = torch.diff(cu) > 0
    at = torch.where(has, cu[:-1], torch.full_like(cu[:-1], n))
    last = at
    for i in range(case["depth"] + 1):
        state["accepted"][:, i] = torch.where(at < n, at - cu[:-1], -1)
        last = torch.where(at < n, at, last)
        at = child[at]
    state["count"].copy_((state["accepted"] >= 0).sum(1))
    state["next"].copy_(torch.where(has, target[last.clamp(max=n - 1)], -1))
    return {name: state[name] for name in ("target", "accepted", "count", "next")}


def _plain_compact(state):
    case, table, accepted, count = state["case"], state["table"].long(), state["accepted"].long(), state["count"]
    bs, prior = case["block_size"], _prior(state)
    i = torch.arange(accepted.shape[1], device=DEVICE).expand_as(accepted)
    moves = (i < count[:, None]) & (accepted != i)
    old, new = (prior[:, None] + accepted)[moves], (prior[:, None] + i)[moves]
    seq = torch.arange(case["batch"], device=DEVICE)[:, None].expand_as(i)[moves]
    for x in (state["k"], state["v"]) + ((state["scores"],) if case["scores"] else ()):
        x[:, table[seq, new // bs], :, new % bs] = x[:, table[seq, old // bs], :, old % bs]
    state["new_lens"].copy_(prior + count)
    return {"pool": state["pool"], "scores": state["scores"], "new_lens": state["new_lens"]}


@functools.lru_cache(maxsize=None)
def _kernels():
    from railgun_amd.ops import PagedAttentionKernels

    return PagedAttentionKernels(0)


def _own(state):
    case, kernels = state["case"], _kernels()
    table, ctx, cu, parents = (state.get(name) for name in ("table", "ctx", "cu", "parents"))
    if case["kind"] == "layout":
        kernels.launch_tree_layout(parents, cu, ctx, table, state["mask"], state["positions"], state["slots"],
                                   case["block_size"], state["nodes"], state["place"])
        return {"mask": state["mask"], "positions": state["positions"], "slots": state["slots"]}
    if case["kind"] == "verify":
        outs = state["accepted"], state["count"], state["next"]
        if case["sampled"]:
            kernels.launch_accept_tree(state["target"], state["draft"], parents, cu, state["nodes"], *outs)
        else:
            kernels.launch_verify_tree(state["logits"], state["draft"], parents, cu, state["nodes"], state["target"],
                                       *outs)
        return {name: state[name] for name in ("target", "accepted", "count", "next")}
    if case["kind"] == "compact":
        kernels.launch_compact_tree(state["k"], state["v"], state["scores"], table, ctx, cu, state["accepted"],
                                    state["count"], state["new_lens"])
        return {"pool": state["pool"], "scores": state["scores"], "new_lens": state["new_lens"]}
    from railgun_amd.ops import PagedAttentionOp

    op = PagedAttentionOp(state["scale"], case["heads"], case["kv_heads"], case["head_dim"], case["block_size"], kernels)
    return op.execute_tree(state["q"], state["k"], state["v"], table, ctx, cu, state["mask"], state["nodes"])


def run(state):
    if own:
        return _own(state)
    return {"layout": _plain_layout, "tree": _plain_tree, "verify": _plain_verify,
            "compact": _plain_compact}[state["case"]["kind"]](state)


# -------------------------------------------------- floors and 64 bits ----


def _moved(case):
    """Accepted nodes that do not lie in place already, as the paths to all nodes have them on average."""
    cu, parents = _forest(case)
    seen = _ancestors(cu, parents)
    per = np.array([sum(i != j for i, j in enumerate(path)) for path in seen], float)
    return sum(per[cu[s]:cu[s + 1]].mean() for s in range(len(cu) - 1) if cu[s + 1] > cu[s])


def work(case):
    cu, parents = _forest(case)
    n, nodes = len(parents), np.diff(cu).astype(np.float64)
    if case["kind"] == "verify":
        logits = 4 if case["sampled"] else case["vocab"] * ELEMENT[case["dtype"]] + 4
        return {"bytes": float(n * (logits + 8) + case["batch"] * (case["depth"] + 4) * 4), "flops": 0.0}
    if case["kind"] == "layout":
        return {"bytes": float(n * (4 * _mask_words(case) + 12) + case["batch"] * 12), "flops": 0.0}
    row = case["kv_heads"] * case["head_dim"] * ELEMENT[case["dtype"]]
    if case["kind"] == "compact":
        token = case["layers"] * (4 * row + (8 * case["kv_heads"] if case["scores"] else 0))
        return {"bytes": float(_moved(case) * token + case["batch"] * (case["depth"] + 5) * 4), "flops": 0.0}
    ctx = _lengths(case).astype(np.float64)
    pairs = ((ctx - nodes) * nodes).sum() + sum(len(path) for path in _ancestors(cu, parents))
    width = case["heads"] * case["head_dim"]
    return {"bytes": float(ctx.sum() * row * 2 + n * (2 * width * ELEMENT[case["dtype"]] + 4 * _mask_words(case))),
            "flops": float(4.0 * width * pairs)}


def _exact_tree(case, s):
    cu, parents = _forest(case)
    seen, bs, hkv = _ancestors(cu, parents), case["block_size"], case["kv_heads"]
    group, q = case["heads"] // hkv, s["q"].double()
    out = torch.zeros_like(q)
    for b, n in enumerate(s["ctx"].tolist()):
        count = int(cu[b + 1] - cu[b])
        if count == 0:
            continue
        hides = np.ones((count, count), bool)
        for j, path in enumerate(seen[cu[b]:cu[b + 1]]):
            hides[j, path] = False
        hides = torch.from_numpy(hides).to(DEVICE).repeat_interleave(group, 0)
        blocks = s["table"][b, :(n + bs - 1) // bs].long()
        k, v = (c[blocks].transpose(0, 1).flatten(1, 2)[:, :n] for c in (s["k"], s["v"]))
        for h in range(hkv):
            heads = slice(h * group, (h + 1) * group)
            a = (q[cu[b]:cu[b + 1], heads].reshape(count * group, -1) @ k[h].double().t().contiguous()) * s["scale"]
            a[:, n - count:].masked_fill_(hides, -math.inf)
            a = torch.exp(a - a.max(1, keepdim=True).values)
            o = (a / a.sum(1, keepdim=True)) @ v[h].double()
            out[cu[b]:cu[b + 1], heads] = o.view(count, group, -1)
    return out


def _exact_verify(case, s):
    cu, parents = _forest(case)
    draft = s["draft"].cpu().numpy()
    if case["sampled"]:
        target = s["target"].cpu().numpy()
    else:
        target = np.array([int(torch.nonzero(row == row.max())[0]) for row in s["logits"]], np.int32)
    accepted, count = np.full((case["batch"], case["depth"] + 1), -1, np.int32), np.zeros(case["batch"], np.int32)
    following = np.full(case["batch"], -1, np.int32)
    for b in range(case["batch"]):
        nodes = range(int(cu[b + 1] - cu[b]))
        path = [0][:len(nodes)]
        while path:
            fits = [j for j in nodes if parents[cu[b] + j] == path[-1] and draft[cu[b] + j] == target[cu[b] + path[-1]]]
            if not fits:
                break
            path.append(fits[0])
        accepted[b, :len(path)], count[b] = path, len(path)
        if path:
            following[b] = target[cu[b] + path[-1]]
    return {name: torch.from_numpy(np.ascontiguousarray(x)) for name, x in
            (("target", target), ("accepted", accepted), ("count", count), ("next", following))}


def _exact_layout(case, s):
    cu, parents = _forest(case)
    seen, ctx, table, bs = _ancestors(cu, parents), _lengths(case), s["table"].cpu().numpy(), case["block_size"]
    positions, slots = np.zeros(len(parents), np.int32), np.zeros(len(parents), np.int32)
    for b in range(case["batch"]):
        first = ctx[b] - (cu[b + 1] - cu[b])
        root = first if s["place"] is None else int(s["place"][b])
        for j in range(int(cu[b + 1] - cu[b])):
            positions[cu[b] + j] = root + len(seen[cu[b] + j]) - 1
            slots[cu[b] + j] = table[b, (first + j) // bs] * bs + (first + j) % bs
    return {"mask": torch.from_numpy(_mask(case).copy()), "positions": torch.from_numpy(positions),
            "slots": torch.from_numpy(slots)}


def _exact_compact(case, s):
    cu = _forest(case)[0]
    ctx, table, accepted, count = (s[name].cpu().numpy() for name in ("ctx", "table", "accepted", "count"))
    bs, lens = case["block_size"], np.zeros(case["batch"], np.int32)
    for b in range(case["batch"]):
        first = int(ctx[b] - (cu[b + 1] - cu[b]))
        lens[b] = first + count[b]
        old = first + accepted[b, :count[b]].astype(np.int64)
        new = first + np.arange(count[b])
        src = torch.from_numpy(np.stack([table[b, old // bs], old % bs]).astype(np.int64)).to(DEVICE)
        dst = torch.from_numpy(np.stack([table[b, new // bs], new % bs]).astype(np.int64)).to(DEVICE)
        for x in (s["k"], s["v"]) + ((s["scores"],) if case["scores"] else ()):
            x[:, dst[0], :, dst[1]] = x[:, src[0], :, src[1]].clone()
    return {"pool": s["pool"], "scores": s["scores"], "new_lens": torch.from_numpy(lens)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"layout": _exact_layout, "tree": _exact_tree, "verify": _exact_verify,
            "compact": _exact_compact}[case["kind"]](case, s)
