"""Layout, verification and compaction of trees of drafted tokens, value for value against plain loops."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import TORCH_DT, i32
from railgun_amd.kv_pool import GpuBlockPool
from railgun_amd.ops import RailgunError
from tree64 import accept, ancestors, first_largest, random_tree, words_of

pytestmark = pytest.mark.gpu


def forest(rng, sizes, **kw):
    trees = [random_tree(rng, n, **kw) for n in sizes]
    return trees, np.concatenate([[0], np.cumsum(sizes)]), np.asarray(sum(trees, []), np.int32)


# ------------------------------------------------------------------ layout --


def run_layout(kernels, device, cu, parents, ctx, table, bs, max_nodes, words, text=None):
    n = len(parents)
    out = [torch.full(s, -7, dtype=torch.int32, device=device) for s in ((n, words), (n,), (n,))]
    kernels.launch_tree_layout(i32(parents, device), i32(cu, device), i32(ctx, device), i32(table, device), *out, bs,
                               max_nodes, None if text is None else i32(text, device))
    return [t.cpu().numpy() for t in out]


def check_layout(kernels, device, trees, prior, bs=16, words=None, text=None, short=0, behind=0, seed=0):
    rng = np.random.default_rng(seed)
    sizes = [len(t) for t in trees]
    cu, parents = np.concatenate([[0], np.cumsum(sizes)]), np.asarray(sum(trees, []) + [0] * behind, np.int32)
    ctx = np.asarray(prior) + sizes
    mb = max(1, int(-(-ctx.max() // bs)))
    table = rng.permutation(len(trees) * mb).reshape(-1, mb).astype(np.int32)
    words = words or max(1, -(-max(sizes) // 32))
    lens = np.maximum(ctx - short, 0)
    mask, positions, slots = run_layout(kernels, device, cu, parents, lens, table, bs, max(sizes), words, text)
    for s, tree in enumerate(trees):
        sees = ancestors(tree)
        rows = slice(cu[s], cu[s + 1])
        first = max(int(lens[s]) - len(tree), 0)
        np.testing.assert_array_equal(mask[rows], words_of(sees, words))
        root = first if text is None else text[s]
        np.testing.assert_array_equal(positions[rows], root + sees.sum(1) - 1)
        at = first + np.arange(len(tree))
        want = np.where(at < lens[s], table[s, np.minimum(at, mb * bs - 1) // bs] * bs + at % bs, -1)
        np.testing.assert_array_equal(slots[rows], want)
    assert (mask[cu[-1]:] == -7).all() and (positions[cu[-1]:] == -7).all() and (slots[cu[-1]:] == -7).all()


@pytest.mark.parametrize("sizes", [[1], [2], [0, 1, 0], [31, 32, 33], [64], [65, 3, 128], [256, 255, 257, 1], [1024, 1000]])
@pytest.mark.parametrize("depth", [1, 6, 2000])
def test_layout(device, kernels, sizes, depth):
    rng = np.random.default_rng(sum(sizes) + depth)
    trees = [random_tree(rng, n, depth) for n in sizes]
    check_layout(kernels, device, trees, rng.integers(0, 300, len(sizes)), seed=depth)


@pytest.mark.parametrize("n", [2, 33, 256, 1024])
def test_layout_of_a_chain(device, kernels, n):
    """As deep as it can be, and every node its own tree."""
    check_layout(kernels, device, [list(range(-1, n - 1)), [-1] * n], [5, 9])


@pytest.mark.parametrize("bs", [1, 5, 16, 32, 256])
def test_layout_blocks(device, kernels, bs):
    rng = np.random.default_rng(bs)
    trees = [random_tree(rng, n, 5, roots=3) for n in (40, 7, 90)]
    check_layout(kernels, device, trees, [0, 31, 250], bs, text=[1000, 31, 7], words=9, behind=5)


def test_layout_parents_that_are_none(device, kernels):
    """A node itself, a later one, something far off: no parent."""
    tree = [0, 0, 2, 5, 1000000, -2**31, 4, 2**31 - 1]
    check_layout(kernels, device, [tree, [5, -1]], [3, 0])


@pytest.mark.parametrize("short", [1, 3, 400])
def test_layout_short_contexts(device, kernels, short):
    """Lengths that do not count all of the tree: no slot for the nodes that they leave out."""
    rng = np.random.default_rng(short)
    check_layout(kernels, device, [random_tree(rng, 6), random_tree(rng, 2)], [0, 20], short=short)


def test_layout_many(device, kernels):
    rng = np.random.default_rng(1)
    check_layout(kernels, device, [random_tree(rng, int(n)) for n in rng.integers(0, 70, 700)], rng.integers(0, 99, 700))


# ------------------------------------------------------------ verification --


def run_verify(kernels, device, logits, draft, parents, cu, most, target=None, rows=None):
    seqs, n = len(cu) - 1, len(parents)
    outs = [torch.full(s, -9, dtype=torch.int32, device=device) for s in ((seqs, most), (seqs,), (seqs,))]
    common = (i32(draft, device), i32(parents, device), i32(cu, device), int(np.diff(cu).max()))
    if target is None:
        tokens = torch.full((n,), -9, dtype=torch.int32, device=device)
        nbytes = kernels.verify_tree_workspace_bytes(n, logits.shape[1])
        ws = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=device)
        kernels.launch_verify_tree(logits, *common, tokens, *outs, workspace=ws)
    else:
        tokens = i32(target, device)
        kernels.launch_accept_tree(tokens, *common, *outs)
    return [t.cpu().numpy() for t in (tokens, *outs)]


def check_verify(kernels, device, trees, logits, agree=0.8, most=6, behind=0, seed=0, sampled=None):
    rng = np.random.default_rng(seed)
    cu = np.concatenate([[0], np.cumsum([len(t) for t in trees])])
    parents = np.asarray(sum(trees, []) + [0] * behind, np.int32)
    real = int(cu[-1])
    if sampled is None:
        x = logits.float().cpu().numpy()
        target = np.array([first_largest(r) for r in x[:real]] + [0] * behind, np.int64)
    else:
        target = sampled
    draft = rng.integers(0, 3, len(parents))
    for s, t in enumerate(trees):
        for j, p in enumerate(t):
            if 0 <= p < j and rng.random() < agree:
                draft[cu[s] + j] = target[cu[s] + p]
    got = run_verify(kernels, device, logits, draft, parents, cu, most, sampled)
    if sampled is None:
        np.testing.assert_array_equal(got[0][:real], target[:real])
        assert (got[0][real:] == -9).all()
    lengths = []
    for s, t in enumerate(trees):
        path, following = accept(t, draft[cu[s]:cu[s + 1]], target[cu[s]:cu[s + 1]], most)
        np.testing.assert_array_equal(got[1][s], path + [-1] * (most - len(path)))
        assert got[2][s] == len(path) and got[3][s] == following
        lengths.append(len(path))
    return lengths


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 3, 7, 8, 9, 63, 1000, 4096, 32000, 49999, 128256])
def test_verify(device, kernels, dtype, vocab):
    """Few values and many ties; rows on 16 bytes and not."""
    rng = np.random.default_rng(vocab)
    trees, _, parents = forest(rng, [7, 0, 1, 20, 33])
    g = torch.Generator(device=device).manual_seed(vocab)
    logits = torch.randint(-20, 20, (len(parents), vocab), device=device, generator=g).to(TORCH_DT[dtype]) / 4
    check_verify(kernels, device, trees, logits, seed=vocab)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("stride,offset", [(1001, 0), (1024, 0), (1003, 5), (2000, 3)])
def test_verify_strides(device, kernels, dtype, stride, offset):
    rng = np.random.default_rng(stride)
    trees, _, parents = forest(rng, [9, 30])
    base = torch.full((len(parents) * stride + 8,), 1e4, device=device).to(TORCH_DT[dtype])
    logits = base[offset:offset + len(parents) * stride].view(-1, stride)[:, :1000]
    logits.copy_(torch.randn(len(parents), 1000, device=device, generator=torch.Generator(device).manual_seed(1)))
    check_verify(kernels, device, trees, logits)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_verify_special_values(device, kernels, dtype):
    """Infinities, NaN, signed zeros, rows of nothing else: the first of the largest."""
    nan, inf = float("nan"), float("inf")
    rows = [[nan] * 40, [-inf] * 40, [nan] * 5 + [-inf] * 35, [nan] * 20 + [-3.0] + [nan] * 19, [-0.0] * 7 + [0.0] * 33,
            [-1.0] * 11 + [0.0] + [-0.0] * 28, [-1.0] * 11 + [-0.0] + [0.0] * 28, [1.0] * 3 + [inf] * 2 + [nan] * 35,
            [-inf] * 39 + [-5.0], [0.0] * 39 + [nan], [-5.0] + [-inf] * 39, [nan] * 39 + [inf]]
    logits = torch.tensor(rows, device=device).to(TORCH_DT[dtype])
    tree = list(range(-1, len(rows) - 1))
    for _ in range(2):
        check_verify(kernels, device, [tree], logits, agree=1.0, most=20)
        logits = torch.cat([logits, logits[:, :3].abs() * nan], 1)      # the same, off the 16 bytes


@pytest.mark.parametrize("place", [0, 1, 8, 4095, 4096, 60000, 128254, 128255])
def test_verify_ties_far_apart(device, kernels, place):
    """Of equal largest logits the first, whichever split of the row has it."""
    logits = torch.zeros((1, 128256), device=device, dtype=torch.bfloat16)
    logits[0, place:] = torch.where(torch.arange(128256 - place, device=device) % 1000 == 0, 3.0, 1.0).to(torch.bfloat16)
    check_verify(kernels, device, [[-1]], logits)


@pytest.mark.parametrize("most", [1, 2, 12])
def test_accept(device, kernels, most):
    """Given targets; twin children, roots beside node 0 (never accepted), the most that is asked for."""
    rng = np.random.default_rng(most)
    sizes = [0, 1, 2, 40, 200, 1024, 33] * 20
    trees = [random_tree(rng, n, 9, roots=1 + n % 3) for n in sizes]
    n = sum(sizes)
    lengths = check_verify(kernels, device, trees, None, agree=0.9, most=most, behind=9, seed=most,
                           sampled=rng.integers(0, 3, n + 9))
    assert max(lengths) == min(most, 10) or most > 9


def test_accept_whole_chain(device, kernels):
    chain = list(range(-1, 1023))
    check_verify(kernels, device, [chain, chain[:500]], None, agree=1.0, most=1024, sampled=np.arange(1524) % 7)


def test_verify_many_rows(device, kernels):
    rng = np.random.default_rng(3)
    trees, _, parents = forest(rng, rng.integers(0, 40, 150))
    g = torch.Generator(device=device).manual_seed(3)
    check_verify(kernels, device, trees, torch.randint(0, 9, (len(parents) + 11, 777), device=device,
                                                       generator=g).to(torch.bfloat16), behind=11)


def test_verify_without_nodes(device, kernels):
    outs = [torch.full(s, 3, dtype=torch.int32, device=device) for s in ((2, 4), (2,), (2,))]
    none = torch.zeros(0, dtype=torch.int32, device=device)
    cu = torch.zeros(3, dtype=torch.int32, device=device)
    kernels.launch_verify_tree(torch.zeros((0, 50), device=device), none, none, cu, 0, none, *outs)
    assert (outs[0] == -1).all() and (outs[1] == 0).all() and (outs[2] == -1).all()


# -------------------------------------------------------------- compaction --


def check_compact(kernels, device, prior, sizes, paths, dtype="bf16", layers=2, hkv=2, d=64, bs=16, scores=True,
                  fused=True, most=None, seed=0):
    rng = np.random.default_rng(seed)
    prior, sizes = np.asarray(prior), np.asarray(sizes)
    ctx = prior + sizes
    mb = max(1, int(-(-ctx.max() // bs)))
    blocks = len(ctx) * mb + 2
    table = rng.permutation(blocks)[:len(ctx) * mb].reshape(-1, mb).astype(np.int32)
    g = torch.Generator(device=device).manual_seed(seed)
    pool = torch.randn((layers, blocks, 2, hkv, bs, d), generator=g, device=device).to(TORCH_DT[dtype])
    k, v = pool[:, :, 0], pool[:, :, 1]
    if not fused:
        k, v = k.contiguous(), v.contiguous()
    cells = torch.randn((layers, blocks, hkv, bs), generator=g, device=device) if scores else None
    most = most or max(1, max(len(p) for p in paths))
    accepted = np.full((len(ctx), most), -1, np.int32)
    for s, p in enumerate(paths):
        accepted[s, :len(p)] = p[:most]
    count = [len(p) for p in paths]
    want = [x.clone() for x in (k, v) + ((cells,) if scores else ())]
    for s, p in enumerate(paths):
        src = prior[s] + np.asarray(p, np.int64)
        dst = prior[s] + np.arange(len(p))
        real = (np.asarray(p) >= 0) & (np.asarray(p) < sizes[s]) if len(p) else np.zeros(0, bool)
        sb, so = (torch.as_tensor(a, device=device) for a in (table[s, src[real] // bs].astype(np.int64), src[real] % bs))
        db, do = (torch.as_tensor(a, device=device) for a in (table[s, dst[real] // bs].astype(np.int64), dst[real] % bs))
        for x in want:
            x[:, db, :, do] = x[:, sb, :, so].clone()
    lens = torch.full((len(ctx),), -1, dtype=torch.int32, device=device)
    args = [i32(a, device) for a in (table, ctx, np.concatenate([[0], np.cumsum(sizes)]), accepted, count)]
    kernels.launch_compact_tree(k, v, cells, *args, lens)
    for x, w in zip((k, v, cells), want):
        assert torch.equal(x, w)
    np.testing.assert_array_equal(lens.cpu().numpy(), prior + np.asarray(count))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 16), (2, 64, 32), (3, 20, 5), (1, 1, 1), (4, 80, 16), (2, 7, 3), (16, 256, 16)])
def test_compact(device, kernels, dtype, hkv, d, bs):
    """Nothing, the root, a path in place, one that steps over what others leave, the last node alone."""
    check_compact(kernels, device, [20, 0, 7, 33, 0, 15], [12, 3, 6, 20, 0, 9],
                  [[0, 2, 5, 11], [0], [0, 1, 2], [0, 1, 4, 5, 6, 7, 19], [], [8]], dtype, 3, hkv, d, bs, seed=d)


@pytest.mark.parametrize("n", [8, 9, 63, 64, 65, 130, 700])
def test_compact_long_paths(device, kernels, n):
    """Every source is a later destination: by one place, and by a growing number of them."""
    step = np.sort(np.random.default_rng(n).choice(np.arange(1, 1024), n, replace=False))
    check_compact(kernels, device, [3, 50], [n + 1, 1024], [list(range(1, n + 1)), list(step)], d=32, seed=n)


def test_compact_without_scores(device, kernels):
    check_compact(kernels, device, [20, 5], [9, 9], [[0, 3, 4], [0, 8]], scores=False, fused=False)


def test_compact_entries_outside(device, kernels):
    """Entries that are no node of the tree are not moved."""
    check_compact(kernels, device, [20, 0], [9, 4], [[0, -1, 4, 9, 2**30, 8], [0, -5, 3]])


def test_compact_many(device, kernels):
    rng = np.random.default_rng(2)
    sizes = rng.integers(1, 40, 90)
    paths = [list(np.sort(rng.choice(n, rng.integers(0, n) + 1, replace=False))) for n in sizes]
    check_compact(kernels, device, rng.integers(0, 60, 90), sizes, paths, layers=5, d=64, seed=4)


def test_compact_far_blocks(device, kernels):
    """Blocks, layers and offsets past 2^32 elements."""
    hkv, bs, d = 8, 16, 128
    nb = (1 << 32) // (2 * hkv * bs * d) + 9
    pool = torch.zeros((2, nb, 2, hkv, bs, d), dtype=torch.float16, device=device)
    table = np.array([[nb - 1, nb - 2]], np.int32)
    for layer in range(2):
        for t in range(30):
            pool[layer, table[0, t // bs], :, :, t % bs] = 100 * layer + t
    args = [i32(a, device) for a in (table, [30], [0, 20], [[0, 5, 19]], [3])]
    kernels.launch_compact_tree(pool[:, :, 0], pool[:, :, 1], None, *args, None)
    for layer in range(2):
        got = [float(x) for x in pool[layer, nb - 1, 1, 7, 10:14, 127]]
        assert got == [100 * layer + t for t in (10, 15, 29, 13)]


def test_refusals(device, kernels):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
    layout = dict(parents=i(4), cu_nodes=i(3), context_lens=i(2), block_table=i(2, 3), tree_mask=i(4, 1), positions=i(4),
                  slot_mapping=i(4), block_size=16, max_nodes=4)
    kernels.launch_tree_layout(**layout)
    for change in [dict(parents=i(3)), dict(positions=i(5)), dict(cu_nodes=i(0)), dict(context_lens=i(3)),
                   dict(block_table=i(3, 3)), dict(tree_mask=i(3, 1)), dict(max_nodes=33), dict(max_nodes=-1),
                   dict(block_size=0), dict(text_positions=i(1)), dict(text_positions=i(2).long()),
                   dict(parents=i(4).cpu()), dict(slot_mapping=i(4).long()), dict(tree_mask=i(1, 4).t()[:, :1].expand(4, 2)),
                   dict(max_nodes=1025, tree_mask=i(4, 40))]:
        with pytest.raises(RailgunError):
            kernels.launch_tree_layout(**{**layout, **change})
    verify = dict(logits=torch.zeros((4, 9), device=device), draft_tokens=i(4), parents=i(4), cu_nodes=i(3), max_nodes=4,
                  target_tokens=i(4), accepted=i(2, 3), num_accepted=i(2), next_tokens=i(2))
    kernels.launch_verify_tree(**verify)
    for change in [dict(logits=torch.zeros((3, 9), device=device)), dict(logits=torch.zeros((4, 0), device=device)),
                   dict(logits=torch.zeros((9, 4), device=device).t()), dict(logits=torch.zeros((1, 9), device=device).expand(4, 9)),
                   dict(logits=torch.zeros((4, 9), device=device, dtype=torch.float64)), dict(draft_tokens=i(5)),
                   dict(accepted=i(2, 0)), dict(accepted=i(3, 3)), dict(num_accepted=i(1)), dict(next_tokens=i(3)),
                   dict(target_tokens=i(4).long()), dict(max_nodes=1025),
                   dict(workspace=torch.empty(8, dtype=torch.uint8, device=device))]:
        with pytest.raises(RailgunError):
            kernels.launch_verify_tree(**{**verify, **change})
    pool = torch.zeros((2, 6, 2, 2, 16, 64), device=device)
    compact = dict(key_cache=pool[:, :, 0], value_cache=pool[:, :, 1], scores=None, block_table=i(2, 3), context_lens=i(2),
                   cu_nodes=i(3), accepted=i(2, 3), num_accepted=i(2), new_context_lens=i(2))
    kernels.launch_compact_tree(**compact)
    lens = i(2)
    for change in [dict(key_cache=pool[:, :, 0, :, :, :32]), dict(value_cache=pool[:1, :, 1]), dict(accepted=i(3, 3)),
                   dict(num_accepted=i(3)), dict(new_context_lens=i(1)), dict(scores=torch.zeros((2, 6, 2, 15), device=device)),
                   dict(context_lens=lens, new_context_lens=lens), dict(num_accepted=lens, new_context_lens=lens),
                   dict(block_table=i(2, 3).cpu()), dict(key_cache=pool[:, :1, 0].expand(-1, 6, -1, -1, -1),
                                                         value_cache=pool[:, :1, 1].expand(-1, 6, -1, -1, -1))]:
        with pytest.raises(RailgunError):
            kernels.launch_compact_tree(**{**compact, **change})


def test_captured(device, kernels):
    """Layout, verification and compaction replayed as one graph on other contents."""
    rng = np.random.default_rng(5)
    pool = GpuBlockPool(2, 40, 2, 16, 64, device, fill=torch.Generator(device).manual_seed(1), kernels=kernels)
    table = i32(rng.permutation(40)[:12].reshape(3, 4), device)
    cu, ctx = i32([0, 12, 12, 30], device), i32([40, 0, 50], device)
    parents, draft = i32(np.zeros(30), device), i32(np.zeros(30), device)
    logits = torch.zeros((30, 500), device=device, dtype=torch.bfloat16)
    mask, positions, slots, target = (torch.zeros(s, dtype=torch.int32, device=device) for s in ((30, 1), 30, 30, 30))
    accepted, count, following, lens = (torch.zeros(s, dtype=torch.int32, device=device) for s in ((3, 6), 3, 3, 3))

    def step():
        kernels.launch_tree_layout(parents, cu, ctx, table, mask, positions, slots, 16, 18)
        kernels.launch_verify_tree(logits, draft, parents, cu, 18, target, accepted, count, following)
        kernels.launch_compact_tree(pool.storage[:, :, 0], pool.storage[:, :, 1], None, table, ctx, cu, accepted, count,
                                    lens)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for seed in range(3):
        r = np.random.default_rng(seed)
        parents.copy_(i32(random_tree(r, 12) + random_tree(r, 18), device))
        logits.copy_(torch.randint(0, 4, (30, 500), device=device))
        draft.copy_(torch.randint(0, 5, (30,), device=device))
        before = pool.storage.clone()
        outs = (mask, positions, slots, target, accepted, count, following, lens)
        g.replay()
        torch.cuda.synchronize()
        got, after = [t.clone() for t in outs], pool.storage.clone()
        pool.storage.copy_(before)
        for t in outs:
            t.fill_(-3)
        step()
        torch.cuda.synchronize()
        assert torch.equal(pool.storage, after) and all(torch.equal(a, b) for a, b in zip(got, outs))
