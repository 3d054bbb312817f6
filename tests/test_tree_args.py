"""Argument checks of the entries for steps over drafted tokens: they return before any HIP call, so they
run without a GPU."""
from __future__ import annotations

import numpy as np
import pytest

import railgun_amd
from railgun_amd import _lib

INVALID, UNSUPPORTED, WORKSPACE = _lib.RG_ERR_INVALID_ARGUMENT, _lib.RG_ERR_NOT_SUPPORTED, _lib.RG_ERR_WORKSPACE
BUF = np.zeros(64, np.float64)
P = BUF.ctypes.data + 16 - BUF.ctypes.data % 16  # a non-null, 16-byte aligned address: never followed
BF16 = _lib.RG_DTYPE_BF16


def call(name, defaults, change):
    assert set(change) <= set(defaults)
    lib = railgun_amd.load_library()
    return getattr(lib, name)(*{**defaults, **change}.values()), _lib.last_error()


def expect(got, code, text):
    assert got[0] == code and text in got[1], got


LAYOUT = dict(parents=P, cu=P, lens=P, table=P, text=None, mask=P, positions=P, slots=P, bs=16, mb=4, seqs=2, nodes=9,
              most=6, words=1, stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(most=-1), INVALID, "max_nodes"), (dict(most=1025, words=33), UNSUPPORTED, "1024"),
    (dict(words=0), INVALID, "mask_words"), (dict(most=33), INVALID, "mask_words"), (dict(words=33), INVALID, "mask_words"),
    (dict(seqs=-1), INVALID, "num_seqs"), (dict(nodes=-1), INVALID, "num_nodes"), (dict(bs=0), INVALID, "block_size"),
    (dict(mb=-1), INVALID, "max_blocks"), (dict(mb=2**31 - 1), UNSUPPORTED, "block table"),
    (dict(parents=None), INVALID, "null"), (dict(cu=None), INVALID, "null"), (dict(lens=None), INVALID, "null"),
    (dict(table=None), INVALID, "null"), (dict(mask=None), INVALID, "null"), (dict(positions=None), INVALID, "null"),
    (dict(slots=None), INVALID, "null"),
])
def test_layout_refusals(change, code, text):
    expect(call("rg_tree_layout", LAYOUT, change), code, text)


ATTENTION = dict(q=P, k=P, v=P, table=P, lens=P, cu=P, mask=P, out=P, scale=1.0, heads=8, hkv=2, d=64, bs=16, mb=4, seqs=2,
                 nodes=9, most=6, words=1, dtype=BF16, stride=0, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=7), UNSUPPORTED, "dtype"), (dict(d=66), UNSUPPORTED, "head_dim"), (dict(d=260), UNSUPPORTED, "head_dim"),
    (dict(d=0), UNSUPPORTED, "head_dim"), (dict(heads=0), INVALID, "heads"), (dict(hkv=0), INVALID, "heads"),
    (dict(heads=7), INVALID, "multiple"), (dict(bs=0), INVALID, "block_size"), (dict(mb=-1), INVALID, "max_blocks"),
    (dict(seqs=-1), INVALID, "num_seqs"), (dict(nodes=-1), INVALID, "num_nodes"), (dict(most=-1), INVALID, "max_nodes"),
    (dict(most=1025, words=40), UNSUPPORTED, "1024"), (dict(most=33), INVALID, "mask_words"),
    (dict(words=-1), INVALID, "mask_words"), (dict(stride=2 * 16 * 64 - 1), INVALID, "smaller than a block"),
    (dict(mb=2**27), UNSUPPORTED, "block table"), (dict(seqs=65536), UNSUPPORTED, "65536 sequences"),
    (dict(q=None), INVALID, "null"), (dict(k=None), INVALID, "null"), (dict(v=None), INVALID, "null"),
    (dict(table=None), INVALID, "null"), (dict(lens=None), INVALID, "null"), (dict(cu=None), INVALID, "null"),
    (dict(mask=None), INVALID, "null"), (dict(out=None), INVALID, "null"),
])
def test_attention_refusals(change, code, text):
    expect(call("rg_paged_attention_tree", ATTENTION, change), code, text)


VERIFY = dict(logits=P, draft=P, parents=P, cu=P, target=P, accepted=P, count=P, next=P, seqs=2, nodes=9, most=6, width=4,
              vocab=100, dtype=BF16, stride=100, ws=P, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(seqs=-1), INVALID, "num_seqs"), (dict(nodes=-1), INVALID, "num_nodes"), (dict(width=0), INVALID, "max_accepted"),
    (dict(most=-1), INVALID, "max_nodes"), (dict(most=1025), UNSUPPORTED, "1024"), (dict(dtype=3), UNSUPPORTED, "dtype"),
    (dict(vocab=0), INVALID, "vocabulary"), (dict(stride=99), INVALID, "row stride"), (dict(logits=None), INVALID, "null"),
    (dict(draft=None), INVALID, "null"), (dict(parents=None), INVALID, "null"), (dict(cu=None), INVALID, "null"),
    (dict(target=None), INVALID, "null"), (dict(accepted=None), INVALID, "null"), (dict(count=None), INVALID, "null"),
    (dict(next=None), INVALID, "null"), (dict(logits=P + 1), INVALID, "aligned"), (dict(ws=None), WORKSPACE, "required"),
    (dict(ws_bytes=9), WORKSPACE, "required"), (dict(ws=P + 4), WORKSPACE, "aligned"),
])
def test_verify_refusals(change, code, text):
    expect(call("rg_verify_tree", VERIFY, change), code, text)


ACCEPT = dict(target=P, draft=P, parents=P, cu=P, accepted=P, count=P, next=P, seqs=2, nodes=9, most=6, width=4, stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(seqs=-1), INVALID, "num_seqs"), (dict(nodes=-1), INVALID, "num_nodes"), (dict(width=0), INVALID, "max_accepted"),
    (dict(most=1025), UNSUPPORTED, "1024"), (dict(most=-2), INVALID, "max_nodes"), (dict(target=None), INVALID, "null"),
    (dict(draft=None), INVALID, "null"), (dict(parents=None), INVALID, "null"), (dict(cu=None), INVALID, "null"),
    (dict(accepted=None), INVALID, "null"), (dict(count=None), INVALID, "null"), (dict(next=None), INVALID, "null"),
])
def test_accept_refusals(change, code, text):
    expect(call("rg_accept_tree", ACCEPT, change), code, text)


COMPACT = dict(k=P, v=P, scores=P, table=P, lens=P, cu=P, accepted=P, count=P, new_lens=P + 64, width=4, layers=2, hkv=2,
               d=64, bs=16, mb=4, seqs=2, nodes=9, dtype=BF16, layer_stride=1 << 20, stride=0, score_layer_stride=1 << 14,
               score_stride=0, stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=9), UNSUPPORTED, "dtype"), (dict(d=0), UNSUPPORTED, "head_dim"), (dict(d=257), UNSUPPORTED, "head_dim"),
    (dict(layers=-1), INVALID, "layers"), (dict(seqs=-1), INVALID, "sequences"), (dict(nodes=-1), INVALID, "nodes"),
    (dict(hkv=0), INVALID, "positive"), (dict(bs=0), INVALID, "positive"), (dict(mb=-1), INVALID, "table"),
    (dict(width=0), INVALID, "max_accepted"), (dict(stride=5), INVALID, "smaller than a block"),
    (dict(score_stride=5), INVALID, "smaller than a block"), (dict(layer_stride=0), INVALID, "layer strides"),
    (dict(score_layer_stride=0), INVALID, "layer strides"), (dict(mb=2**31 - 1), UNSUPPORTED, "block table"),
    (dict(hkv=2**15, bs=2**10, stride=2**31), UNSUPPORTED, "elements"), (dict(layers=65536), UNSUPPORTED, "layers"),
    (dict(k=None), INVALID, "null"), (dict(v=None), INVALID, "null"), (dict(table=None), INVALID, "null"),
    (dict(lens=None), INVALID, "null"), (dict(cu=None), INVALID, "null"), (dict(accepted=None), INVALID, "null"),
    (dict(count=None), INVALID, "null"), (dict(new_lens=P), INVALID, "overlaps"), (dict(new_lens=P + 4), INVALID, "overlaps"),
    (dict(lens=P + 128, count=P + 160, accepted=P + 32, cu=P + 192, new_lens=P + 60), INVALID, "overlaps"),
    (dict(lens=P + 128, count=P + 160, accepted=P + 192, cu=P + 32, new_lens=P + 40), INVALID, "overlaps"),
])
def test_compact_refusals(change, code, text):
    expect(call("rg_compact_tree", COMPACT, change), code, text)


def test_nothing_to_do():
    """Calls of no sequence or layer return without looking at a pointer."""
    none = dict.fromkeys(["parents", "cu", "lens", "table", "mask", "positions", "slots"])
    assert call("rg_tree_layout", LAYOUT, dict(none, seqs=0))[0] == 0
    assert call("rg_tree_layout", LAYOUT, dict(none, nodes=0))[0] == 0
    for change in (dict(seqs=0), dict(nodes=0), dict(most=0)):
        assert call("rg_paged_attention_tree", ATTENTION, dict(change, q=None, k=None, ws=None))[0] == 0
    assert call("rg_verify_tree", VERIFY, dict(seqs=0, cu=None))[0] == 0
    assert call("rg_accept_tree", ACCEPT, dict(seqs=0, cu=None))[0] == 0
    assert call("rg_compact_tree", COMPACT, dict(layers=0, k=None))[0] == 0
    assert call("rg_compact_tree", COMPACT, dict(seqs=0, k=None))[0] == 0


def test_workspace_queries():
    lib = railgun_amd.load_library()
    assert lib.rg_verify_tree_workspace_bytes(0, 100) == 0 and lib.rg_verify_tree_workspace_bytes(5, 0) == 0
    assert lib.rg_verify_tree_workspace_bytes(1, 128256) >= 8
    assert lib.rg_verify_tree_workspace_bytes(2**31 - 1, 2**31 - 1) >= 8 * (2**31 - 1)
    for bad in ((-1, 6, 8, 2, 64, 16, 4), (2, 0, 8, 2, 64, 16, 4), (2, 6, 7, 2, 64, 16, 4), (2, 6, 8, 0, 64, 16, 4),
                (2, 2000, 8, 2, 64, 16, 4)):
        assert lib.rg_paged_attention_tree_workspace_bytes(*bad) == 0


def test_attention_of_more_pieces_than_a_grid_has():
    """Segments past the 2^32 threads of a grid go to the form that has a workgroup per node and head (no workspace)."""
    lib = railgun_amd.load_library()
    assert lib.rg_paged_attention_tree_workspace_bytes(65535, 1024, 64, 8, 128, 16, 40) == 0
    assert lib.rg_paged_attention_tree_workspace_bytes(32768, 1024, 64, 8, 128, 16, 40) == 0     # 2^24 segments
    assert lib.rg_paged_attention_tree_workspace_bytes(32000, 1024, 64, 8, 128, 16, 40) > 0


def test_compaction_refuses_lengths_over_the_block_table():
    """Every layer's workgroups read the table while the new lengths are written."""
    for at in (P + 60, P + 64, P + 92):                                # (two rows of four entries from P + 64 on)
        expect(call("rg_compact_tree", COMPACT, dict(table=P + 64, new_lens=at)), INVALID, "overlaps")
