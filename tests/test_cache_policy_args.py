"""Argument checks of the shared-prefix, scoring and eviction entries: they return before any HIP
call, so they run without a GPU."""
from __future__ import annotations

import numpy as np
import pytest

import railgun_amd
from railgun_amd import _lib

INVALID, UNSUPPORTED, WORKSPACE = _lib.RG_ERR_INVALID_ARGUMENT, _lib.RG_ERR_NOT_SUPPORTED, _lib.RG_ERR_WORKSPACE
P = np.zeros(64, np.float32).ctypes.data  # any non-null, 4-byte aligned address: never followed


def call(name, *args):
    return getattr(railgun_amd.load_library(), name)(*args), _lib.last_error()


def evict(**change):
    a = dict(k=P, v=P, scores=P, table=P, dst=P, lens=P, new_lens=P, kept=P, budget=64, recent=8, protected=4, layers=2,
             kv_heads=8, d=64, bs=16, mb=10, mdb=4, batch=3, dtype=_lib.RG_DTYPE_BF16, layer_stride=1 << 20,
             kv_stride=0, score_layer_stride=1 << 14, score_stride=0, ws=P, ws_bytes=256, stream=None)
    assert set(change) <= set(a)
    return call("rg_evict_cache", *{**a, **change}.values())


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=9), UNSUPPORTED, "unknown dtype"),
    (dict(d=0), UNSUPPORTED, "head_dim"),
    (dict(d=257), UNSUPPORTED, "head_dim"),
    (dict(batch=-1), INVALID, "batch"),
    (dict(layers=-1), INVALID, "num_layers"),
    (dict(kv_heads=0), INVALID, "positive heads"),
    (dict(bs=0), INVALID, "block_size"),
    (dict(mb=-1), INVALID, "table widths"),
    (dict(mdb=-1), INVALID, "table widths"),
    (dict(budget=0), INVALID, "budget >= 1"),
    (dict(recent=-1), INVALID, "recent"),
    (dict(protected=-1), INVALID, "recent"),
    (dict(recent=61), INVALID, "<= budget"),
    (dict(recent=2**31 - 1, protected=2**31 - 1), INVALID, "<= budget"),
    (dict(kv_stride=8 * 16 * 64 - 1), INVALID, "smaller than a block"),
    (dict(score_stride=8 * 16 - 1), INVALID, "smaller than a block"),
    (dict(layer_stride=0), INVALID, "layer strides"),
    (dict(score_layer_stride=-5), INVALID, "layer strides"),
    (dict(mdb=3), INVALID, "destination rows"),
    (dict(mb=2**31 - 1), UNSUPPORTED, "block table of"),
    (dict(k=None), INVALID, "null pointer"),
    (dict(scores=None), INVALID, "null pointer"),
    (dict(table=None), INVALID, "null pointer"),
    (dict(lens=None), INVALID, "null pointer"),
    (dict(layers=2**16, batch=2**16), UNSUPPORTED, "segments"),
    (dict(ws=None), WORKSPACE, "required"),
    (dict(ws_bytes=255), WORKSPACE, "256 required"),
    (dict(ws=P + 2), WORKSPACE, "aligned"),
    (dict(kept=None), WORKSPACE, "required"),          # the list goes to the workspace then
    (dict(), INVALID, "overlaps"),                      # lengths read while the new ones are written
    (dict(new_lens=P + 8), INVALID, "overlaps"),
    (dict(new_lens=P - 8), INVALID, "overlaps"),
    (dict(mb=2**27 - 1), UNSUPPORTED, "block table of"),
    (dict(layers=0), _lib.RG_OK, ""),
    (dict(batch=0), _lib.RG_OK, ""),
])
def test_evict_arguments(change, code, text):
    st, msg = evict(**change)
    assert st == code and text in msg, msg


def test_evict_workspace_bytes():
    f = railgun_amd.load_library().rg_evict_cache_workspace_bytes
    assert f(2, 3, 8, 64) == 256 + 48 * 64 * 4
    assert f(0, 3, 8, 64) == f(2, 0, 8, 64) == f(2, 3, 8, 0) == f(2**20, 2**20, 1, 1) == 0


def scores(**change):
    a = dict(q=P, k=P, v=P, table=P, lens=P, out=P, scores=P, scored=P, first=0, scale=0.125, heads=8, kv_heads=2, d=64,
             bs=16, mb=4, batch=3, dtype=_lib.RG_DTYPE_BF16, kv_stride=0, score_stride=0, ws=P, ws_bytes=1 << 30,
             stream=None)
    assert set(change) <= set(a)
    return call("rg_paged_attention_v1_scores", *{**a, **change}.values())


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=9), UNSUPPORTED, "unknown dtype"),
    (dict(d=66), UNSUPPORTED, "multiple of 4"),
    (dict(d=260), UNSUPPORTED, "multiple of 4"),
    (dict(heads=7), INVALID, "not a multiple"),
    (dict(kv_heads=0), INVALID, "positive heads"),
    (dict(batch=-1), INVALID, "batch"),
    (dict(mb=-1), INVALID, "max_blocks"),
    (dict(heads=1026), UNSUPPORTED, "query heads to a kv-head"),
    (dict(first=-1), INVALID, "first_scored"),
    (dict(kv_stride=2 * 16 * 64 - 1), INVALID, "kv_block_stride"),
    (dict(score_stride=31), INVALID, "score_block_stride"),
    (dict(mb=2**31 - 1), UNSUPPORTED, "block table of"),
    (dict(batch=65536), UNSUPPORTED, "sequences"),
    (dict(q=None), INVALID, "null pointer"),
    (dict(scores=None), INVALID, "null pointer"),
    (dict(lens=None), INVALID, "null pointer"),
    (dict(ws=None), WORKSPACE, "required"),
    (dict(ws_bytes=1000), WORKSPACE, "required"),
    (dict(ws=P // 16 * 16 + 4), WORKSPACE, "aligned"),
    (dict(batch=0), _lib.RG_OK, ""),
])
def test_scores_arguments(change, code, text):
    st, msg = scores(**change)
    assert st == code and text in msg, msg


def test_scores_workspace_bytes():
    f = railgun_amd.load_library().rg_paged_attention_v1_scores_workspace_bytes
    assert f(3, 8, 2, 64, 16, 4) > 3 * 8 * 64 * 4 and f(3, 8, 2, 64, 16, 4) % 256 == 0
    assert f(0, 8, 2, 64, 16, 4) == f(3, 7, 2, 64, 16, 4) == f(3, 8, 2, 64, 16, 0) == 0


def shared(**change):
    a = dict(q=P, k=P, v=P, table=P, lens=P, out=P, scale=0.125, heads=8, kv_heads=2, d=64, bs=16, mb=4, batch=3,
             shared_blocks=2, dtype=_lib.RG_DTYPE_BF16, kv_stride=0, ws=P, ws_bytes=1 << 30, stream=None)
    assert set(change) <= set(a)
    return call("rg_paged_attention_shared_prefix", *{**a, **change}.values())


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=9), UNSUPPORTED, "unknown dtype"),
    (dict(d=66), UNSUPPORTED, "multiple of 4"),
    (dict(d=260), UNSUPPORTED, "multiple of 4"),
    (dict(heads=7), INVALID, "not a multiple"),
    (dict(bs=0), INVALID, "block_size"),
    (dict(batch=-1), INVALID, "batch"),
    (dict(shared_blocks=-1), INVALID, "shared_blocks"),
    (dict(shared_blocks=5), INVALID, "shared_blocks"),
    (dict(kv_stride=2 * 16 * 64 - 1), INVALID, "kv_block_stride"),
    (dict(mb=2**31 - 1), UNSUPPORTED, "block table of"),
    (dict(batch=65536), UNSUPPORTED, "sequences"),
    (dict(q=None), INVALID, "null pointer"),
    (dict(table=None), INVALID, "null pointer"),
    (dict(out=None), INVALID, "null pointer"),
    (dict(ws=None), WORKSPACE, "required"),
    (dict(ws_bytes=1000), WORKSPACE, "required"),
    (dict(ws=P // 16 * 16 + 4), WORKSPACE, "aligned"),
    (dict(batch=0), _lib.RG_OK, ""),
])
def test_shared_prefix_arguments(change, code, text):
    st, msg = shared(**change)
    assert st == code and text in msg, msg


def test_shared_prefix_workspace_bytes():
    f = railgun_amd.load_library().rg_paged_attention_shared_prefix_workspace_bytes
    assert f(3, 8, 2, 64, 16, 40, 20) >= railgun_amd.load_library().rg_paged_attention_v1_workspace_bytes(3, 8, 2, 64, 16, 40)
    assert f(0, 8, 2, 64, 16, 4, 2) == f(3, 7, 2, 64, 16, 4, 2) == f(3, 8, 2, 64, 16, 4, 5) == 0


def test_shared_prefix_pays():
    f = railgun_amd.load_library().rg_paged_attention_shared_prefix_pays
    assert f(64, 32, 8, 128, 16, 200, 128, _lib.RG_DTYPE_BF16) == 1
    assert f(1, 32, 8, 128, 16, 2000, 1280, _lib.RG_DTYPE_BF16) == 0    # one sequence
    assert f(3, 32, 8, 64, 16, 9, 6, _lib.RG_DTYPE_F32) == 0            # little to save
    assert f(64, 32, 8, 96, 16, 200, 128, _lib.RG_DTYPE_BF16) == 0      # no such tile
    assert f(64, 32, 7, 128, 16, 200, 128, _lib.RG_DTYPE_BF16) == f(64, 32, 8, 128, 16, 200, 201, _lib.RG_DTYPE_BF16) == 0
    assert f(64, 32, 8, 128, 16, 200, 0, _lib.RG_DTYPE_BF16) == f(64, 32, 8, 128, 16, 200, 128, 9) == 0
