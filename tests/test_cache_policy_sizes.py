"""Size queries of the shared-prefix, scoring and eviction entries at sizes that the entries refuse: host
arithmetic, run without a GPU."""
from __future__ import annotations

import pytest

import railgun_amd
from railgun_amd import _lib

BF16 = _lib.RG_DTYPE_BF16
TOP = 2**31 - 1


@pytest.mark.parametrize("batch,heads,kv_heads,d,bs,mb,shared", [
    (2**30, 32, 8, 128, 16, 40, 20),         # rows (batch x heads to a kv-head) past 32 bits: 2^32 of them
    (TOP, 32, 8, 128, 16, 40, 20),
    (65535, 2**20, 1, 128, 16, 40, 20),
    (65536, 32, 8, 128, 16, 40, 20),         # more sequences than a grid has
    (4, 32, 8, 128, TOP, TOP, TOP),          # prefix tokens past 32 bits
    (4, 32, 8, 128, 32, 2**27, 2**27),
    (4, 32, 8, 128, 16, 2**27, 1),
])
def test_shared_prefix_sizes_past_the_entry(batch, heads, kv_heads, d, bs, mb, shared):
    lib = railgun_amd.load_library()
    shape = (batch, heads, kv_heads, d, bs, mb, shared)
    assert lib.rg_paged_attention_shared_prefix_workspace_bytes(*shape) == 0
    assert lib.rg_paged_attention_shared_prefix_pays(*shape, BF16) == 0


def test_shared_prefix_sizes_at_the_limits():
    lib = railgun_amd.load_library()
    for shape in ((65535, 32, 8, 128, 16, 40, 20), (2, 32, 8, 128, 16, 2**27 - 1, 2**27 - 1),
                  (1, TOP, 1, 4, 16, 4, 2), (65535, 32767, 1, 4, 16, 4, 2)):
        assert lib.rg_paged_attention_shared_prefix_workspace_bytes(*shape) > 0
        assert lib.rg_paged_attention_shared_prefix_pays(*shape, BF16) in (0, 1)


@pytest.mark.parametrize("batch,heads,kv_heads,d,bs,mb", [
    (65536, 32, 8, 128, 16, 40), (3, 65536, 8, 128, 16, 40), (3, 32, 8, 128, TOP, TOP), (3, 32, 8, 128, 16, 2**27),
    (65535, 65535, 65535, 128, 16, 2**26),   # raw scores of 2^62 tokens and heads: more bytes than 64 bits count
    (65535, 65535, 65535, 128, 16, 2**20),
])
def test_scores_sizes_past_the_entry(batch, heads, kv_heads, d, bs, mb):
    lib = railgun_amd.load_library()
    assert lib.rg_paged_attention_v1_scores_workspace_bytes(batch, heads, kv_heads, d, bs, mb) == 0
    p = 64  # never followed
    st = lib.rg_paged_attention_v1_scores(p, p, p, p, p, p, p, None, 0, 0.1, heads, kv_heads, d, bs, mb, batch, BF16, 0,
                                          0, p, 0, None)
    assert st == _lib.RG_ERR_NOT_SUPPORTED, _lib.last_error()


def test_scores_sizes_at_the_limits():
    f = railgun_amd.load_library().rg_paged_attention_v1_scores_workspace_bytes
    assert f(4096, 4096, 4096, 128, 16, 2**20) >= 4 << 48
    assert f(1, 32, 8, 128, 16, 2**27 - 1) >= 4 * 32 * 16 * (2**27 - 1)


@pytest.mark.parametrize("budget,kept,need", [(64, None, 256 + 48 * 64 * 4), (160, None, 256 + 48 * 160 * 4),
                                              (161, None, 256 + 48 * 160 * 4), (TOP, None, 256 + 48 * 160 * 4),
                                              (TOP, 64, 256)])
def test_eviction_asks_for_no_more_than_the_table_holds(budget, kept, need):
    """Ten blocks of 16 tokens, 48 segments: the call with one byte less says what it needs."""
    p = 64  # never followed
    st = railgun_amd.load_library().rg_evict_cache(p, p, p, p, None, p, None, kept, budget, 8, 4, 2, 8, 64, 16, 10, 0, 3,
                                                   BF16, 1 << 20, 0, 1 << 14, 0, p, need - 1, None)
    assert st == _lib.RG_ERR_WORKSPACE and f"{need} required" in _lib.last_error()
