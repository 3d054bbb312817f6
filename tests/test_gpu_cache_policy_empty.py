"""Block tables of no blocks: every sequence is empty, the size queries ask for nothing, and the entries write
zeros without a workspace, as rg_paged_attention_v1 does."""
from __future__ import annotations

import pytest
import torch

from railgun_amd import _lib
from railgun_amd.ops import dtype_code

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,hkv,d,bs", [(8, 2, 64, 16), (8, 2, 128, 32), (6, 3, 80, 5), (32, 2, 256, 16)])
@pytest.mark.parametrize("given", [0, 64])
def test_table_without_blocks(device, kernels, dtype, heads, hkv, d, bs, given):
    lib, b = kernels.lib, 3
    q = torch.randn((b, heads, d), device=device).to(dtype)
    cache = torch.zeros((1, hkv, bs, d), device=device, dtype=dtype)
    scores = torch.full((1, hkv, bs), 5.0, device=device)
    table = torch.zeros(4, dtype=torch.int32, device=device)  # (an address; nothing of it is an entry)
    lens = torch.zeros(b, dtype=torch.int32, device=device)
    ws = torch.empty(given, dtype=torch.uint8, device=device)
    ws_ptr = ws.data_ptr() if given else None
    stream = torch.cuda.current_stream(device).cuda_stream
    shape = (heads, hkv, d, bs, 0, b)
    assert lib.rg_paged_attention_v1_scores_workspace_bytes(b, heads, hkv, d, bs, 0) == 0
    assert lib.rg_paged_attention_shared_prefix_workspace_bytes(b, heads, hkv, d, bs, 0, 0) == 0
    for entry in ("v1", "scores", "shared"):
        out = torch.full_like(q, float("nan"))
        six = [t.data_ptr() for t in (q, cache, cache, table, lens, out)]
        code = dtype_code(q)
        if entry == "v1":
            st = lib.rg_paged_attention_v1(*six, 0.1, *shape, code, 0, ws_ptr, given, stream)
        elif entry == "scores":
            st = lib.rg_paged_attention_v1_scores(*six, scores.data_ptr(), None, 0, 0.1, *shape, code, 0, 0, ws_ptr,
                                                  given, stream)
        else:
            st = lib.rg_paged_attention_shared_prefix(*six, 0.1, *shape, 0, code, 0, ws_ptr, given, stream)
        assert st == _lib.RG_OK, f"{entry}: {_lib.last_error()}"
        torch.cuda.synchronize()
        assert float(out.float().abs().max()) == 0, entry
    assert (scores == 5.0).all()
