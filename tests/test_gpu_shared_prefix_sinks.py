"""The shared-prefix decode where one token takes nearly all of the weight and tens of thousands share the rest."""
from __future__ import annotations

import math

import pytest
import torch

from attention64 import assert_within, attention64
from helpers import dev_f32
from test_gpu_shared_prefix import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("gap", [17.0, 25.5, 28.0])
@pytest.mark.parametrize("at", [0, 7000])
def test_many_small_weights_beside_a_large_one(device, kernels, dtype, gap, at):
    """Weights of 2^-gap of the largest each, whose value is 0, so the output is theirs alone.  Rows enough that
    the prefix is in two parts, and the large weight stands before half of the others.

    In fp16 they are held times 2^7 or more, and below 2^-14 rounded by half a step of 2^-25 at most: 2^-32 of
    the largest weight a token, times its value, beside the bounds of the other types."""
    shared, rows = 1024, 1025
    b = Batch(device, [shared * 16 + 1] * rows, shared, dtype, 32, 32, 64, seed=3)
    g = torch.Generator(device=device).manual_seed(1)
    k = 0.05 * torch.randn(b.kc.shape, generator=g, device=device)
    v = 1 + 0.1 * torch.randn(b.kc.shape, generator=g, device=device)
    where = int(b.table[0, at // 16]), slice(None), at % 16
    k[where + (0,)] = gap * math.log(2)
    v[where] = 0
    b.kc.copy_(k)
    b.vc.copy_(v)
    b.q.zero_()
    b.q[..., 0] = 8.0                                # times 1/8: a score is the key's first element
    some = [0, 500, 1024]
    want, tol, _, _ = attention64(b.q[some], b.kc, b.vc, b.table[some], b.ctx[some], b.scale, dtype, rounded_p=True)
    if dtype == "f16":
        tol = tol + shared * 16 * 2.0 ** -32 * float(v.abs().max())
    assert want.min() > 0.5 * shared * 16 * 2.0 ** -gap
    assert_within(dev_f32(b.run(kernels))[some], want, tol)
