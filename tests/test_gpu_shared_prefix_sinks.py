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
@pytest.mark.parametrize("gap,at", [(14.5, 0), (15.5, 7000), (17.0, 0), (21.3, 0), (21.8, 7000), (22.5, 0), (25.5, 0),
                                    (25.5, 7000), (28.0, 0), (28.0, 7000)])
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


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("power", range(12, 27, 2))
def test_scores_as_large_as_the_steps_between_them(device, kernels, dtype, power):
    """Scores around 2^power in log2 units, where fp32 tells them apart by whole powers of two in the end.  All
    values are 1, so every output is 1 whatever the weights: off by the roundings of the probabilities, which
    the sum takes too, by the fp32 sums of 16,384 terms (2^-23 each) and by its own rounding."""
    shared = 1024
    b = Batch(device, [shared * 16 + 1] * 300, shared, dtype, 32, 32, 64, seed=power)
    g = torch.Generator(device=device).manual_seed(power)
    k = torch.randn(b.kc.shape, generator=g, device=device)
    k[..., 0] = 256.0                                # 2^16 of a raw score; the others' part some hundreds
    b.kc.copy_(k)
    b.vc.fill_(1.0)
    b.q.copy_(32 * torch.randn(b.q.shape, generator=g, device=device))
    b.q[..., 0] = 256.0
    b.scale = 2.0 ** (power - 16) / math.log2(math.e)
    out = dev_f32(b.run(kernels))
    assert_within(out, 1.0, 16384 * 2.0 ** -23 + {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype])
