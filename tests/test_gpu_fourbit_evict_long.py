"""Evictions of sequences whose weights do not fit the picking workgroup's LDS (24576 of them), beside some that do."""
import numpy as np
import pytest
import torch

from tests.test_gpu_fourbit import Both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16")])
@pytest.mark.parametrize("keep,recent", [(1, 0), (700, 64), (4000, 0), (24000, 500), (24576, 0), (29000, 64), (29999, 29999), (6000, 5424)])
def test_evicts(dim, dtype, keep, recent):
    """Random weights, many of the same, all of the same, NaN and infinities; 30000, 24640 (within and beyond LDS,
    as `recent` is) and 20000 tokens."""
    S, H = 3, 2
    b = Both(S, H, dim, 30000, dtype, seed=keep)
    b.append(30000, counts=[30000, 24640, 20000])
    w = np.exp(3 * b.rng.standard_normal((S, H, 30000))).astype(np.float32)
    w[0, 0, b.rng.random(30000) < 0.6] = 0
    w[0, 1] = np.round(w[0, 1])
    w[1, 0, 5000:25000:7] = np.nan
    w[1, 0, 3::11] = np.inf
    w[1, 1] = 1.0
    w[2, 1, ::2] = -w[2, 1, ::2]
    b.c.add_weights(torch.from_numpy(w).cuda())
    for s in range(S):
        for h in range(H):
            b.r.w[s][h][:] = w[s, h, :b.r.length(s)]
    got = b.c.evict(keep, recent=recent).cpu().numpy()
    assert np.array_equal(got, b.r.evict(keep, recent))
    b.same(n=keep + 2)
    left = b.c.weights(keep).cpu().numpy()
    for s in range(S):
        for h in range(H):
            assert np.array_equal(left[s, h, :b.r.length(s)], b.r.w[s][h].astype(np.float32), equal_nan=True)
