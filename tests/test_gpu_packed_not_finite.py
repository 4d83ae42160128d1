"""Packed attention: what keys and queries that are not finite do, type by type."""
import numpy as np
import pytest
import torch

from rusttorch_amd.attention import packed_attention
from tests.fourbit_ref import attention
from tests.test_gpu_fourbit import TYPES, ints, near
from tests.test_gpu_packed import prob_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("at", [0, 40, 90])   # within the tile on the diagonal and before it
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_key(dtype, dim, at, bad):
    """f32: the rows that see it are NaN. bf16 and f16: NaN as well where it gives NaN or +infinity; a key whose score
    is -infinity is as if it were not there, but in a row that sees no other, which is NaN."""
    n, scale = 300, dim ** -0.5
    print(f"[gpu] packed, key {at} holds {bad}, {dim}, {dtype}", flush=True)
    g = torch.Generator().manual_seed(dim + at)
    q, k, v = (torch.randn(n, 1, dim, generator=g).to(TYPES[dtype]) for _ in range(3))
    q[200, 0, 3] = 0
    kn = k[:, 0].double().numpy()
    k[at, 0, 3] = bad
    got = packed_attention(q.cuda(), k.cuda(), v.cuda(), ints([0, n]))[:, 0]
    qn, vn = q[:, 0].double().numpy(), v[:, 0].double().numpy()
    score = qn[:, 3] * bad if dtype != "f32" else np.full(n, np.nan)
    without = (score == -np.inf) & (np.arange(n) >= at)
    least = 2.0 ** -31 if dtype == "f16" else 2.0 ** -125
    want, off, *_ = attention(qn, kn, vn, np.arange(n) + 1, scale, prob_step(dtype), least)
    others = np.arange(n) != at
    w2, o2, *_ = attention(qn, kn[others], vn[others], np.arange(n) + (np.arange(n) < at), scale, prob_step(dtype), least)
    want[without], off[without] = w2[without], o2[without]
    sees = np.arange(n) >= at
    nan = sees & ~without | (sees & (np.arange(n) == 0))
    want[nan], off[nan] = np.nan, 0
    assert torch.isnan(got[torch.from_numpy(nan).cuda()]).all()
    near(got, want, off, dtype)
    assert dtype == "f32" or bad != bad or without.sum() > 50


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_query(dtype, bad):
    q, k, v = (torch.randn(300, 1, 64, generator=torch.Generator().manual_seed(i)).to(TYPES[dtype]).cuda() for i in range(3))
    want = packed_attention(q, k, v, ints([0, 300]))
    rows = torch.tensor([0, 1, 63, 64, 130, 299], device="cuda")
    q[rows, 0, 17] = bad
    got = packed_attention(q, k, v, ints([0, 300]))
    others = torch.ones(300, dtype=torch.bool, device="cuda")
    others[rows] = False
    assert torch.isnan(got[rows]).all() and torch.equal(got[others], want[others])
