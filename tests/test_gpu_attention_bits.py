"""How many bits attention's probabilities have, where results show it: keys in pairs of nearly the same score whose
values cancel, so that results are small, their own rounding with them, and a rounding of the probabilities is not."""
import numpy as np
import pytest
import torch

from rusttorch_amd.attention import packed_attention
from rusttorch_amd.q4cache import FourBitCache
from tests.fourbit_ref import attention, held
from tests.test_gpu_fourbit import TYPES, ints, near

pytestmark = pytest.mark.gpu

# A probability as two parts: 8 bits cut and 8 of the rest to nearest, 2^-7 2^-9; two of f16, 2^-11 2^-11.
STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -16, "f16": 2.0 ** -16}
PACKED_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -16, "f16": 2.0 ** -22}


def pairs(n, heads, kv, dim, dtype, seed):
    """Rows q [n, heads, dim], k, v [n, kv, dim] on the GPU, and the same as float64. Scores are within about 1, a
    pair's a few hundredths apart."""
    rng = np.random.default_rng(seed)
    q, k, v = (rng.standard_normal((n, h, dim)) * size for h, size in ((heads, 0.25), (kv, 1.0), (kv, 1.0)))
    k[1::2] = k[0::2] * (1 + 0.3 * rng.random((n // 2, kv, dim)))
    v[1::2] = -v[0::2]
    out = [torch.from_numpy(x).to(TYPES[dtype]) for x in (q, k, v)]
    return [x.cuda() for x in out], [x.double().numpy() for x in out]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("n", [48, 700])
def test_packed(dim, dtype, n):
    print(f"[gpu] packed pairs {n} x 4 over 2 of {dim}, {dtype}", flush=True)
    (q, k, v), (qn, kn, vn) = pairs(n, 4, 2, dim, dtype, n + dim)
    got = packed_attention(q, k, v, ints([0, n]))
    want, off = np.zeros(qn.shape), np.zeros(qn.shape)
    for h in range(4):
        want[:, h], off[:, h], *_ = attention(qn[:, h], kn[:, h // 2], vn[:, h // 2], np.arange(n) + 1, dim ** -0.5,
                                              PACKED_STEP[dtype], 2.0 ** -31 if dtype == "f16" else 2.0 ** -125)
    near(got, want, off, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("capacity", [100, 1300000])
def test_over_the_cache_whatever_its_capacity(dim, dtype, capacity):
    """The kernel is chosen by the capacity: what a result is off by is not."""
    n, heads, tokens = 60, 4, 64
    print(f"[gpu] pairs over a 4-bit cache of {capacity}, {heads} x {dim}, {dtype}", flush=True)
    (q, k, v), (qn, kn, vn) = pairs(tokens, heads, 1, dim, dtype, dim)
    c = FourBitCache(1, 1, dim, capacity)
    c.append(k[None], v[None])
    got = c.attend(q[None, tokens - n:])
    kn, vn = held(kn[:, 0]), held(vn[:, 0])
    want, off = np.zeros((1, n, heads, dim)), np.zeros((1, n, heads, dim))
    for h in range(heads):
        want[0, :, h], off[0, :, h], *_ = attention(qn[tokens - n:, h], kn, vn, tokens - n + np.arange(n) + 1, dim ** -0.5,
                                                    STEP[dtype])
    near(got, want, off, dtype)
