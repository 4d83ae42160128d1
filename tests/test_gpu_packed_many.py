"""Packed attention of thousands of sequences: a workgroup finds its own among the offsets."""
import numpy as np
import pytest
import torch

from rusttorch_amd.attention import packed_attention
from tests.test_gpu_fourbit import TYPES, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,dtype,heads,kv", [(200, "f32", 2, 2), (256, "f32", 3, 1), (257, "bf16", 4, 2), (1023, "f16", 2, 1),
                                              (1024, "bf16", 2, 2), (1300, "f32", 5, 1), (2560, "bf16", 2, 1), (5003, "f32", 2, 1)])
def test_as_the_same_sequences_in_several_calls(n, dtype, heads, kv):
    """Lengths 0 to 30 with a long one here and there, offsets that descend: each as in a call of up to 60 sequences."""
    print(f"[gpu] {n} packed sequences, {heads} heads over {kv}, {dtype}", flush=True)
    rng = np.random.default_rng(n)
    lengths = rng.integers(0, 31, n) * (rng.random(n) < 0.7)
    lengths[rng.integers(0, n, 5)] = rng.integers(100, 600, 5)
    meant = np.cumsum(np.r_[7, lengths])
    rows = int(meant[-1]) + 9
    given = meant.copy()
    for i in rng.integers(1, n, n // 9):    # (an offset within a run of the same may be any smaller one)
        if meant[i] == meant[i - 1]:
            given[i] = rng.integers(-5, meant[i] + 1)
    q, k, v = (torch.randn(rows, h, 64, device="cuda").to(TYPES[dtype]) for h in (heads, kv, kv))
    got = packed_attention(q, k, v, ints(given))
    assert (got[:7] == 0).all() and (got[meant[-1]:] == 0).all()
    for i in range(0, n, 60):
        part = meant[i:i + 61]
        a, b = int(part[0]), int(part[-1])
        want = packed_attention(q[a:b], k[a:b], v[a:b], ints(part - a))
        assert torch.equal(got[a:b], want), i   # (the same kernel: no call is of one long sequence)


def test_time_grows_with_the_sequences():
    """Ten times as many short sequences take about ten times as long, not fifty."""
    def best(n):
        x = torch.randn(20 * n, 12, 64, device="cuda")
        o = torch.arange(0, 20 * n + 1, 20, dtype=torch.int32, device="cuda")
        took = []
        for _ in range(6):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            packed_attention(x, x, x, o)
            end.record()
            end.synchronize()
            took.append(start.elapsed_time(end))
        return min(took)

    few, many = best(1000), best(10000)
    assert many < 30 * few, (few, many)
