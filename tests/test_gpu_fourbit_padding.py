"""Calls over the 4-bit cache where most query rows are padding: few queries of a sequence beside many of another."""
import pytest
import torch

from rusttorch_amd.q4cache import FourBitCache
from tests.test_gpu_fourbit import Both, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16"), (128, "f16"), (80, "f32")])
def test_split_keys_with_blocks_of_padding(dim, dtype):
    """Sequences of 5000, 900 and 1 tokens, keys split: none, some and all of a sequence's blocks are padding."""
    b = Both(3, 2, dim, 5100, dtype, seed=dim)
    b.append(5000, counts=[5000, 900, 1])
    for counts in ([16, 16, 16], [1, 16, 3], [16, 0, 0], [0, 9, 1], [0, 0, 16], [0, 0, 0], [-3, 2, 100]):
        b.attend(16, 4, counts=counts, weigh=0.5)
    b.append(70)
    b.attend(32, 2, counts=[17, 1, 32])
    b.attend(6, 10, counts=[1, 6, 0])


def test_many_sequences_with_blocks_of_padding():
    """More sequences than a wave has lanes, keys split."""
    b = Both(100, 1, 64, 1100, seed=3)
    lengths = [1100 if s % 7 == 0 else s % 50 for s in range(100)]
    b.append(1100, counts=lengths)
    b.attend(1, 1, counts=[s % 2 for s in range(100)])
    b.attend(1, 1, counts=[int(s == 63) for s in range(100)], weigh=1.0)


def test_padding_reads_no_keys():
    """One query of each sequence in room for 32 takes about what it takes alone: a block of 16 padding rows is not
    worked on (the keys and values are 590 MB, read once in one case and twice in the other if it were)."""
    S, H, D, n = 128, 8, 64, 8000
    c = FourBitCache(S, H, D, n)
    k = torch.randn(1, n, H, D, device="cuda").expand(S, n, H, D)
    c.append(k, k)
    q = torch.randn(S, 32, H, D, device="cuda")
    one = ints([1] * S)

    def best(call):
        took = []
        for i in range(12):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(5):
                call()
            end.record()
            end.synchronize()
            took.append(start.elapsed_time(end))
        return min(took)

    alone, padded = best(lambda: c.attend(q[:, :1])), best(lambda: c.attend(q, counts=one))
    assert padded < 1.5 * alone, (padded, alone)
    assert torch.equal(c.attend(q, counts=one)[:, :1], c.attend(q[:, :1]))
