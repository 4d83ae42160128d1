"""What a 4-bit cache takes of the device's memory: less than half of bf16 rows, also where it is small."""
import gc

import pytest
import torch

from rusttorch_amd.q4cache import FourBitCache
from tests.test_gpu_fourbit import Both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_seq,heads,dim,capacity", [(1, 12, 64, 1024), (1, 12, 64, 4096), (2, 8, 128, 2048), (16, 8, 128, 8192)])
def test_memory(n_seq, heads, dim, capacity):
    gc.collect()
    FourBitCache(1, 1, 64, 10)  # (the library's own, and the runtime's)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    caches = [FourBitCache(n_seq, heads, dim, capacity) for _ in range(24)]
    took = (before - torch.cuda.mem_get_info()[0]) / len(caches)
    rows = n_seq * heads * dim * capacity * 2 * 2  # keys and values in bf16
    # (pages of 2 MB, and 64 KB of tickets)
    assert len(caches) == 24 and took < rows / 2 + 2 ** 21 + 2 ** 16, (took / 1e6, rows / 1e6)


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16"), (80, "f16")])
@pytest.mark.parametrize("capacity", [1030, 2500])
def test_small_caches_split_their_keys(dim, dtype, capacity):
    """Room for the partial results of a few workgroups only."""
    b = Both(1, 1, dim, capacity, dtype, seed=capacity)
    b.append(capacity - 5)
    for n, heads in ((1, 1), (1, 5), (8, 2), (5, 8), (120, 1), (130, 2), (200, 3)):
        b.attend(n, heads, weigh=0.5)
    b.append(5)
    b.attend(1, 16)
