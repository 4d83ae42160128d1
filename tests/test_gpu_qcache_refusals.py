"""Calls of the 8-bit cache that are refused before any device work, or that have to leave a capture alone."""
import gc

import numpy as np
import pytest
import torch

from rusttorch_amd.gpt2 import Gpt2Error
from rusttorch_amd.qcache import QuantisedCache
from tests.test_gpu_qcache_model import TINY, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [2 ** 31, 2 ** 32, 2 ** 63, 400000])
def test_batches_that_sequences_are_not_counted_for(batch):
    m, _ = model(TINY)
    with pytest.raises(Gpt2Error, match=f"batch {batch} is too large for a quantised cache \\(3 heads, 2 layers\\)"):
        m.new_cache(batch, bits=8)
    c = m.new_cache(2, bits=8)
    m.forward_cached_batched(np.zeros((2, 3), int), c)
    assert c.len() == 3


@pytest.mark.parametrize("how", ["close", "collect"])
@pytest.mark.parametrize("what", ["tensors", "model"])
def test_a_cache_that_ends_during_a_capture(what, how):
    gc.collect()
    keep = QuantisedCache(1, 2, 64, 100)
    x = torch.ones(1, 3, 2, 64, device="cuda")
    keep.append(x, x)
    if what == "tensors":
        gone = QuantisedCache(1, 2, 64, 100)
        gone.append(x, x)
        gone.attend(x)
    else:
        m, _ = model(TINY)
        gone = m.new_cache(bits=8)
        for n in (5, 1, 1, 1, 1):   # (the last ones from a graph)
            m.forward_cached([1] * n, gone)
        del m
    if how == "collect":
        gone.me = gone      # (only the collector takes it)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep.append(x, x)
        if how == "close":
            gone.close()
        else:
            del gone
            gc.collect()
        keep.append(x, x)
    for i in range(3):
        g.replay()
        assert keep.lengths() == [9 + 6 * i]
    more = [QuantisedCache(1, 2, 64, 100) for _ in range(3)]
    for c in more:
        c.append(x, x)
        assert c.lengths() == [3]


def test_a_cache_that_is_made_during_a_capture():
    x = torch.ones(1, 3, 2, 64, device="cuda")
    keep = QuantisedCache(1, 2, 64, 100)
    keep.append(x, x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep.append(x, x)
        new = QuantisedCache(1, 2, 64, 100)
        keep.append(x, x)
    for i in range(3):
        g.replay()
        new.append(x, x)
        assert keep.lengths() == [9 + 6 * i] and new.lengths() == [3 + 3 * i]
        assert torch.equal(new.read(3)[0], x)
