"""Calls of the 8-bit cache that are refused before any device work, or that have to leave others alone."""
import numpy as np
import pytest

from rusttorch_amd.gpt2 import Gpt2Error
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
