"""Host side of the 8-bit key/value cache that needs no GPU: refusals before
any device work, and the definition that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

from rusttorch_amd import _lib
from rusttorch_amd._lib import Gpt2Error, check
from tests.qcache_ref import Cache


@pytest.mark.parametrize("args,what", [
    ((1, 1, 0, 10, 32), "head_dim 0 is not supported"), ((1, 1, 129, 10, 32), "head_dim 129 is not supported"),
    ((1, 1, 64, 10, 48), "block 48 is not supported"), ((1, 1, 64, 10, 0), "block 0 is not supported"),
    ((0, 1, 64, 10, 32), "must be >= 1"), ((1, 0, 64, 10, 32), "must be >= 1"), ((1, 1, 64, 0, 32), "must be >= 1"),
    ((1, 1, 64, 4000001, 32), "capacity 4000001 exceeds"), ((2 ** 33, 1, 64, 10, 32), "n_seq \\* n_head exceeds"),
    ((1001, 1000, 64, 10, 32), "n_seq \\* n_head exceeds"),
])
def test_new_refuses(args, what):
    h = C.c_void_p()
    with pytest.raises(Gpt2Error, match=what):
        check(_lib.load().rtg_qcache_new(*args, C.byref(h)))
    assert not h.value


def test_null_arguments():
    lib, r, out = _lib.load(), bytes(32), C.c_uint32()
    for res in (lib.rtg_qcache_new(1, 1, 64, 10, 32, None), lib.rtg_qcache_append(None, 0, r, r, 1, None, None, None),
                lib.rtg_qcache_read(None, 0, r, r, 1, None, None),
                lib.rtg_qcache_attend(None, 0, r, 1, 1, None, 1.0, r, None), lib.rtg_qcache_lengths(None, C.byref(out), None)):
        with pytest.raises(Gpt2Error, match="null argument"):
            check(res)
    lib.rtg_qcache_destroy(None)


def test_definition():
    """A block's values are within half a step of its largest / 127, codes reach 127, attention of one key is its value."""
    rng = np.random.default_rng(0)
    c = Cache(1, 1, 8, 100, 16)
    x = rng.standard_normal((1, 40, 1, 8)).astype(np.float32)
    assert c.append(x, x) == []
    got = c.read(40)[0][0, :, 0]
    for a in range(0, 40, 16):
        b = x[0, a:a + 16, 0]
        top = np.abs(b).max()
        assert np.abs(got[a:a + 16] - b).max() <= top / 254 * 1.0001
        assert np.isclose(np.abs(got[a:a + 16]).max(), top, rtol=1e-6)
    assert c.append(x, x, start=[41]) == [0] and c.append(x, x, start=[1], counts=[0]) == []
    assert c.length(0) == 1
    assert np.allclose(c.attend(np.ones((1, 1, 1, 8)))[0, 0, 0], c.read(1)[1][0, 0, 0])


@pytest.mark.parametrize("args,what", [((-1, 1, 64, 10), "n_seq must not be negative"),
                                       ((1, 1, 64, 2 ** 64 + 10), "capacity is too large")])
def test_sizes_that_the_library_could_not_tell_apart(args, what):
    from rusttorch_amd.qcache import QuantisedCache

    with pytest.raises(Gpt2Error, match=what):
        QuantisedCache(*args)
