"""Host side of the 4-bit key/value cache and of packed attention that needs no
GPU: refusals before any device work, and the definition that the GPU tests
compare with."""
import ctypes as C

import numpy as np
import pytest
import torch

from rusttorch_amd import _lib
from rusttorch_amd._lib import Gpt2Error, check
from rusttorch_amd.attention import packed_attention
from rusttorch_amd.q4cache import FourBitCache
from tests.fourbit_ref import Cache, attention, held


@pytest.mark.parametrize("args,what", [
    ((1, 1, 0, 10), "head_dim 0 is not supported"), ((1, 1, 129, 10), "head_dim 129 is not supported"),
    ((0, 1, 64, 10), "must be >= 1"), ((1, 0, 64, 10), "must be >= 1"), ((1, 1, 64, 0), "must be >= 1"),
    ((1, 1, 64, 4000001), "capacity 4000001 exceeds"), ((2 ** 33, 1, 64, 10), "n_seq \\* n_head exceeds"),
    ((1001, 1000, 64, 10), "n_seq \\* n_head exceeds"),
])
def test_new_refuses(args, what):
    h = C.c_void_p()
    with pytest.raises(Gpt2Error, match=what):
        check(_lib.load().rtg_fourbit_new(*args, C.byref(h)))
    assert not h.value


def test_null_arguments():
    lib, r, out, f = _lib.load(), bytes(32), C.c_uint32(), C.c_void_p(256)
    for res in (lib.rtg_fourbit_new(1, 1, 64, 10, None), lib.rtg_fourbit_append(None, 0, r, r, 1, None, None, None),
                lib.rtg_fourbit_read(None, 0, r, r, 1, None, None), lib.rtg_fourbit_attend(None, 0, r, 1, 1, None, 1.0, r, None, 0.0, None),
                lib.rtg_fourbit_weights(None, f, 1, None),
                lib.rtg_fourbit_add_weights(None, f, 1, None), lib.rtg_fourbit_evict(None, 1, 0, f, None),
                lib.rtg_fourbit_lengths(None, C.byref(out), None),
                lib.rtg_attend_packed(0, r, r, r, 1, 1, 1, 64, None, 1, 1.0, r, None),
                lib.rtg_attend_packed(0, r, r, r, 1, 1, 1, 64, f, 1, 1.0, r, None)):
        with pytest.raises(Gpt2Error, match="null argument"):
            check(res)
    lib.rtg_fourbit_destroy(None)


@pytest.mark.parametrize("n_rows,q_heads,heads,dim,n_seq,scale,dtype,what", [
    (1, 1, 1, 0, 1, 1.0, 0, "head_dim 0 is not supported"), (1, 1, 1, 129, 1, 1.0, 0, "head_dim 129 is not supported"),
    (1, 3, 2, 64, 1, 1.0, 0, "3 query heads are not a multiple of 2 heads"), (1, 0, 1, 64, 1, 1.0, 0, "multiple"),
    (1, 1, 0, 64, 1, 1.0, 0, "multiple"), (1, 1025, 1, 64, 1, 1.0, 0, "exceed 1024"),
    (1, 1, 1, 64, 0, 1.0, 0, "n_seq must be within"), (1, 1, 1, 64, 10 ** 6 + 1, 1.0, 0, "n_seq must be within"),
    (10 ** 8 + 1, 1, 1, 64, 1, 1.0, 0, "exceed"), (10 ** 8, 32, 32, 64, 1, 1.0, 0, "exceed"),
    (1, 10 ** 6, 10 ** 6, 64, 10 ** 6, 1.0, 0, "too many"), (4 * 10 ** 7, 32, 32, 64, 1, 1.0, 0, "too many"), (1, 1, 1, 64, 1, float("inf"), 0, "scale must be finite"),
    (1, 1, 1, 64, 1, float("nan"), 0, "scale must be finite"), (1, 1, 1, 64, 1, 1.0, 3, "takes f32, bf16 or f16"),
])
def test_packed_refuses(n_rows, q_heads, heads, dim, n_seq, scale, dtype, what):
    r, f = bytes(32), C.c_void_p(256)
    with pytest.raises(Gpt2Error, match=what):
        check(_lib.load().rtg_attend_packed(dtype, r, r, r, n_rows, q_heads, heads, dim, f, n_seq, scale, r, None))


def test_no_rows_is_no_work():
    r, f = bytes(32), C.c_void_p(256)
    check(_lib.load().rtg_attend_packed(0, r, r, r, 0, 1, 1, 64, f, 1, 1.0, r, None))


@pytest.mark.parametrize("args,what", [((-1, 1, 64, 10), "n_seq must not be negative"),
                                       ((1, 1, 64, 2 ** 64 + 10), "capacity is too large")])
def test_sizes_that_the_library_could_not_tell_apart(args, what):
    with pytest.raises(Gpt2Error, match=what):
        FourBitCache(*args)


def test_packed_attention_refuses_host_tensors():
    x, o = torch.zeros(4, 2, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(Gpt2Error, match="needs tensors on a GPU"):
        packed_attention(x, x, x, o)
    with pytest.raises(Gpt2Error, match="must be \\[rows"):
        packed_attention(x[0], x, x, o)
    with pytest.raises(Gpt2Error, match="must be f32, bf16 or f16"):
        packed_attention(x.double(), x, x, o)


def test_definition():
    """Every number a group can hold reads back as itself, ties go to the even code, all are within a
    fifth of the largest (which lies in 3.5 .. 7 of its scale: the widest step, 4 to 6, is off by 1 at 5)."""
    x = np.zeros((1, 32))
    x[0, :8] = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    x[0, 8:15] = [-0.25, 0.75, -1.25, 1.75, 2.5, 3.5, 5]
    want = x.copy()
    want[0, 8:15] = [0, 1, -1, 2, 2, 4, 4]
    for e in (-99, 0, 60):
        assert np.array_equal(held(x * 2.0 ** e), want * 2.0 ** e)
    x[0, 0] = 7.0  # (a tie between 6 and 8: the scale stays)
    assert held(x)[0, 0] == 6
    x[0, 0] = 7.001
    assert held(x)[0, 0] == 8
    rng = np.random.default_rng(0)
    y = rng.standard_normal((50, 80))
    h = held(y)
    for c in (0, 32, 64):
        top = np.abs(y[:, c:c + 32]).max(-1)
        assert (np.abs(h - y)[:, c:c + 32].max(-1) <= top / 5 + 1e-12).all()
    y[3, 40] = np.inf
    assert np.isnan(held(y)[3, 32:64]).all() and np.isfinite(held(y)[3, :32]).all()
    tiny = np.full((1, 4), 2.0 ** -104)
    assert (held(tiny) == 0).all()
    assert held(np.full((1, 4), 3.4e38))[0, 0] == 6 * 2.0 ** 125


def test_reference_cache():
    rng = np.random.default_rng(1)
    c = Cache(2, 1, 32, 20)
    x = rng.standard_normal((2, 12, 1, 32))
    assert c.append(x, x, counts=[12, 5]) == [] and c.append(x, x) == [0]
    assert c.length(0) == 12 and c.length(1) == 17
    q = rng.standard_normal((2, 3, 2, 32))
    out, off = c.attend(q, counts=[3, 2], weigh=1.0)
    assert np.allclose([w[0].sum() for w in c.w], [6, 4]) and (out[1, 2] == 0).all()
    p = np.exp(c.k[0][0] @ q[0, 2, 0] / 32 ** 0.5)
    assert np.allclose(out[0, 2, 0], p @ c.v[0][0] / p.sum()) and (off[0] < 1e-4).all()
    w, k = c.w[0][0].copy(), c.k[0][0].copy()
    kept = c.evict(6, 2)
    assert list(kept[0, 0, -2:]) == [10, 11] and set(kept[0, 0, :4]) == set(np.argsort(-w[:10], kind="stable")[:4])
    assert np.array_equal(c.k[0][0], k[kept[0, 0]])
    out, _, p, _ = attention(np.ones((1, 4)), np.ones((3, 4)), np.arange(12.).reshape(3, 4), [2], 1.0)
    assert np.allclose(out[0], [2, 3, 4, 5]) and np.allclose(p[0], [0.5, 0.5, 0])
