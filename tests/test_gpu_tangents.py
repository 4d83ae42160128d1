"""Calls over device tensors refuse forward-mode tangents, which they would drop without a word."""
import pytest
import torch
from torch.autograd import forward_ad

from rusttorch_amd._lib import Gpt2Error
from rusttorch_amd.attention import packed_attention
from rusttorch_amd.q4cache import FourBitCache
from rusttorch_amd.qcache import QuantisedCache
from tests.test_gpu_fourbit import ints

pytestmark = pytest.mark.gpu


def test_refuses_tangents():
    x, offsets = torch.randn(1, 6, 2, 64, device="cuda"), ints([0, 6])
    four, eight = FourBitCache(1, 2, 64, 20), QuantisedCache(1, 2, 64, 20)
    w = torch.zeros(1, 2, 6, device="cuda")
    with forward_ad.dual_level():
        d, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: packed_attention(d[0], x[0], x[0], offsets), lambda: packed_attention(x[0], d[0], x[0], offsets),
                     lambda: packed_attention(x[0], x[0], d[0], offsets), lambda: packed_attention(x[0], x[0], x[0], offsets, out=d[0]),
                     lambda: four.append(d, x), lambda: four.append(x, d), lambda: four.attend(d), lambda: four.attend(x, out=d),
                     lambda: four.add_weights(dw), lambda: eight.append(d, x), lambda: eight.append(x, d), lambda: eight.attend(d)):
            with pytest.raises(Gpt2Error, match="forward-mode tangent"):
                call()
            with torch.no_grad(), pytest.raises(Gpt2Error, match="forward-mode tangent"):
                call()
        want = packed_attention(x[0], x[0], x[0], offsets)
        primal = forward_ad.unpack_dual(d).primal
        assert torch.equal(packed_attention(primal[0], primal[0], primal[0], offsets), want)
    assert four.lengths() == eight.lengths() == [0]
    for transformed in (lambda t: packed_attention(t[0], t[0], t[0], offsets), lambda t: four.attend(t), lambda t: eight.attend(t)):
        with pytest.raises((Gpt2Error, RuntimeError)):
            torch.func.jvp(transformed, (x,), (x,))
