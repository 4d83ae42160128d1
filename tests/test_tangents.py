"""Tensors whose derivative would be lost without a word are refused (the GPU's calls: test_gpu_tangents.py)."""
import pytest
import torch
from torch.autograd import forward_ad

from rusttorch_amd._lib import Gpt2Error
from rusttorch_amd.qcache import _no_gradient


def test_refuses_what_has_a_gradient_or_a_tangent():
    x = torch.zeros(3)
    _no_gradient("x", x, "it")
    with pytest.raises(Gpt2Error, match="x requires a gradient, which it has none of"):
        _no_gradient("x", x.clone().requires_grad_(), "it")
    with torch.no_grad():
        _no_gradient("x", x.clone().requires_grad_(), "it")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        _no_gradient("x", x, "it")
        _no_gradient("x", forward_ad.unpack_dual(dual).primal, "it")
        for y in (dual, dual.view(3, 1), 2 * dual):
            with pytest.raises(Gpt2Error, match="x has a forward-mode tangent, which it does not carry on"):
                _no_gradient("x", y, "it")
            with torch.no_grad(), pytest.raises(Gpt2Error, match="tangent"):
                _no_gradient("x", y, "it")
