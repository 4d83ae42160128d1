"""Attention over packed prompts on device tensors: torch's side of
rtg_attend_packed (include/rtgpu.h). There is no counterpart in the reference,
whose prompts are one sequence at a time."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import Gpt2Error, check
from .qcache import _TYPES, _no_gradient, _one_runtime, _pack_rows, _raw_stream

__all__ = ["packed_attention"]

# the current device as an integer: 0.1 us, where current_device() takes 1
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_call = None  # rtg_attend_packed, once the library is loaded


def _load():
    global _call
    lib = _lib.load()
    if torch.cuda.is_available():
        _one_runtime()
    _call = lib.rtg_attend_packed
    return _call


def _rows(what: str, x: torch.Tensor, shape, dtype, index: int) -> bytes:
    """x as an rtg_rows, once it is known to be [rows, heads, head_dim] of dtype on GPU `index`."""
    if x.shape != shape:
        raise Gpt2Error(f"{what} must be {list(shape)}, not {list(x.shape)}")
    if x.dtype is not dtype:
        raise Gpt2Error(f"{what} must be {dtype}, not {x.dtype}")
    if x.get_device() != index:
        raise Gpt2Error(f"{what} is on {x.device}, q on GPU {index}")
    _no_gradient(what, x, "packed_attention")
    row, head, col = x.stride()
    if col != 1 and shape[2] > 1 and x.numel():
        raise Gpt2Error(f"{what}'s last dimension must be contiguous")
    return _pack_rows(x.data_ptr(), 0, row, head)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, scale=None,
                     out=None) -> torch.Tensor:
    """Causal attention of sequences packed one behind the other, each over itself.

    q [rows, query heads, head_dim], k and v [rows, heads, head_dim] (query head h reads head h / (query heads /
    heads)), f32, bf16 or f16 on one GPU, in any strides whose last is 1; offsets: n + 1 int32 on that GPU, sequence s
    has rows offsets[s] .. offsets[s + 1] - 1. scale: 1 / sqrt(head_dim). Returns [rows, query heads, head_dim] (out,
    where it is given, which must not overlap the others); rows of no sequence are 0.

    Goes to the current stream of the tensors' device and does not wait for it; has no gradient."""
    shape, dtype, index = q.shape, q.dtype, q.get_device()
    if len(shape) != 3:
        raise Gpt2Error(f"q must be [rows, heads, head_dim], not {list(shape)}")
    if dtype not in _TYPES:
        raise Gpt2Error(f"q must be f32, bf16 or f16, not {dtype}")
    if index < 0:
        raise Gpt2Error(f"packed_attention needs tensors on a GPU, not on {q.device}")
    rows, heads, dim = shape
    kv = k.shape
    if len(kv) != 3 or kv[0] != rows or kv[2] != dim:
        raise Gpt2Error(f"k must be [{rows}, heads, {dim}], not {list(kv)}")
    to_q, to_k, to_v = _rows("q", q, shape, dtype, index), _rows("k", k, kv, dtype, index), _rows("v", v, kv, dtype, index)
    n = offsets.numel() - 1
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or n < 1 or not offsets.is_contiguous():
        raise Gpt2Error("offsets must be n + 1 contiguous int32, n >= 1")
    if offsets.get_device() != index:
        raise Gpt2Error(f"offsets is on {offsets.device}, q on GPU {index}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        to = _pack_rows(out.data_ptr(), 0, heads * dim, dim)
    else:
        to = _rows("out", out, shape, dtype, index)
    call = _call or _load()
    args = (_TYPES[dtype], to_q, to_k, to_v, rows, heads, kv[1], dim, offsets.data_ptr(), n,
            (dim or 1) ** -0.5 if scale is None else scale, to, _raw_stream(index))
    if index == _device():
        check(call(*args))
    else:
        with torch.cuda.device(index):
            check(call(*args))
    return out
