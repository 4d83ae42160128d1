"""Attention over packed prompts on device tensors: torch's side of
rtg_attend_packed (include/rtgpu.h). There is no counterpart in the reference,
whose prompts are one sequence at a time."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import Gpt2Error, check
from .qcache import _TYPES, _one_runtime, _pack_rows, _raw_stream

__all__ = ["packed_attention"]

_lib_once = None


def _library():
    global _lib_once
    if _lib_once is None:
        lib = _lib.load()
        if torch.cuda.is_available():
            _one_runtime()
        _lib_once = lib
    return _lib_once


def _rows(what: str, x: torch.Tensor, like: torch.Tensor, rows: int, heads, dim: int) -> bytes:
    if x.dim() != 3 or x.shape[0] != rows or x.shape[2] != dim or (heads is not None and x.shape[1] != heads):
        raise Gpt2Error(f"{what} must be [{rows}, {'heads' if heads is None else heads}, {dim}], not {list(x.shape)}")
    if x.dtype is not like.dtype:
        raise Gpt2Error(f"{what} must be {like.dtype}, not {x.dtype}")
    if x.device != like.device:
        raise Gpt2Error(f"{what} is on {x.device}, q on {like.device}")
    if x.requires_grad and torch.is_grad_enabled():
        raise Gpt2Error(f"{what} requires a gradient, which packed_attention has none of: detach it or use torch.no_grad()")
    row, head, col = x.stride()
    if col != 1 and dim > 1 and x.numel():
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
    lib = _library()
    if q.dim() != 3:
        raise Gpt2Error(f"q must be [rows, heads, head_dim], not {list(q.shape)}")
    if q.dtype not in _TYPES:
        raise Gpt2Error(f"q must be f32, bf16 or f16, not {q.dtype}")
    if q.device.type != "cuda":
        raise Gpt2Error(f"packed_attention needs tensors on a GPU, not on {q.device}")
    rows, heads, dim = q.shape
    index = q.get_device()
    to_q, to_k = _rows("q", q, q, rows, heads, dim), _rows("k", k, q, rows, None, dim)
    to_v = _rows("v", v, q, rows, k.shape[1], dim)
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or len(offsets) < 2 or not offsets.is_contiguous():
        raise Gpt2Error("offsets must be n + 1 contiguous int32, n >= 1")
    if offsets.get_device() != index:
        raise Gpt2Error(f"offsets is on {offsets.device}, q on {q.device}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        to = _pack_rows(out.data_ptr(), 0, heads * dim, dim)
    else:
        to = _rows("out", out, q, rows, heads, dim)
    args = (_TYPES[q.dtype], to_q, to_k, to_v, rows, heads, k.shape[1], dim, offsets.data_ptr(), len(offsets) - 1,
            dim ** -0.5 if scale is None else scale, to, _raw_stream(index))
    if index == torch.cuda.current_device():
        check(lib.rtg_attend_packed(*args))
    else:
        with torch.cuda.device(index):
            check(lib.rtg_attend_packed(*args))
    return out
