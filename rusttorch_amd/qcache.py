"""An 8-bit key/value cache over device tensors: torch's side of rtg_qcache_*
(include/rtgpu.h has what the cache holds and what each call does).

Programs that run their own layers write keys and values with `append`, run
attention over them with `attend` and get them back with `read`; the calls go
to the current stream of the cache's device and do not wait for it. Tensors are
[n_seq, tokens, heads, head_dim] on that device, f32, bf16 or f16, in any strides
whose last is 1. Nothing here has a gradient. There is no counterpart in the
reference.

One cache takes one call at a time, reading ones included: they share a
workspace. Calls on two streams, replays of two graphs, or a replay beside a call
need the streams' own ordering (`wait_stream`, events); different caches do not.
A cache has to live as long as the graphs that hold its calls.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import Gpt2Error, check

__all__ = ["QuantisedCache"]

_pack_rows = struct.Struct("Pnnn").pack  # an rtg_rows
# the current stream of a device as an integer: 0.1 us, where the object that current_stream() makes costs 1 to 2
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)

_TYPES = {torch.float32: _lib.RTG_F32, torch.bfloat16: _lib.RTG_BF16, torch.float16: _lib.RTG_F16}


def _one_runtime() -> None:
    """torch and the library must have loaded the same HIP runtime: streams and
    memory of one mean nothing to another. They do when torch comes first."""
    with open("/proc/self/maps") as f:
        paths = {line.split(None, 5)[5].strip() for line in f if "libamdhip64" in line}
    if len(paths) > 1:
        raise Gpt2Error("two HIP runtimes are loaded (" + ", ".join(sorted(paths)) +
                        "): import torch before the library is first used")


def _no_gradient(what: str, x: torch.Tensor, whose: str) -> None:
    """Refuses an x whose gradient, backward or forward, would be lost."""
    if x.requires_grad and torch.is_grad_enabled():
        raise Gpt2Error(f"{what} requires a gradient, which {whose} has none of: detach it or use torch.no_grad()")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise Gpt2Error(f"{what} has a forward-mode tangent, which {whose} does not carry on: take its primal")


class QuantisedCache:
    """Keys and values of `n_seq` sequences and `n_head` heads, up to `capacity`
    tokens each, in 8 bits with a scale per `block` (16, 32 or 64) tokens and head."""

    def __init__(self, n_seq: int, n_head: int, head_dim: int, capacity: int, block: int = 32, device=None):
        self._h = None
        for name, x in (("n_seq", n_seq), ("n_head", n_head), ("head_dim", head_dim), ("capacity", capacity),
                        ("block", block)):
            if x < 0:
                raise Gpt2Error(f"{name} must not be negative")
            if x >= 1 << 63:
                raise Gpt2Error(f"{name} is too large")
        self._lib = _lib.load()
        self._index = -1  # of the device
        h = C.c_void_p()
        if torch.cuda.is_available():
            _one_runtime()
            self.device = torch.device("cuda" if device is None else device)
            if self.device.type != "cuda":
                raise Gpt2Error("the cache's device must be a GPU")
            if self.device.index is None:
                self.device = torch.device("cuda", torch.cuda.current_device())
            self._index = self.device.index
            with torch.cuda.device(self.device):
                check(self._lib.rtg_qcache_new(n_seq, n_head, head_dim, capacity, block, C.byref(h)))
        else:
            check(self._lib.rtg_qcache_new(n_seq, n_head, head_dim, capacity, block, C.byref(h)))
        self._h = h
        self.n_seq, self.n_head, self.head_dim, self.capacity, self.block = n_seq, n_head, head_dim, capacity, block

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.rtg_qcache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- arguments --

    def _stream(self):
        if self._h is None:
            raise Gpt2Error("the cache is closed")
        return _raw_stream(self._index)

    def _rows(self, what: str, x: torch.Tensor, dtype, tokens: int, heads: int) -> bytes:
        """x as an rtg_rows, once it is known to be [n_seq, tokens, heads, head_dim] of dtype on the cache's device."""
        shape = (self.n_seq, tokens, heads, self.head_dim)
        if x.shape != shape:
            raise Gpt2Error(f"{what} must be {list(shape)}, not {list(x.shape)}")
        if x.dtype is not dtype:
            raise Gpt2Error(f"{what} must be {dtype}, not {x.dtype}")
        if x.get_device() != self._index:
            raise Gpt2Error(f"{what} is on {x.device}, the cache on {self.device}")
        _no_gradient(what, x, "the cache")
        seq, tok, head, col = x.stride()
        if col != 1 and self.head_dim > 1 and x.numel():
            raise Gpt2Error(f"{what}'s last dimension must be contiguous")
        return _pack_rows(x.data_ptr(), seq, tok, head)

    def _type(self, what: str, x: torch.Tensor) -> int:
        if x.dim() != 4:
            raise Gpt2Error(f"{what} must be [n_seq, tokens, heads, head_dim], not {list(x.shape)}")
        if x.dtype not in _TYPES:
            raise Gpt2Error(f"{what} must be f32, bf16 or f16, not {x.dtype}")
        return _TYPES[x.dtype]

    def _ints(self, what: str, x):
        if x is None:
            return None
        if x.dtype is not torch.int32 or x.shape != (self.n_seq,) or not x.is_contiguous():
            raise Gpt2Error(f"{what} must be {self.n_seq} contiguous int32")
        if x.get_device() != self._index:
            raise Gpt2Error(f"{what} is on {x.device}, the cache on {self.device}")
        return x.data_ptr()

    # -- calls --

    def append(self, k: torch.Tensor, v: torch.Tensor, counts=None, start=None) -> None:
        """Writes k, v [n_seq, tokens, n_head, head_dim] behind the sequences, or from token start[s] on (what lay
        there and behind is dropped); of sequence s the first counts[s] tokens (clamped to 0 .. tokens)."""
        stream, dtype, n = self._stream(), self._type("k", k), k.shape[1]
        check(self._lib.rtg_qcache_append(self._h, dtype, self._rows("k", k, k.dtype, n, self.n_head),
                                          self._rows("v", v, k.dtype, n, self.n_head), n,
                                          self._ints("counts", counts), self._ints("start", start), stream))

    def attend(self, q: torch.Tensor, counts=None, scale=None, out=None) -> torch.Tensor:
        """Attention of the last counts[s] tokens of each sequence, q [n_seq, tokens, query heads, head_dim], over
        the keys up to their own position; scale: 1 / sqrt(head_dim). Padding rows are 0."""
        stream, dtype = self._stream(), self._type("q", q)
        n, heads = q.shape[1], q.shape[2]
        rows = self._rows("q", q, q.dtype, n, heads)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            tok = heads * self.head_dim
            to = _pack_rows(out.data_ptr(), n * tok, tok, self.head_dim)
        else:
            to = self._rows("out", out, q.dtype, n, heads)
        check(self._lib.rtg_qcache_attend(self._h, dtype, rows, n, heads, self._ints("counts", counts),
                                          self.head_dim ** -0.5 if scale is None else scale, to, stream))
        return out

    def read(self, n: int, first=None, dtype: torch.dtype = torch.float32, k=None, v=None):
        """(k, v) [n_seq, n, n_head, head_dim]: the values of tokens first[s] (0) .. + n, 0 where there is none."""
        stream = self._stream()
        if n < 0:
            raise Gpt2Error("n must not be negative")
        if dtype not in _TYPES:
            raise Gpt2Error(f"dtype must be f32, bf16 or f16, not {dtype}")
        first = self._ints("first", first)
        if k is None and v is None:
            head, tok = self.head_dim, self.n_head * self.head_dim
            k = torch.empty((self.n_seq, n, self.n_head, head), dtype=dtype, device=self.device)
            v = torch.empty_like(k)
            to_k, to_v = (_pack_rows(x.data_ptr(), n * tok, tok, head) for x in (k, v))
        else:
            k = torch.empty_like(v) if k is None else k  # (checked below, as the other's are)
            v = torch.empty_like(k) if v is None else v
            to_k, to_v = self._rows("k", k, dtype, n, self.n_head), self._rows("v", v, dtype, n, self.n_head)
        check(self._lib.rtg_qcache_read(self._h, _TYPES[dtype], to_k, to_v, n, first, stream))
        return k, v

    def lengths(self) -> list:
        """Tokens of each sequence (waits for the current stream). Raises once where an append since the last call
        left a sequence as it was because its tokens did not fit."""
        out = (C.c_uint32 * self.n_seq)()
        check(self._lib.rtg_qcache_lengths(self._h, out, self._stream()))
        return list(out)
