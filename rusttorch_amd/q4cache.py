"""A 4-bit key/value cache over device tensors: torch's side of rtg_fourbit_*
(include/rtgpu.h has what the cache holds and what each call does).

The calls of `QuantisedCache` (qcache.py), for half its memory: `append`,
`attend`, `read`, `lengths`; and what a program needs to keep a cache within a
budget: `attend(..., weigh=decay)` sums the attention that each token gets,
`evict` keeps the tokens that have got most. There is no counterpart in the
reference.

Tensors are [n_seq, tokens, heads, head_dim] on the cache's device, f32, bf16 or
f16, in any strides whose last is 1. Calls go to the current stream of that device
and do not wait for it; nothing here has a gradient. One cache takes one call at a
time, reading ones included: they share a workspace. Calls on two streams, replays
of two graphs, or a replay beside a call need the streams' own ordering. A cache has
to live as long as the graphs that hold its calls.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import Gpt2Error, check
from .qcache import _TYPES, QuantisedCache, _no_gradient, _one_runtime, _pack_rows

__all__ = ["FourBitCache"]


class FourBitCache(QuantisedCache):
    """Keys and values of `n_seq` sequences and `n_head` heads, up to `capacity` tokens each, in 4 bits with a power
    of two for every 32 channels of a token."""

    def __init__(self, n_seq: int, n_head: int, head_dim: int, capacity: int, device=None):
        self._h = None
        for name, x in (("n_seq", n_seq), ("n_head", n_head), ("head_dim", head_dim), ("capacity", capacity)):
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
                check(self._lib.rtg_fourbit_new(n_seq, n_head, head_dim, capacity, C.byref(h)))
        else:
            check(self._lib.rtg_fourbit_new(n_seq, n_head, head_dim, capacity, C.byref(h)))
        self._h = h
        self.n_seq, self.n_head, self.head_dim, self.capacity = n_seq, n_head, head_dim, capacity

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.rtg_fourbit_destroy(self._h)
            self._h = None

    def _floats(self, what: str, x: torch.Tensor, shape: tuple):
        if x.dtype is not torch.float32 or tuple(x.shape) != shape or not x.is_contiguous():
            raise Gpt2Error(f"{what} must be contiguous float32 {list(shape)}, not {x.dtype} {list(x.shape)}")
        if x.get_device() != self._index:
            raise Gpt2Error(f"{what} is on {x.device}, the cache on {self.device}")
        _no_gradient(what, x, "the cache")
        return x.data_ptr()

    # -- calls --

    def append(self, k: torch.Tensor, v: torch.Tensor, counts=None, start=None) -> None:
        """Writes k, v [n_seq, tokens, n_head, head_dim] behind the sequences, or from token start[s] on (what lay
        there and behind is dropped); of sequence s the first counts[s] tokens (clamped to 0 .. tokens)."""
        stream, dtype, n = self._stream(), self._type("k", k), k.shape[1]
        check(self._lib.rtg_fourbit_append(self._h, dtype, self._rows("k", k, k.dtype, n, self.n_head),
                                           self._rows("v", v, k.dtype, n, self.n_head), n,
                                           self._ints("counts", counts), self._ints("start", start), stream))

    def attend(self, q: torch.Tensor, counts=None, scale=None, out=None, weigh=None) -> torch.Tensor:
        """Attention of the last counts[s] tokens of each sequence, q [n_seq, tokens, query heads, head_dim], over
        the keys up to their own position; scale: 1 / sqrt(head_dim). Padding rows are 0.

        weigh (0 .. 1): the tokens' weights become so many times what they are (0: they begin anew), plus the
        probabilities that these queries give them."""
        stream, dtype = self._stream(), self._type("q", q)
        n, heads = q.shape[1], q.shape[2]
        rows = self._rows("q", q, q.dtype, n, heads)
        if weigh is not None and not 0 <= weigh <= 1:
            raise Gpt2Error("weigh must be within 0 .. 1")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            tok = heads * self.head_dim
            to = _pack_rows(out.data_ptr(), n * tok, tok, self.head_dim)
        else:
            to = self._rows("out", out, q.dtype, n, heads)
        # (the library works in stats; the allocator keeps it from others until this stream is behind the call)
        stats = None if weigh is None else torch.empty(max(self.n_seq * n * heads * 2, 1), dtype=torch.float32,
                                                       device=self.device)
        check(self._lib.rtg_fourbit_attend(self._h, dtype, rows, n, heads, self._ints("counts", counts),
                                           self.head_dim ** -0.5 if scale is None else scale, to,
                                           None if stats is None else stats.data_ptr(),
                                           0.0 if weigh is None else weigh, stream))
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
        check(self._lib.rtg_fourbit_read(self._h, _TYPES[dtype], to_k, to_v, n, first, stream))
        return k, v

    def weights(self, n: int) -> torch.Tensor:
        """The weights [n_seq, n_head, n] of tokens 0 .. n - 1, 0 where there is none."""
        stream = self._stream()
        if n < 0:
            raise Gpt2Error("n must not be negative")
        out = torch.empty((self.n_seq, self.n_head, n), dtype=torch.float32, device=self.device)
        check(self._lib.rtg_fourbit_weights(self._h, out.data_ptr(), n, stream))
        return out

    def add_weights(self, x: torch.Tensor) -> None:
        """Adds x [n_seq, n_head, n] to the weights of tokens 0 .. n - 1, as far as there are."""
        stream = self._stream()
        n = x.shape[2] if x.dim() == 3 else -1
        check(self._lib.rtg_fourbit_add_weights(self._h, self._floats("x", x, (self.n_seq, self.n_head, n)), n, stream))

    def evict(self, keep: int, recent: int = 0) -> torch.Tensor:
        """Cuts every sequence longer than `keep` to that many tokens: each head keeps the last `recent` and those of
        the largest weights (of equal ones the first), in their order. Returns which tokens these were
        [n_seq, n_head, keep] int32, -1 behind those of a shorter sequence. Positions count what is left."""
        stream = self._stream()
        if keep < 1 or recent < 0 or recent > keep or keep > self.capacity:
            raise Gpt2Error(f"keep {keep} must be within 1 .. {self.capacity} and recent {recent} within 0 .. keep")
        kept = torch.empty((self.n_seq, self.n_head, keep), dtype=torch.int32, device=self.device)
        check(self._lib.rtg_fourbit_evict(self._h, keep, recent, kept.data_ptr(), stream))
        return kept

    def lengths(self) -> list:
        """Tokens of each sequence (waits for the current stream). Raises once where an append since the last call
        left a sequence as it was because its tokens did not fit."""
        out = (C.c_uint32 * self.n_seq)()
        check(self._lib.rtg_fourbit_lengths(self._h, out, self._stream()))
        return list(out)
