"""Packed attention of rows that lie in ways of their own, in each of the kernel's forms: two groups of waves (one long
sequence) and one, whole heads and padded ones, aligned rows and others."""
import numpy as np
import pytest
import torch

from rusttorch_amd.attention import packed_attention
from tests.test_gpu_fourbit import TYPES, ints, near, rows
from tests.test_gpu_packed import check, want_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [80, 33, 24, 120, 7])
@pytest.mark.parametrize("rows_of,heads,kv", [(600, 4, 2), (1100, 3, 3)])
def test_one_sequence_of_padded_heads(rows_of, heads, kv, dim, dtype):
    check([rows_of], heads, kv, dim, dtype, before=3, behind=5, seed=dim)
    check([rows_of, rows_of + 77], heads, kv, dim, dtype, seed=dim + 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 48])
@pytest.mark.parametrize("lengths", [[700], [1030, 900], [150, 3, 90, 60]])
def test_rows_that_are_not_aligned(dim, dtype, lengths):
    """An odd stride between rows, a start that is not a multiple of 16 bytes, results the same way."""
    print(f"[gpu] packed {lengths}, 2 heads over 1 of {dim}, {dtype}, odd strides", flush=True)
    rng, offsets = np.random.default_rng(dim), np.cumsum([0, *lengths])
    n = int(offsets[-1])
    x, xn = rows(rng, (n, 4, dim + 3), dtype)
    q, k, v = x[:, :2, 1:dim + 1], x[:, 2:3, 3:], x[:, 3:4, :dim]
    out = torch.full((n, 2, dim + 1), 7.0, dtype=TYPES[dtype], device="cuda")
    packed_attention(q, k, v, ints(offsets), out=out[..., :dim])
    want, off = want_of(xn[:, :2, 1:dim + 1], xn[:, 2:3, 3:], xn[:, 3:4, :dim], offsets, dim ** -0.5, dtype)
    near(out[..., :dim], want, off, dtype)
    assert (out[..., dim:] == 7).all()


@pytest.mark.parametrize("dim", [64, 128, 72])
@pytest.mark.parametrize("lengths", [[700], [150, 3, 90, 60]])
def test_f32_rows_aligned_to_16_bytes_only(dim, lengths):
    print(f"[gpu] packed {lengths}, 2 heads over 1 of {dim}, f32, 16 bytes behind a multiple of 32", flush=True)
    rng, offsets = np.random.default_rng(dim), np.cumsum([0, *lengths])
    x, xn = rows(rng, (int(offsets[-1]), 4, dim + 4))
    x, xn = x[..., 4:], xn[..., 4:]
    assert x.data_ptr() % 32 == 16 and x.stride(1) % 8 == 4
    got = packed_attention(x[:, :2], x[:, 2:3], x[:, 3:4], ints(offsets))
    want, off = want_of(xn[:, :2], xn[:, 2:3], xn[:, 3:4], offsets, dim ** -0.5, "f32")
    near(got, want, off, "f32")
    assert torch.equal(got, packed_attention(*(y.contiguous() for y in (x[:, :2], x[:, 2:3], x[:, 3:4])), ints(offsets)))
