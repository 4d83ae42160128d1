"""The 4-bit cache's attention for many rows against the definition in 64 bits
(fourbit_ref.py). The kernel for it is chosen where columns (pairs of query and head of a
key/value head) fill most of its 128 rows and the capacity allows many keys, so
capacities here are large and sequences short: the keys of a few workgroups are then
split as far as they can be."""
import numpy as np
import pytest
import torch

from tests.test_gpu_fourbit import TYPES, Both, ints, near, prob_step, rows

pytestmark = pytest.mark.gpu


class Many(Both):
    def same(self, n=None, first=None, dtype="f32"):
        longest = max(self.r.length(s) for s in range(self.shape[0]))
        super().same(longest + 3 if n is None else n, first, dtype)

    def weights(self):
        cap, self.r.cap = self.r.cap, max(self.r.length(s) for s in range(self.shape[0]))
        super().weights()
        self.r.cap = cap

    def attend(self, columns, heads, counts=None, **how):
        """columns: of a key/value head, in all; counts: of columns."""
        S, H, _ = self.shape
        group = heads // H
        n = columns // group
        filled = n * group % 128
        assert (filled == 0 or filled > 96) and S * H * self.r.cap >= 1200000, "not the kernel of many rows"
        return super().attend(n, heads, counts=counts and [-(-c // group) for c in counts], **how)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 80, 24])
@pytest.mark.parametrize("heads", [2, 6, 10])
def test_attends(dim, dtype, heads):
    b = Many(3, 2, dim, 200000, dtype, seed=dim + heads)
    b.attend(105, heads)                           # (nothing there)
    b.append(1)
    b.attend(125, heads)
    b.append(40, counts=[40, 0, 13])
    b.attend(128, heads, counts=[41, 128, 0])      # (the second may ask for more than there are)
    b.append(300, counts=[300, 62, 97])
    b.attend(105, heads, scale=-0.3)
    b.attend(250, heads, counts=[250, 63, 7], weigh=1.0)
    b.append(200, counts=[150, 1, 181])
    b.attend(126, heads, scale=0.0)
    b.attend(128, heads, counts=[0, 1, 128], weigh=0.5)
    b.attend(380, heads)


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "f32"), (128, "bf16"), (64, "f16"), (128, "f16"), (20, "bf16")])
def test_more_tiles_than_the_device_takes_at_once(dim, dtype):
    b = Many(5, 27, dim, 9000, dtype, seed=dim)
    b.append(270, counts=[270, 70, 0, 1, 130])
    b.attend(230, 27, counts=[230, 65, 3, 2, 100], weigh=1.0)
    b.attend(256, 27)


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16"), (128, "f16"), (128, "f32")])
def test_long_sequences_are_split(dim, dtype):
    b = Many(2, 1, dim, 600000, dtype, seed=dim)
    b.append(6500, counts=[6500, 4111])
    b.attend(110, 1)
    b.attend(250, 2, counts=[250, 6])
    b.append(64, start=[63, 4111])
    b.attend(256, 4, counts=[0, 240], weigh=1.0)
    b.attend(128, 1, counts=[127, 1], weigh=0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_finite_reaches_those_that_see_it(dim, dtype):
    S, T, H = 3, 150, 2
    b = Many(S, H, dim, 200000, dtype, seed=dim)
    (k, kn), (v, vn) = (rows(b.rng, (S, T, H, dim), dtype) for _ in range(2))
    k[0, 100, 0, 5] = v[0, 60, 1, 40] = v[1, 147, 0, 0] = k[2, 149, 1, 3] = v[2, 120:, :, 7] = float("nan")
    kn[:], vn[:] = k.double().cpu().numpy(), v.double().cpu().numpy()
    b.c.append(k, v)
    b.r.append(kn, vn)
    for n in (128, 500):
        for counts in (None, [n, n - 12, n // 2]):
            b.attend(n, 4 * H, counts=counts)
    b.c.append(k[:, :0], v[:, :0], start=ints([99, 60, 110]))
    b.r.append(kn[:, :0], vn[:, :0], start=[99, 60, 110])
    for n in (236, 360):
        got = b.attend(n, 4 * H)
        assert torch.isfinite(got[1:]).all() and torch.isfinite(got[0, :, :4]).all()
    q = torch.zeros(S, 42, 3 * H, dim, dtype=TYPES[dtype], device="cuda")
    q[1, 0, 3, dim - 1], q[1, 41, 2, 0] = float("inf"), float("nan")
    got = b.c.attend(q)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[1, 0, 3] = bad[1, 41, 2] = True
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[1:][~bad[1:]]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_ranges(dtype):
    for sk, sq, sv, scale in ((1e15, 1e-15, 1e30, 0.1), (1e-18, 1e10, 1e-25, 1e8), (1.0, 1e-30, 1.0, 1e30), (30.0, 1.0, 1.0, 1.0)):
        b = Many(1, 1, 64, 1300000, dtype, seed=4)
        (k, kn), (v, vn) = rows(b.rng, (1, 300, 1, 64), dtype, sk), rows(b.rng, (1, 300, 1, 64), dtype, sv)
        b.put(k, v, kn, vn)
        b.attend(250, 2, scale=scale, size=sq)
    b = Many(1, 1, 64, 1300000, dtype, seed=6)
    (k, kn), (v, vn) = rows(b.rng, (1, 1300, 1, 64), dtype), rows(b.rng, (1, 1300, 1, 64), dtype)
    rise = torch.linspace(0, 40, 1300).to(TYPES[dtype])
    k[0, :, 0, 0], kn[0, :, 0, 0] = rise.cuda(), rise.double().numpy()
    b.put(k, v, kn, vn)
    q, qn = rows(b.rng, (1, 125, 1, 64), dtype, 0.1)
    q[..., 0], qn[..., 0] = 20.0, 20.0
    want, off = b.r.attend(qn, prob=prob_step(dtype, True))
    near(b.c.attend(q), want, off, dtype)


def test_rows_in_any_strides():
    for dtype in ("f32", "bf16", "f16"):
        for dim in (64, 80, 128):
            b = Many(2, 2, dim, 300000, dtype, seed=dim)
            b.append(170, counts=[170, 81])
            big, _ = rows(b.rng, (2, 6, 126, dim + 3), dtype)
            for q in (big.transpose(1, 2)[..., 1:dim + 1], big.transpose(1, 2)[:, ::1, :4, :dim], big.transpose(1, 2)[:, :, 2:, 3:]):
                out = torch.full((2, 126, q.shape[2], dim + 5), 7.0, dtype=q.dtype, device="cuda")
                got = b.c.attend(q, out=out[..., 2:dim + 2])
                assert torch.equal(got, b.c.attend(q.contiguous()))
                assert (out[..., :2] == 7).all() and (out[..., dim + 2:] == 7).all()


def test_captured_beside_eager_calls():
    """A chunk appended and attended to with its weights, replayed, against the same calls one by one."""
    a, c = (Many(2, 2, 64, 300000, "f32", seed=3) for _ in range(2))
    for x in (a, c):
        x.append(900, counts=[900, 300])
    q, _ = rows(a.rng, (2, 125, 4, 64))
    k, _ = rows(a.rng, (2, 125, 2, 64))
    counts = ints([125, 125])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.c.append(k, k, counts=counts)
        got = a.c.attend(q, counts=counts, weigh=0.5)
    for n in ([125, 125], [125, 0], [17, 101]):
        q.normal_()
        k.normal_()
        counts.copy_(torch.tensor(n))
        graph.replay()
        c.c.append(k, k, counts=counts)
        want = c.c.attend(q, counts=counts, weigh=0.5)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and a.c.lengths() == c.c.lengths()
        assert torch.equal(a.c.weights(1200), c.c.weights(1200))


def test_results_are_the_same_every_time():
    for dim, dtype in ((64, "f32"), (128, "bf16")):
        b = Many(2, 2, dim, 300000, dtype, seed=9)
        b.append(3000, counts=[3000, 1777])
        q, _ = rows(b.rng, (2, 128, 8, dim), dtype)
        first = b.c.attend(q, weigh=0.0)
        w = b.c.weights(3000)
        for _ in range(4):
            assert torch.equal(b.c.attend(q, weigh=0.0), first) and torch.equal(b.c.weights(3000), w)


def test_rows_of_a_tile_do_not_depend_on_the_others():
    """A query by itself among padding, and among others that see keys of quite other sizes."""
    b = Many(1, 1, 64, 1300000, "bf16", seed=2)
    b.append(700)
    q, _ = rows(b.rng, (1, 120, 1, 64), "bf16")
    alone = b.c.attend(q)
    loud = q.clone()
    loud[:, ::2] *= 50
    assert torch.equal(b.c.attend(loud)[:, 1::2], alone[:, 1::2])
    assert np.isfinite(alone.double().cpu().numpy()).all()
