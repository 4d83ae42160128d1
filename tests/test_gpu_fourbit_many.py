"""The 4-bit cache's attention for many rows against the definition in 64 bits
(fourbit_ref.py). The kernel for it is chosen where the columns of the queries
times the tiles that the capacity allows are many, so capacities here are large and
sequences short: the keys of a few workgroups are then split as far as they can be."""
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

    def attend(self, n, heads, **how):
        S, H, _ = self.shape
        columns = n * heads // H
        assert columns > 96 and -(-columns // 16) * S * H * (self.r.cap // 32) > 60000, "not the kernel of many rows"
        return super().attend(n, heads, **how)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 80, 24])
@pytest.mark.parametrize("heads", [2, 6, 10])
def test_attends(dim, dtype, heads):
    b = Many(3, 2, dim, 60000, dtype, seed=dim + heads)
    b.attend(100, heads)                           # (nothing there)
    b.append(1)
    b.attend(99, heads)
    b.append(40, counts=[40, 0, 13])
    b.attend(130, heads, counts=[41, 130, 0])      # (the second asks for more than there are)
    b.append(300, counts=[300, 62, 97])
    b.attend(100, heads, scale=-0.3)
    b.attend(200, heads, counts=[200, 63, 7], weigh=1.0)
    b.append(200, counts=[150, 1, 181])
    b.attend(101, heads, scale=0.0)
    b.attend(129, heads, counts=[0, 1, 129], weigh=0.5)
    b.attend(257, heads)


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "f32"), (128, "bf16"), (64, "f16"), (128, "f16"), (20, "bf16")])
def test_more_tiles_than_the_device_takes_at_once(dim, dtype):
    b = Many(5, 27, dim, 3200, dtype, seed=dim)
    b.append(210, counts=[210, 70, 0, 1, 130])
    b.attend(131, 27, counts=[131, 65, 3, 2, 100], weigh=1.0)
    b.attend(258, 27)


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16"), (128, "f16"), (128, "f32")])
def test_long_sequences_are_split(dim, dtype):
    b = Many(2, 1, dim, 200000, dtype, seed=dim)
    b.append(6500, counts=[6500, 4111])
    b.attend(110, 1)
    b.attend(150, 2, counts=[150, 3])
    b.append(64, start=[63, 4111])
    b.attend(75, 4, counts=[0, 70], weigh=1.0)
    b.attend(128, 1, counts=[127, 1], weigh=0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_finite_reaches_those_that_see_it(dim, dtype):
    S, T, H = 3, 150, 2
    b = Many(S, H, dim, 60000, dtype, seed=dim)
    (k, kn), (v, vn) = (rows(b.rng, (S, T, H, dim), dtype) for _ in range(2))
    k[0, 100, 0, 5] = v[0, 60, 1, 40] = v[1, 147, 0, 0] = k[2, 149, 1, 3] = v[2, 120:, :, 7] = float("nan")
    kn[:], vn[:] = k.double().cpu().numpy(), v.double().cpu().numpy()
    b.c.append(k, v)
    b.r.append(kn, vn)
    for n in (60, 130):
        for counts in (None, [n, n - 3, n // 2]):
            b.attend(n, 4 * H, counts=counts)
    b.c.append(k[:, :0], v[:, :0], start=ints([99, 60, 110]))
    b.r.append(kn[:, :0], vn[:, :0], start=[99, 60, 110])
    for n in (59, 90):
        got = b.attend(n, 4 * H)
        assert torch.isfinite(got[1:]).all() and torch.isfinite(got[0, :, :4]).all()
    q = torch.zeros(S, 60, 3 * H, dim, dtype=TYPES[dtype], device="cuda")
    q[1, 0, 3, dim - 1], q[1, 59, 2, 0] = float("inf"), float("nan")
    got = b.c.attend(q)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[1, 0, 3] = bad[1, 59, 2] = True
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[1:][~bad[1:]]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_ranges(dtype):
    for sk, sq, sv, scale in ((1e15, 1e-15, 1e30, 0.1), (1e-18, 1e10, 1e-25, 1e8), (1.0, 1e-30, 1.0, 1e30), (30.0, 1.0, 1.0, 1.0)):
        b = Many(1, 1, 64, 200000, dtype, seed=4)
        (k, kn), (v, vn) = rows(b.rng, (1, 300, 1, 64), dtype, sk), rows(b.rng, (1, 300, 1, 64), dtype, sv)
        b.put(k, v, kn, vn)
        b.attend(150, 2, scale=scale, size=sq)
    b = Many(1, 1, 64, 400000, dtype, seed=6)
    (k, kn), (v, vn) = rows(b.rng, (1, 1300, 1, 64), dtype), rows(b.rng, (1, 1300, 1, 64), dtype)
    rise = torch.linspace(0, 40, 1300).to(TYPES[dtype])
    k[0, :, 0, 0], kn[0, :, 0, 0] = rise.cuda(), rise.double().numpy()
    b.put(k, v, kn, vn)
    q, qn = rows(b.rng, (1, 140, 1, 64), dtype, 0.1)
    q[..., 0], qn[..., 0] = 20.0, 20.0
    want, off = b.r.attend(qn, prob=prob_step(dtype, True))
    near(b.c.attend(q), want, off, dtype)


def test_rows_in_any_strides():
    for dtype in ("f32", "bf16", "f16"):
        for dim in (64, 80, 128):
            b = Many(2, 2, dim, 60000, dtype, seed=dim)
            b.append(170, counts=[170, 81])
            big, _ = rows(b.rng, (2, 6, 130, dim + 3), dtype)
            for q in (big.transpose(1, 2)[..., 1:dim + 1], big.transpose(1, 2)[:, ::1, :4, :dim], big.transpose(1, 2)[:, :, 2:, 3:]):
                out = torch.full((2, 130, q.shape[2], dim + 5), 7.0, dtype=q.dtype, device="cuda")
                got = b.c.attend(q, out=out[..., 2:dim + 2])
                assert torch.equal(got, b.c.attend(q.contiguous()))
                assert (out[..., :2] == 7).all() and (out[..., dim + 2:] == 7).all()


def test_captured_beside_eager_calls():
    """A chunk appended and attended to with its weights, replayed, against the same calls one by one."""
    a, c = (Many(2, 2, 64, 60000, "f32", seed=3) for _ in range(2))
    for x in (a, c):
        x.append(900, counts=[900, 300])
    q, _ = rows(a.rng, (2, 130, 4, 64))
    k, _ = rows(a.rng, (2, 130, 2, 64))
    counts = ints([130, 130])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.c.append(k, k, counts=counts)
        got = a.c.attend(q, counts=counts, weigh=0.5)
    for n in ([130, 130], [130, 0], [17, 101]):
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
        b = Many(2, 2, dim, 60000, dtype, seed=9)
        b.append(3000, counts=[3000, 1777])
        q, _ = rows(b.rng, (2, 130, 8, dim), dtype)
        first = b.c.attend(q, weigh=0.0)
        w = b.c.weights(3000)
        for _ in range(4):
            assert torch.equal(b.c.attend(q, weigh=0.0), first) and torch.equal(b.c.weights(3000), w)


def test_rows_of_a_tile_do_not_depend_on_the_others():
    """A query by itself among padding, and among others that see keys of quite other sizes."""
    b = Many(1, 1, 64, 400000, "bf16", seed=2)
    b.append(700)
    q, _ = rows(b.rng, (1, 120, 1, 64), "bf16")
    alone = b.c.attend(q)
    loud = q.clone()
    loud[:, ::2] *= 50
    assert torch.equal(b.c.attend(loud)[:, 1::2], alone[:, 1::2])
    assert np.isfinite(alone.double().cpu().numpy()).all()
