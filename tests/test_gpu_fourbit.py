"""The 4-bit key/value cache on the GPU against its definition in 64 bits
(fourbit_ref.py): what it holds, exactly, attention over it, weights and eviction."""
import numpy as np
import pytest
import torch

from rusttorch_amd.q4cache import FourBitCache, Gpt2Error
from tests.fourbit_ref import U, Cache, held

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rows(rng, shape, dtype="f32", size=1.0):
    """Values of dtype on the GPU, and the same as float64."""
    x = torch.from_numpy(rng.standard_normal(shape) * size).to(TYPES[dtype])
    return x.cuda(), x.double().numpy()


def ints(x):
    return None if x is None else torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def prob_step(dtype, many):
    """What a probability is rounded by, relative: three bf16 parts for f32, two cut ones (16 bits) for the others,
    bf16 to nearest for bf16 rows where the kernel of many rows may be chosen."""
    return 2.0 ** -24 if dtype == "f32" else 2.0 ** -9 if dtype == "bf16" and many else 2.0 ** -15


def near(got, want, off, dtype):
    """got against want, which is off by `off` at most before it is rounded to dtype."""
    g = got.double().cpu().numpy()
    # (half a step of the type, of what is off too, and f16's and f32's subnormals)
    step = torch.finfo(TYPES[dtype]).eps / 2
    most = off + (np.abs(want) + off) * step + torch.finfo(TYPES[dtype]).smallest_normal * step
    bad = ~(np.abs(g - want) <= most)
    bad &= ~((np.isnan(g) & np.isnan(want)))
    assert not bad.any(), (f"{bad.sum()} of {bad.size} values, first at {np.argwhere(bad)[0]}: "
                           f"{g[bad][0]} for {want[bad][0]}, off by {np.abs(g - want)[bad][0]}, may be {most[bad][0]}")


class Both:
    """A cache on the GPU and its definition, fed the same."""

    def __init__(self, n_seq, n_head, dim, cap, dtype="f32", seed=0):
        print(f"[gpu] fourbit {n_seq} x {n_head} x {dim}, capacity {cap}, {dtype}, seed {seed}", flush=True)
        self.c = FourBitCache(n_seq, n_head, dim, cap)
        self.r = Cache(n_seq, n_head, dim, cap)
        self.shape, self.dtype, self.rng = (n_seq, n_head, dim), dtype, np.random.default_rng(seed)

    def append(self, n, counts=None, start=None, size=1.0):
        S, H, D = self.shape
        (k, kn), (v, vn) = (rows(self.rng, (S, n, H, D), self.dtype, size) for _ in range(2))
        self.put(k, v, kn, vn, counts, start)

    def put(self, k, v, kn, vn, counts=None, start=None):
        self.c.append(k, v, counts=ints(counts), start=ints(start))
        refused = self.r.append(kn, vn, counts, start)
        if refused:
            with pytest.raises(Gpt2Error, match=f"sequence {refused[0]}:"):
                self.c.lengths()
        self.same()

    def same(self, n=None, first=None, dtype="f32"):
        assert self.c.lengths() == [self.r.length(s) for s in range(self.shape[0])]
        n = self.r.cap + 3 if n is None else n
        got = self.c.read(n, first=ints(first), dtype=TYPES[dtype])
        for g, w in zip(got, self.r.read(n, first)):
            g, w = g.double().cpu().numpy(), torch.from_numpy(w).to(TYPES[dtype]).double().numpy()
            assert np.array_equal(g, w, equal_nan=True), f"{np.sum(g != w)} values differ"

    def attend(self, n, heads, counts=None, scale=None, dtype=None, weigh=None, size=1.0):
        S, H, D = self.shape
        dtype = self.dtype if dtype is None else dtype
        print(f"[gpu]   attend {n} x {heads}, counts {counts}, scale {scale}, {dtype}, weigh {weigh}", flush=True)
        q, qn = rows(self.rng, (S, n, heads, D), dtype, size)
        got = self.c.attend(q, counts=ints(counts), scale=scale, weigh=weigh)
        want, off = self.r.attend(qn, counts, scale, prob_step(dtype, n * heads // H > 32), weigh)
        near(got, want, off, dtype)
        if weigh is not None:
            self.weights()
        return got

    def weights(self):
        n = self.r.cap + 2
        got = self.c.weights(n).double().cpu().numpy()
        for s in range(self.shape[0]):
            for h in range(self.shape[1]):
                w, off = self.r.w[s][h], self.r.w_off[s][h]
                far = np.abs(got[s, h, :len(w)] - w) - off * (1 + 2 * U) - np.abs(w) * U
                assert far.max(initial=0) <= 0, f"sequence {s}, head {h}: {far.max()} further off than the sums' rounding"
                assert (got[s, h, len(w):] == 0).all()


@pytest.mark.parametrize("heads,dim,dtype", [(3, 64, "f32"), (2, 128, "bf16"), (5, 20, "f16"), (1, 5, "f32"),
                                             (2, 80, "f32"), (2, 33, "bf16"), (1, 1, "f32"), (3, 100, "f16"), (1, 96, "f32")])
def test_holds_what_it_is_given(heads, dim, dtype):
    b = Both(3, heads, dim, 333, dtype, seed=dim)
    b.append(1)
    b.append(2, size=3.0)
    b.append(70, size=0.5)
    b.append(64)
    b.append(129, counts=[129, 0, 63])
    b.append(5, counts=[-4, 7, 5])
    b.same(n=40, first=[250, 130, -7])
    b.same(n=40, first=[2 ** 31 - 1, -2 ** 31, 3], dtype="bf16")
    b.append(200)                # sequence 0 has no room left
    b.append(3, counts=[3, 0, 1])
    b.append(7, start=[100, 5, 0])
    b.append(0, start=[99, 12, 3])
    b.append(2, start=[300, -1, 4], counts=[2, 2, 2])  # 0, 1: refused


@pytest.mark.parametrize("e", [-140, -103, -101, -100, -99, -1, 0, 1, 100, 124, 125])
def test_numbers_and_ties(e):
    """Every number, every border between two, and their neighbours in f32, with every sign, under many scales."""
    at = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], np.float32)
    x = np.concatenate([at, np.nextafter(at, np.float32(9)), np.nextafter(at, np.float32(0)), -at, -np.nextafter(at, np.float32(9))])
    x = (x.astype(np.float64) * 2.0 ** e).astype(np.float32)  # (subnormal ones are rounded here already)
    x = x[np.isfinite(x)]
    rng = np.random.default_rng(e + 200)
    tops = np.array([7, 6, 4, 3.4, 1.75, 1, 0]) * 2.0 ** min(e, 125)
    k = rng.choice(x, (1, 7, 2, 64)).astype(np.float32)
    for i, top in enumerate(tops):
        k[0, i] = np.clip(k[0, i], -top, top)
    b = Both(1, 2, 64, 40, seed=e + 200)
    t = torch.from_numpy(k).cuda()
    b.put(t, -t, k.astype(np.float64), -k.astype(np.float64))


def test_values_that_are_not_finite():
    b = Both(2, 2, 96, 50, seed=3)
    (k, kn), (v, vn) = (rows(b.rng, (2, 40, 2, 96)) for _ in range(2))
    for x, xn in ((k, kn), (v, vn)):
        for at, bad in (((0, 3, 1, 40), np.nan), ((1, 7, 0, 95), np.inf), ((1, 39, 1, 0), -np.inf)):
            x[at], xn[at] = bad, bad
    b.put(k, v, kn, vn)
    b.same(dtype="f16")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 80, 24])
@pytest.mark.parametrize("heads", [2, 6, 10])
def test_attends(dim, dtype, heads):
    b = Both(3, 2, dim, 700, dtype, seed=dim + heads)
    b.append(1)
    b.attend(1, heads)
    b.append(30, counts=[30, 0, 13])
    b.attend(1, heads)
    b.attend(7, heads, counts=[7, 1, 0])
    b.attend(40, heads, counts=[31, 40, 14])   # (the last two ask for more than there are)
    b.append(200, counts=[200, 64, 97])
    b.attend(1, heads, counts=[1, 0, 1])
    b.attend(9, heads)
    b.attend(65, heads, counts=[65, 33, 2])
    b.append(300, counts=[300, 0, 199])
    b.attend(3, heads)
    b.attend(130, heads, counts=[130, 60, 7])
    b.attend(66, heads, scale=-0.3)
    b.attend(2, heads, scale=0.0)
    b.attend(70, heads, scale=0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_groups_that_are_large(dtype):
    b = Both(1, 1, 64, 300, dtype, seed=5)
    b.append(257)
    for heads in (7, 16, 17, 33, 129, 300):
        b.attend(1, heads)
        b.attend(3, heads)


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16"), (128, "f16"), (128, "f32")])
def test_long_sequences_are_split(dim, dtype):
    b = Both(2, 1, dim, 9000, dtype, seed=dim)
    b.append(8800, counts=[8800, 4111])
    b.attend(1, 4)
    b.attend(2, 1, counts=[2, 1])
    b.append(1)
    b.attend(5, 2)
    b.attend(80, 1)
    b.attend(150, 2, counts=[150, 3])
    b.attend(70, 4, counts=[0, 70], weigh=1.0)


def test_rows_in_any_strides():
    rng = np.random.default_rng(8)
    for dtype in ("f32", "bf16"):
        for dim in (64, 80):
            big, _ = rows(rng, (2, 3, 50, 4, dim + 3), dtype)
            views = [big[:, 0, :, :2, 1:dim + 1], big[:, 1, :, 2:, 3:], big[:, 2, ::2, ::2, :dim], big.transpose(1, 2)[:, :, 1, 1:3, :dim]]
            for k, v in ((views[0], views[1]), (views[2], views[2]), (views[3], views[0])):
                a, c = FourBitCache(2, 2, dim, 60), FourBitCache(2, 2, dim, 60)
                a.append(k, v)
                c.append(k.contiguous(), v.contiguous())
                assert all(torch.equal(x, y) for x, y in zip(a.read(60), c.read(60)))
                for q in (k[:, :5], k):
                    out = torch.full((2, q.shape[1], 2, dim + 5), 7.0, dtype=k.dtype, device="cuda")
                    got = a.attend(q, out=out[..., 2:dim + 2])
                    assert torch.equal(got, c.attend(q.contiguous())) and (out[..., :2] == 7).all() and (out[..., dim + 2:] == 7).all()
                kk = torch.full((2, 70, 2, dim + 1), 7.0, dtype=k.dtype, device="cuda")
                a.read(65, dtype=k.dtype, k=kk[:, 2:67, :, :dim])
                assert torch.equal(kk[:, 2:67, :, :dim], c.read(65, dtype=k.dtype)[0])
                assert (kk[:, :2] == 7).all() and (kk[:, 67:] == 7).all() and (kk[..., dim] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_finite_reaches_those_that_see_it(dim, dtype):
    """A key: the rows that see it; a value: those rows' channels of its 32; a query: its row. Stale ones behind a
    sequence: nobody."""
    S, T, H = 3, 150, 2
    b = Both(S, H, dim, 200, dtype, seed=dim)
    (k, kn), (v, vn) = (rows(b.rng, (S, T, H, dim), dtype) for _ in range(2))
    k[0, 100, 0, 5] = v[0, 60, 1, 40] = v[1, 147, 0, 0] = k[2, 149, 1, 3] = v[2, 120:, :, 7] = float("nan")
    kn[:], vn[:] = k.double().cpu().numpy(), v.double().cpu().numpy()
    b.c.append(k, v)
    b.r.append(kn, vn)
    for n in (1, 4, 60, 130):
        for counts in (None, [n, max(n - 3, 0), n // 2]):
            b.attend(n, 2 * H, counts=counts)
    b.c.append(k[:, :0], v[:, :0], start=ints([99, 60, 110]))
    b.r.append(kn[:, :0], vn[:, :0], start=[99, 60, 110])
    for n in (1, 3, 59, 90):
        got = b.attend(n, 2 * H)
        assert torch.isfinite(got[1:]).all() and torch.isfinite(got[0, :, :2]).all()
    q = torch.zeros(S, 70, H, dim, dtype=TYPES[dtype], device="cuda")
    q[1, 0, 1, dim - 1], q[1, 69, 0, 0] = float("inf"), float("nan")
    for n, group in ((3, 1), (60, 3)):
        part = torch.cat([q[:, :1], q[:, 71 - n:]], 1).repeat_interleave(group, 2)
        got = b.c.attend(part)
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[1, 0, group:2 * group] = bad[1, n - 1, :group] = True
        assert torch.isnan(got[bad]).all() and torch.isfinite(got[1:][~bad[1:]]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_ranges(dtype):
    """Keys, queries and values of very different sizes, channels of a query far apart, scores that rise all the way."""
    for sk, sq, sv, scale in ((1e15, 1e-15, 1e30, 0.1), (1e-18, 1e10, 1e-25, 1e8), (1.0, 1e-30, 1.0, 1e30), (30.0, 1.0, 1.0, 1.0)):
        b = Both(1, 1, 64, 400, dtype, seed=4)
        (k, kn), (v, vn) = rows(b.rng, (1, 300, 1, 64), dtype, sk), rows(b.rng, (1, 300, 1, 64), dtype, sv)
        b.put(k, v, kn, vn)
        for n in (2, 150):
            b.attend(n, 2, scale=scale, size=sq)
    b = Both(1, 1, 64, 400, dtype, seed=6)
    (k, kn), (v, vn) = rows(b.rng, (1, 300, 1, 64), dtype), rows(b.rng, (1, 300, 1, 64), dtype)
    rise = torch.linspace(0, 40, 300).to(TYPES[dtype])
    k[0, :, 0, 0], kn[0, :, 0, 0] = rise.cuda(), rise.double().numpy()
    b.put(k, v, kn, vn)
    q, qn = rows(b.rng, (1, 140, 1, 64), dtype, 0.1)
    q[..., 0], qn[..., 0] = 20.0, 20.0
    for n in (1, 140):
        want, off = b.r.attend(qn[:, 140 - n:], prob=prob_step(dtype, n > 32))
        near(b.c.attend(q[:, 140 - n:]), want, off, dtype)


# -- weights and eviction --


@pytest.mark.parametrize("dim,dtype,heads", [(64, "f32", 3), (128, "bf16", 12), (80, "f16", 6), (128, "f32", 3)])
def test_weights(dim, dtype, heads):
    b = Both(3, 3, dim, 500, dtype, seed=dim + heads)
    b.append(100, counts=[100, 0, 33])
    b.attend(1, heads, weigh=1.0)
    b.attend(5, heads, counts=[5, 3, 0], weigh=1.0)
    b.append(250, counts=[250, 2, 64])
    b.weights()
    b.attend(1, heads, weigh=0.5)
    b.attend(40, heads, counts=[40, 1, 7], weigh=1.0)
    b.attend(100, heads, counts=[100, 0, 50], weigh=0.25)
    b.append(3, start=[200, 1, 97])
    b.weights()
    b.attend(2, heads, weigh=0.0)
    x = torch.rand(3, 3, 210, generator=torch.Generator().manual_seed(1))
    b.c.add_weights(x.cuda())
    for s in range(3):
        for h in range(3):
            n = min(b.r.length(s), 210)
            b.r.w[s][h][:n] += x[s, h, :n].double().numpy()
            b.r.w_off[s][h] += b.r.w[s][h] * U
    b.weights()
    b.attend(1, heads, weigh=1.0)
    assert b.c.weights(0).shape == (3, 3, 0)


def test_weights_that_begin_anew_forget_what_is_not_finite():
    b = Both(1, 1, 64, 100, seed=2)
    b.append(50)
    b.c.add_weights(torch.full((1, 1, 50), float("nan"), device="cuda"))
    assert torch.isnan(b.c.weights(50)).all()
    b.attend(1, 2, weigh=0.0)


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16"), (80, "f32"), (20, "f16")])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (50, 8), (64, 64), (200, 0), (333, 30), (4999, 100), (5000, 3)])
def test_evicts(dim, dtype, keep, recent):
    S, H = 3, 2
    b = Both(S, H, dim, 5000, dtype, seed=keep + dim)
    b.append(5000, counts=[5000, 333, 20])
    w = np.exp(2 * b.rng.standard_normal((S, H, 5000))).astype(np.float32)
    w[0, 0, ::3] = 0            # (many of the same)
    w[0, 1] = np.round(w[0, 1])
    w[1, 0, 50:90] = np.nan
    w[1, 1, 7], w[1, 1, 8], w[1, 1, 9:30] = np.inf, -np.inf, -1.5
    w[1, 1, 30:40] = -0.0
    b.c.add_weights(torch.from_numpy(w).cuda())
    for s in range(S):
        for h in range(H):
            b.r.w[s][h][:] = w[s, h, :b.r.length(s)]
    got = b.c.evict(keep, recent=recent).cpu().numpy()
    want = b.r.evict(keep, recent)
    assert np.array_equal(got, want)
    b.same()
    left = b.c.weights(keep).cpu().numpy()
    for s in range(S):
        for h in range(H):
            assert np.array_equal(left[s, h, :b.r.length(s)], b.r.w[s][h].astype(np.float32), equal_nan=True)
    b.append(1, counts=[1, 1, 1] if keep < 5000 else [0, 1, 1])
    b.attend(1, 2 * H)


def test_evicts_of_equal_weights():
    b = Both(1, 1, 64, 3000, seed=1)
    b.append(3000)
    got = b.c.evict(1000, recent=10).cpu().numpy()[0, 0]
    assert np.array_equal(got, np.r_[0:990, 2990:3000])
    b.r.evict(1000, 10)
    b.same()


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16")])
def test_a_cache_within_a_budget(dim, dtype):
    """As a program uses it: a prompt, its last positions' attention, a cut, then tokens one by one, each cut again."""
    b = Both(2, 2, dim, 420, dtype, seed=dim)
    b.append(400, counts=[400, 150])
    b.attend(16, 8, weigh=1.0)
    for step in range(6):
        # (whom equal or nearly equal weights keep is the GPU's to say: the definition takes its weights)
        mine = b.c.weights(420).double().cpu().numpy()
        for s in range(2):
            for h in range(2):
                b.r.w[s][h][:], b.r.w_off[s][h][:] = mine[s, h, :b.r.length(s)], 0
        kept = b.c.evict(64, recent=8).cpu().numpy()
        assert np.array_equal(kept, b.r.evict(64, 8))
        b.same()
        b.append(3)
        b.attend(3, 8, weigh=0.9)


def test_a_cache_past_32_bits():
    """600 sequences of 8 heads of 128, 16000 tokens each: 4.9 GB of keys' codes; what the last ones hold."""
    S, H, D, n = 600, 8, 128, 500
    big, small = FourBitCache(S, H, D, 16000), FourBitCache(2, H, D, 16000)
    k, v, q = (torch.randn(1, n, h, D, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").bfloat16()
               for i, h in ((1, H), (2, H), (3, 4 * H)))
    counts = torch.zeros(S, dtype=torch.int32, device="cuda")
    counts[-2:] = n
    big.append(k.expand(S, n, H, D), v.expand(S, n, H, D), counts=counts)
    small.append(k.expand(2, n, H, D), v.expand(2, n, H, D))
    assert big.lengths() == [0] * (S - 2) + [n, n]
    assert all(torch.equal(a[-2:], b) for a, b in zip(big.read(20), small.read(20)))
    for m in (1, 40):
        a = big.attend(q[:, :m].expand(S, m, 4 * H, D), weigh=0.0)
        b = small.attend(q[:, :m].expand(2, m, 4 * H, D), weigh=0.0)
        # (the two may be split differently: f32 sums in another order, bf16's last place)
        assert torch.allclose(a[-2:].float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -9) and (a[:-2] == 0).all()
        assert torch.allclose(big.weights(n)[-2:], small.weights(n), rtol=1e-4, atol=1e-6)
    kept = big.evict(100, recent=10)
    assert (kept[:-2] == -1).all() and big.lengths()[-2:] == [100, 100]
    at = kept[-1].long()
    want = FourBitCache(1, H, D, 600)
    want.append(k, v)
    want = want.read(n)[1][0]
    got = big.read(100)[1][-1]
    assert all(torch.equal(got[:, h], want[at[h], h]) for h in range(H))


# -- streams, captures, refusals --


def test_captured_and_replayed():
    S, H, D = 2, 2, 64
    rng = np.random.default_rng(0)
    k, v, q = (rows(rng, (S, 1, H * (2 if i == 2 else 1), D))[0] for i in range(3))
    prompt = rows(rng, (S, 90, H, D))[0]

    def step(c):
        c.append(k, v)
        out = c.attend(q, weigh=0.5)
        kept = c.evict(80, recent=4)
        return out, kept, c.weights(85), c.read(80)[0]

    plain, graphed = FourBitCache(S, H, D, 100), FourBitCache(S, H, D, 100)
    for c in (plain, graphed):
        c.append(prompt, -prompt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = FourBitCache(S, H, D, 100)
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(graphed)
        with pytest.raises(Gpt2Error, match="being captured"):
            graphed.lengths()
    assert graphed.lengths() == [90, 90]
    for i in range(4):
        k.copy_(rows(rng, k.shape)[0])
        q.copy_(rows(rng, q.shape)[0])
        g.replay()
        want = step(plain)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        assert graphed.lengths() == plain.lengths() == [80, 80]


def test_on_another_stream():
    b = Both(1, 2, 64, 100, seed=1)
    side = torch.cuda.Stream()
    (k, kn), (v, vn) = (rows(b.rng, (1, 70, 2, 64)) for _ in range(2))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        k2 = k * 2
        b.c.append(k2, v)
        out = b.c.attend(k2[:, :3], weigh=1.0)
        b.r.append(kn * 2, vn)
        b.same()
        want, off = b.r.attend(kn[:, :3] * 2, weigh=1.0, prob=2.0 ** -24)
        near(out, want, off, "f32")
        b.weights()


def test_results_are_the_same_every_time():
    b = Both(4, 2, 128, 6000, "bf16", seed=2)
    b.append(6000, counts=[6000, 100, 3000, 1])
    for n in (1, 5, 90):
        q = rows(b.rng, (4, n, 8, 128), "bf16")[0]
        first = b.c.attend(q, weigh=0.0)
        w = b.c.weights(6000)
        for _ in range(4):
            assert torch.equal(b.c.attend(q, weigh=0.0), first) and torch.equal(b.c.weights(6000), w)


def test_refuses():
    c = FourBitCache(2, 2, 64, 50)
    x = torch.zeros(2, 4, 2, 64, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call, what in [
        (lambda: c.append(x[:1], x[:1]), "must be \\[2, 4, 2, 64\\]"), (lambda: c.append(x, x.half()), "must be torch.float32"),
        (lambda: c.append(x.double(), x), "f32, bf16 or f16"), (lambda: c.append(x.cpu(), x), "the cache on"),
        (lambda: c.append(x.requires_grad_(), x), "requires a gradient"),
        (lambda: c.append(x.detach().transpose(2, 3).contiguous().transpose(2, 3), x.detach()), "last dimension"),
        (lambda: c.append(torch.zeros(2, 51, 2, 64, device="cuda"), torch.zeros(2, 51, 2, 64, device="cuda")), "exceed"),
        (lambda: c.append(x.detach(), x.detach(), counts=i.long()), "2 contiguous int32"),
        (lambda: c.attend(x.detach()[:, :, :1].expand(2, 4, 3, 64)), "not a multiple"),
        (lambda: c.attend(x.detach(), scale=float("nan")), "scale must be finite"),
        (lambda: c.attend(x.detach(), weigh=1.5), "weigh must be"), (lambda: c.attend(x.detach(), weigh=-0.1), "weigh must be"),
        (lambda: c.evict(0), "keep 0"), (lambda: c.evict(51), "keep 51"), (lambda: c.evict(5, recent=6), "recent 6"),
        (lambda: c.add_weights(torch.zeros(2, 2, 4)), "the cache on"), (lambda: c.add_weights(x.detach()), "contiguous float32"),
        (lambda: c.weights(-1), "negative"), (lambda: c.read(-1), "negative"), (lambda: c.read(3, dtype=torch.float64), "f32, bf16"),
    ]:
        with pytest.raises(Gpt2Error, match=what):
            call()
    assert c.lengths() == [0, 0]
    out = c.attend(x.detach())      # (nothing there: zeros)
    assert (out == 0).all() and c.attend(x.detach()[:, :0]).shape == (2, 0, 2, 64)
    assert (c.attend(x.detach(), weigh=1.0) == 0).all() and (c.weights(3) == 0).all()
    assert (c.evict(3) == -1).all() and c.lengths() == [0, 0]
    c.close()
    with pytest.raises(Gpt2Error, match="closed"):
        c.append(x.detach(), x.detach())


def test_definition_of_halves():
    """What f16 and bf16 rows are held as is what the same values in f32 are."""
    rng = np.random.default_rng(3)
    for dtype in ("bf16", "f16"):
        x, xn = rows(rng, (1, 30, 1, 64), dtype)
        c = FourBitCache(1, 1, 64, 30)
        c.append(x, x)
        assert np.array_equal(c.read(30)[0].double().cpu().numpy(), held(xn))
    assert U == 2.0 ** -24
