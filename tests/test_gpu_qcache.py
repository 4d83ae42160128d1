"""The 8-bit key/value cache on the GPU against its definition in 64 bits
(qcache_ref.py): what it holds, bit for bit, and attention over it."""
import numpy as np
import pytest
import torch

from rusttorch_amd.qcache import Gpt2Error, QuantisedCache
from tests.qcache_ref import Cache

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 2.0 ** -24


def rows(rng, shape, dtype="f32", size=1.0):
    """Values of dtype on the GPU, and the same as float64."""
    x = torch.from_numpy(rng.standard_normal(shape) * size).to(TYPES[dtype])
    return x.cuda(), x.double().numpy()


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


class Both:
    """A cache on the GPU and its definition, fed the same."""

    def __init__(self, n_seq, n_head, dim, cap, block, dtype="f32", seed=0):
        print(f"[gpu] qcache {n_seq} x {n_head} x {dim}, capacity {cap}, block {block}, {dtype}, seed {seed}", flush=True)
        self.c = QuantisedCache(n_seq, n_head, dim, cap, block=block)
        self.r = Cache(n_seq, n_head, dim, cap, block)
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

    def same(self, n=None, first=None):
        assert self.c.lengths() == [self.r.length(s) for s in range(self.shape[0])]
        n = self.r.cap + 3 if n is None else n
        got = self.c.read(n, first=ints(first))
        for g, w in zip(got, self.r.read(n, first)):
            g = g.cpu().numpy()
            assert np.array_equal(g, w, equal_nan=True), f"{np.sum(g != w)} values differ"


@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("heads,dim,dtype", [(3, 64, "f32"), (2, 128, "bf16"), (5, 20, "f16"), (1, 5, "f32"), (2, 80, "f32")])
def test_holds_what_it_is_given(block, heads, dim, dtype):
    b = Both(3, heads, dim, 333, block, dtype, seed=block + dim)
    b.append(1)
    b.append(2, size=3.0)        # (a larger token: the open block is quantised anew)
    b.append(70, size=0.5)
    b.append(64)
    b.append(129, counts=[129, 0, 63])
    b.append(5, counts=[-4, 7, 5])
    b.same(n=40, first=[250, 130, -7])
    b.append(200)                # sequence 0 has no room left
    b.append(3, counts=[3, 0, 1])


@pytest.mark.parametrize("block", [16, 64])
def test_how_tokens_are_split_does_not_matter(block):
    rng = np.random.default_rng(5)
    (k, _), (v, _) = (rows(rng, (2, 150, 3, 64)) for _ in range(2))
    caches = []
    for cuts in ([150], [1] * 150, [63, 1, 64, 22], [17, 100, 33]):
        c, at = QuantisedCache(2, 3, 64, 160, block=block), 0
        for n in cuts:
            c.append(k[:, at:at + n], v[:, at:at + n])
            at += n
        caches.append(c)
    want = caches[0].read(150)
    for c in caches[1:]:
        got = c.read(150)
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("block", [16, 32, 64])
def test_cuts(block):
    b = Both(4, 2, 64, 260, block, seed=9)
    b.append(150, counts=[150, 97, 64, 33])
    b.append(3, start=[149, 96, 60, 31])              # inside the open block where there is one
    b.append(40, start=[70, 5, 64 // 2, 0])           # into full blocks, and from the first token
    b.append(0, start=[69, 41, 3, 0])                 # nothing new
    b.append(1, start=[68, 41, 2, 0], counts=[1, 0, 1, 1])
    b.append(190, start=[69, 41, 3, 1], counts=[190, 190, 1, 0])
    b.append(2, start=[300, -1, 4, 1], counts=[2, 2, 2, 2])  # 0, 1: refused


@pytest.mark.parametrize("block", [16, 32, 64])
def test_cuts_to_the_end_of_a_block(block):
    # what is left ends with a full block, which later calls go back into
    for by_counts in (False, True):
        b = Both(3, 2, 64, 300, block, seed=21)
        b.append(3 * block + 6)
        ends = [2 * block, 3 * block, block]
        if by_counts:
            b.append(4, start=ends, counts=[0, 0, 0])
        else:
            b.append(0, start=ends)
        b.append(1, start=[x - 2 for x in ends])
        b.append(block + 3, start=[x - 1 for x in ends])
        b.append(0, start=ends)
        b.append(0, start=[x - 1 for x in ends])
        b.append(1)
        b.append(2)
        b.append(0, start=[0, 0, 0])
        b.append(2)


def test_many_cuts():
    rng = np.random.default_rng(22)
    for block in (16, 64):
        b = Both(5, 1, 20, 150, block, seed=block)
        for _ in range(40):
            n = int(rng.choice([0, 1, 1, 2, 17, 70]))
            lens = [b.r.length(s) for s in range(5)]
            start = [int(rng.integers(0, x + 1)) if rng.random() < 0.5 else x for x in lens] if rng.random() < 0.8 else None
            b.append(n, start=start, counts=rng.integers(0, n + 1, 5) if rng.random() < 0.5 else None, size=float(rng.uniform(0.2, 3)))


def test_cut_and_write_again_gives_the_same():
    b = Both(2, 2, 64, 200, 32, seed=11)
    b.append(75)
    (k, kn), (v, vn) = (rows(b.rng, (2, 60, 2, 64)) for _ in range(2))
    b.put(k, v, kn, vn, start=[75, 70])
    want = b.c.read(200)
    for _ in range(3):
        b.put(k, v, kn, vn, start=[75, 70])
        assert all(torch.equal(g, w) for g, w in zip(b.c.read(200), want))


def test_values_next_to_a_border_between_codes():
    # x = (n + 1/2) s and its neighbours, for scales of full and of few digits
    b = Both(1, 1, 64, 64, 16, seed=2)
    x = np.zeros((1, 48, 1, 64), np.float32)
    for t, top in enumerate((1.0, 0.7853982, 3.3333333, 127.0, 126.99999, 1e-30, 5e30, 0.1)):
        s = np.float32(np.float32(top) / np.float32(127))
        for j in range(6):
            n = b.rng.integers(0, 126, 64) * b.rng.choice([-1, 1], 64)
            v = ((n + 0.5) * np.float64(s)).astype(np.float32)
            x[0, t * 6 + j, 0] = [v, np.nextafter(v, np.float32(0)), np.nextafter(v, np.float32(1e38))][j % 3]
            x[0, t * 6 + j, 0, 0] = top
    for t in range(48):  # (one block per value of top: three tokens of it at a time)
        x[0, t] = x[0, t] if t % 16 < 12 else 0
    k = torch.from_numpy(x).cuda()
    b.put(k, -k, x.astype(np.float64), -x.astype(np.float64))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite(bad):
    b = Both(1, 2, 64, 200, 16, seed=4)
    (k, kn), (v, vn) = (rows(b.rng, (1, 70, 2, 64)) for _ in range(2))
    k[0, 20, 0, 7] = bad
    kn[0, 20, 0, 7] = bad
    v[0, 63, 1, 63] = bad
    vn[0, 63, 1, 63] = bad
    b.put(k, v, kn, vn)
    b.append(1)
    b.append(3, start=[25])    # the block keeps its NaN
    b.append(3, start=[20])    # the token is gone, but the block's others read back as NaN
    b.append(3, start=[16])


def test_zeros_and_the_smallest():
    b = Both(1, 1, 64, 100, 16)
    x = np.zeros((1, 64, 1, 64), np.float32)
    x[0, 20, 0, 3] = 1e-38          # below 127 * 2^-126: counts as 0
    x[0, 40, 0, 3] = 1.5e-36        # above
    x[0, 41, 0, :] = 1e-37
    k = torch.from_numpy(x).cuda()
    b.put(k, k, x.astype(np.float64), x.astype(np.float64))


def test_strides_and_alignment():
    rng = np.random.default_rng(8)
    S, T, H, D = 2, 37, 3, 64
    c, r = QuantisedCache(S, H, D, 64, block=32), Cache(S, H, D, 64, 32)
    qkv, n = rows(rng, (S, T, 3, H, D))                  # a fused projection's rows
    c.append(qkv[:, :, 1], qkv[:, :, 2])
    r.append(n[:, :, 1], n[:, :, 2])
    heads_first, m = rows(rng, (S, H, 6, D + 1))         # heads before tokens, rows of odd length and start
    k, v = heads_first[..., 1:].transpose(1, 2), heads_first[..., :D].transpose(1, 2)
    c.append(k, v)
    r.append(m[..., 1:].transpose(0, 2, 1, 3), m[..., :D].transpose(0, 2, 1, 3))
    one, o = rows(rng, (1, 2, 1, D))                     # one row for all
    c.append(one.expand(S, 2, H, D), one.expand(S, 2, H, D))
    r.append(np.broadcast_to(o, (S, 2, H, D)), np.broadcast_to(o, (S, 2, H, D)))
    for g, w in zip(c.read(64), r.read(64)):
        assert np.array_equal(g.cpu().numpy(), w)
    out = torch.full((S, 50, H + 1, D + 3), 7.0, device="cuda")
    k, v = out[:, 1:46, :H, 2:D + 2], torch.empty(S, 45, H, D, device="cuda")
    c.read(45, k=k, v=v)
    assert np.array_equal(k.cpu().numpy(), r.read(45)[0]) and np.array_equal(v.cpu().numpy(), r.read(45)[1])
    k.fill_(7.0)
    assert bool((out == 7.0).all())                      # nothing but the rows was written
    qs, qn = rows(rng, (S, 5, 2 * H, D + 1))
    got = torch.full((S, 5, 2 * H, D + 1), 7.0, device="cuda")
    c.attend(qs[..., 1:], out=got[..., 1:])
    near(got[..., 1:], r, qn[..., 1:], "f32")
    assert bool((got[..., 0] == 7.0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_read_rounds_once(dtype):
    b = Both(2, 2, 64, 100, 32, seed=6)
    b.append(77)
    for g, w in zip(b.c.read(80, dtype=TYPES[dtype]), b.r.read(80)):
        assert torch.equal(g.cpu(), torch.from_numpy(w).to(TYPES[dtype]))


def near(got, ref, q, dtype, counts=None, scale=None):
    """Attention results against 64 bits. The bound, in units of the largest |v| of the head (EPS = 2^-24, D columns,
    n keys, tiles of 64): a query's fixed-point elements are off by half a step, EPS (2^-16 for 16-bit types) of its
    largest, which moves a score by at most scale * D * max|q| * max|k| of those, and the score's own three roundings
    by 3 EPS of its size; twice that is what the probabilities move by. exp2 and its argument: 4 EPS and |score| EPS.
    A tile's probabilities are off by half a step of its largest product each, 64 in all; the sums over tiles round
    twice a tile. Then one rounding to dtype, half a step: 2^-24, 2^-8, 2^-11 of the value."""
    D = q.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    want = ref.attend(q, counts, scale)
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    step = 1.01 * EPS if dtype == "f32" else 1.01 * 2.0 ** -16
    got = got.double().cpu().numpy()
    group = q.shape[2] // ref.heads
    for s in range(q.shape[0]):
        for h in range(q.shape[2]):
            k, v = ref.k[s][h // group].values().astype(float), ref.v[s][h // group].values().astype(float)
            if not len(k):
                assert not got[s, :, h].any()
                continue
            kmax, vmax = np.abs(k).max(), np.abs(v).max()
            for i in range(q.shape[1]):
                qmax = np.abs(q[s, i, h]).max()
                size = scale * D * qmax * kmax
                move = 2 * (size * step + 4 * size * EPS) + (64 * step + 4 * (len(k) / 64 + 16) * EPS)
                w, g = want[s, i, h], got[s, i, h]
                tol = vmax * move + half * np.abs(w) + 2.0 ** -40
                assert np.all(np.abs(g - w) <= tol), (s, h, i, np.max(np.abs(g - w) - tol), np.max(np.abs(g - w)), vmax * move)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("block,kv,group,dim", [(32, 2, 1, 64), (16, 1, 4, 128), (64, 2, 3, 20), (16, 1, 17, 64), (32, 3, 1, 5)])
@pytest.mark.parametrize("lengths", [[1, 2, 16], [15, 17, 0], [63, 64, 65], [128, 130, 300]])
def test_attention(dtype, block, kv, group, dim, lengths):
    b = Both(3, kv, dim, 320, block, dtype, seed=sum(lengths) + dim)
    b.append(max(lengths), counts=lengths)
    for n_q, counts in ((1, None), (5, [5, 0, 2]), (33, None)):
        q, qn = rows(b.rng, (3, n_q, kv * group, dim), dtype, 2.0)
        near(b.c.attend(q, counts=ints(counts)), b.r, qn, dtype, counts)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n_seq,heads,n_q", [(40, 16, 33), (300, 8, 3)])
def test_attention_of_many_columns(dtype, n_seq, heads, n_q):
    # as many blocks of 16 columns as fill the device without a split of the keys
    b = Both(n_seq, heads, 64, 70, 32, dtype, seed=3)
    lens = b.rng.integers(0, 70, n_seq)
    b.append(70, counts=lens)
    counts = b.rng.integers(0, n_q + 1, n_seq)
    q, qn = rows(b.rng, (n_seq, n_q, heads, 64), dtype)
    near(b.c.attend(q, counts=ints(counts)), b.r, qn, dtype, counts)


def test_attention_over_a_long_cache():
    b = Both(1, 1, 64, 9000, 64, seed=12)
    b.append(8800)
    for n_q in (1, 20):
        q, qn = rows(b.rng, (1, n_q, 2, 64))
        near(b.c.attend(q), b.r, qn, "f32")


def test_scales_that_differ_between_blocks():
    # values of later blocks 1e-4 of the first one's, which is masked out by its scores: full precision of the small ones
    b = Both(1, 1, 64, 64, 16, seed=13)
    (k, kn), (v, vn) = (rows(b.rng, (1, 48, 1, 64)) for _ in range(2))
    q = torch.ones(1, 1, 1, 64, device="cuda")
    k[0, :16] = -8.0
    kn[0, :16] = -8.0
    v[0, 16:] *= 1e-4
    vn = v.double().cpu().numpy()
    b.put(k, v, kn, vn)
    got, want = b.c.attend(q).double().cpu().numpy(), b.r.attend(np.ones((1, 1, 1, 64)))
    # (as in near(): scores up to 64 * max|k|, but the largest value that counts is 1e-4 of the block's)
    assert np.all(np.abs(got - want) <= 5e-4 * (2 * 5 * 64 * 4 * 2 / 8 * EPS + 200 * EPS))


def test_large_scores():
    b = Both(1, 2, 64, 300, 32, seed=14)
    b.append(290, size=4.0)
    for scale in (None, 3.0, 0.0, -0.2):
        q, qn = rows(b.rng, (1, 3, 2, 64), size=10.0)
        got = b.c.attend(q, scale=scale)
        assert bool(torch.isfinite(got).all())
        near_scale = 64 ** -0.5 if scale is None else abs(scale)
        want = b.r.attend(qn, None, 64 ** -0.5 if scale is None else scale)
        size = near_scale * 64 * np.abs(qn).max() * 20.0
        assert np.max(np.abs(got.double().cpu().numpy() - want)) <= 20.0 * (2 * 5 * size * EPS + 200 * EPS)


def test_tiny_queries_over_large_keys():
    b = Both(1, 1, 64, 100, 32, seed=23)
    (k, kn), (v, vn) = (rows(b.rng, (1, 90, 1, 64)) for _ in range(2))
    k *= 1e32
    b.put(k, v, k.double().cpu().numpy(), vn)
    q, _ = rows(b.rng, (1, 7, 1, 64))
    for n in (1, 7):
        x = q[:, :n] * 1e-32
        near(b.c.attend(x), b.r, x.double().cpu().numpy(), "f32")


def test_what_is_not_finite_stays_where_it_is():
    b = Both(1, 1, 64, 200, 16, seed=15)
    (k, kn), (v, vn) = (rows(b.rng, (1, 100, 1, 64)) for _ in range(2))
    for x, n in ((k, kn), (v, vn)):
        x[0, 90, 0, 5] = n[0, 90, 0, 5] = np.nan if x is k else np.inf
    b.put(k, v, kn, vn)
    q, qn = rows(b.rng, (1, 60, 1, 64))
    q[0, 3, 0, 1] = qn[0, 3, 0, 1] = np.nan
    q[0, 4, 0, 1] = qn[0, 4, 0, 1] = np.inf
    got = b.c.attend(q).double().cpu().numpy()[0, :, 0]
    seen = np.arange(40, 100) // 16 >= 5          # the block of token 90 begins at 80
    seen[[3, 4]] = True
    assert np.isnan(got[seen]).all() and np.isfinite(got[~seen]).all()
    keep = np.flatnonzero(~seen)
    r = Cache(1, 1, 64, 200, 16)
    r.append(kn[:, :80], vn[:, :80])              # the full blocks that they see, to the last of them
    last = r.k[0][0].values().astype(float), r.v[0][0].values().astype(float)
    assert list(keep) == [i for i in range(40) if i not in (3, 4)]
    for i in keep:
        k, v = (x[:41 + i] for x in last)
        p = np.exp(k @ qn[0, i, 0] / 8 - (k @ qn[0, i, 0] / 8).max())
        # (near()'s bound: scores up to 64 * 4.5 * 4.5 / 8 of size, values up to 4.5)
        assert np.max(np.abs(got[i] - p @ v / p.sum())) <= 4.5 * (2 * 5 * 162 + 150) * EPS


def test_queries_before_the_first_token_and_padding():
    b = Both(3, 2, 64, 100, 32, seed=16)
    b.append(4, counts=[4, 0, 2])
    q, qn = rows(b.rng, (3, 6, 4, 64))
    q[1] = float("nan")
    got = b.c.attend(q, counts=ints([6, 6, 1]))
    assert not got[0, :2].any() and not got[1].any() and not got[2, 1:].any()
    assert got[0, 2:].any(-1).all() and got[2, 0].any()
    near(got, b.r, np.nan_to_num(qn), "f32", [6, 6, 1])


def test_offsets_past_32_bits():
    # 2.5 GB of keys: the last head's codes lie behind byte 2^31
    S, H, D, cap = 3, 64, 128, 100000
    c = QuantisedCache(S, H, D, cap, block=64)
    r = Cache(S, 1, D, cap, 64)
    rng = np.random.default_rng(17)
    (k, kn), (v, vn) = (rows(rng, (S, 70, 1, D)) for _ in range(2))
    c.append(k.expand(S, 70, H, D), v.expand(S, 70, H, D))
    r.append(kn, vn)
    got = c.read(70)
    for g, w in zip(got, r.read(70)):
        assert np.array_equal(g[:, :, -1:].cpu().numpy(), w) and torch.equal(g[:, :, 0], g[:, :, -1])
    q, qn = rows(rng, (S, 2, 1, D))
    out = c.attend(q.expand(S, 2, H, D).contiguous())
    near(out[:, :, -1:], r, qn, "f32")
    c.close()


def test_graph_replays_and_other_streams():
    def feed():
        rng = np.random.default_rng(18)
        return [rows(rng, (2, 1, n, 64))[0] for n in (3, 3, 6)]

    eager, graphed = (QuantisedCache(2, 3, 64, 200, block=16) for _ in range(2))
    k, v, q = feed()
    for c in (eager, graphed):
        c.append(k.expand(2, 30, 3, 64), v.expand(2, 30, 3, 64))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):       # (a warm-up before a capture)
        graphed.append(k, v)
        graphed.attend(q)
    torch.cuda.current_stream().wait_stream(side)
    eager.append(k, v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        graphed.append(k, v)
        out = graphed.attend(q)
        back = graphed.read(100)
    for step in range(40):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, device="cuda"))
        g.replay()
        eager.append(k, v)
        want = eager.attend(q)
        assert torch.equal(out, want), step
        if step % 8 == 0:
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(back, eager.read(100))), step
    assert graphed.lengths() == eager.lengths() == [71, 71]


def test_the_last_token_of_the_capacity():
    b = Both(2, 1, 64, 65, 32, seed=19)
    b.append(64)
    b.append(1, counts=[1, 1])
    b.append(1)                      # both refused
    q, qn = rows(b.rng, (2, 65, 1, 64))
    near(b.c.attend(q), b.r, qn, "f32")


def test_two_runs_are_equal():
    b = Both(1, 4, 64, 4000, 32, seed=20)
    b.append(3900)
    q, _ = rows(b.rng, (1, 1, 4, 64))
    first = b.c.attend(q)
    for _ in range(5):
        assert torch.equal(b.c.attend(q), first)


def test_refusals():
    c = QuantisedCache(2, 2, 64, 100)
    x = torch.zeros(2, 3, 2, 64, device="cuda")
    for what, call in (("k must be", lambda: c.append(x[:1], x)), ("v must be", lambda: c.append(x, x[..., :32])),
                       ("v must be", lambda: c.append(x, x[:, :2])),
                       ("v must be torch.float32", lambda: c.append(x, x.half())),
                       ("f32, bf16 or f16", lambda: c.append(x.double(), x.double())),
                       ("is on cpu", lambda: c.append(x.cpu(), x.cpu())),
                       ("contiguous", lambda: c.append(torch.zeros(2, 3, 2, 128, device="cuda")[..., ::2], x)),
                       ("exceed the cache's capacity", lambda: c.append(*[torch.zeros(2, 101, 2, 64, device="cuda")] * 2)),
                       ("counts must be", lambda: c.append(x, x, counts=torch.zeros(2, device="cuda"))),
                       ("counts is on cpu", lambda: c.append(x, x, counts=torch.zeros(2, dtype=torch.int32))),
                       ("start must be", lambda: c.append(x, x, start=torch.zeros(3, dtype=torch.int32, device="cuda"))),
                       ("not a multiple", lambda: c.attend(torch.zeros(2, 3, 3, 64, device="cuda"))),
                       ("1025 query heads", lambda: c.attend(torch.zeros(2, 1, 2050, 64, device="cuda"))),
                       ("exceed 4000000 rows", lambda: c.attend(torch.zeros(2, 1, 2, 64, device="cuda").expand(2, 4000001, 2, 64), out=torch.zeros(2, 1, 2, 64, device="cuda").expand(2, 4000001, 2, 64))),
                       ("out must be torch.float32", lambda: c.attend(x, out=x.half())),
                       ("out must be", lambda: c.attend(x, out=torch.zeros(2, 3, 4, 64, device="cuda"))),
                       ("scale must be finite", lambda: c.attend(x, scale=float("nan"))),
                       ("must not be negative", lambda: c.read(-1)),
                       ("dtype must be", lambda: c.read(1, dtype=torch.int8))):
        with pytest.raises(Gpt2Error, match=what):
            call()
    assert c.lengths() == [0, 0]
    assert c.attend(x[:, :0]).shape == (2, 0, 2, 64) and c.read(0)[0].shape == (2, 0, 2, 64)
    c.append(x[:, :0], x[:, :0])
    assert c.lengths() == [0, 0]
    c.close()
    with pytest.raises(Gpt2Error, match="closed"):
        c.lengths()


def test_gradients_are_refused():
    c = QuantisedCache(1, 2, 64, 100)
    x = torch.zeros(1, 3, 2, 64, device="cuda")
    leaf = x.clone().requires_grad_()
    for call in (lambda: c.append(leaf, x), lambda: c.append(x, leaf), lambda: c.attend(leaf)):
        with pytest.raises(Gpt2Error, match="requires a gradient"):
            call()
    with torch.no_grad():
        c.append(leaf, leaf)
        c.attend(leaf)
    assert c.lengths() == [3]


def test_a_cache_that_does_not_fit_leaves_no_error_behind():
    with pytest.raises(Gpt2Error, match="rtg_qcache_new"):
        QuantisedCache(1000, 1000, 128, 4000000)
    assert (torch.ones(5, device="cuda") + 1).sum().item() == 10


def test_lengths_refuses_a_stream_in_capture():
    c = QuantisedCache(1, 2, 64, 100)
    x = torch.ones(1, 3, 2, 64, device="cuda")
    c.append(x, x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(Gpt2Error, match="being captured"):
            c.lengths()
        c.append(x, x)
    g.replay()
    assert c.lengths() == [6]


def test_two_graphs_of_one_cache_take_turns():
    """A step and a check of several tokens (splits of both kinds), each its own graph, share the cache's workspace."""
    rng = np.random.default_rng(23)
    c, eager = (QuantisedCache(1, 4, 64, 3000) for _ in range(2))
    k, v, q, q9 = (rows(rng, (1, n, 4, 64))[0] for n in (1, 1, 1, 9))
    start = rows(rng, (1, 2500, 4, 64))[0]
    for x in (c, eager):
        x.append(start, start)
    c.attend(q), c.attend(q9)
    step, nine = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(step):
        c.append(k, v)
        out = c.attend(q)
    with torch.cuda.graph(nine):
        out9 = c.attend(q9)
    for i in range(12):
        for x in (k, v, q, q9):
            x.copy_(torch.randn(x.shape, device="cuda"))
        step.replay()
        nine.replay()
        eager.append(k, v)
        assert torch.equal(out, eager.attend(q)) and torch.equal(out9, eager.attend(q9)), i


def test_two_caches_on_two_streams_at_once():
    rng = np.random.default_rng(24)
    x, q = rows(rng, (2, 5000, 4, 64))[0], rows(rng, (2, 1, 4, 64))[0]
    caches = [QuantisedCache(2, 4, 64, 5000) for _ in range(2)]
    for c, y in zip(caches, (x, x.flip(1).contiguous())):
        c.append(y, y)
    want = [c.attend(q) for c in caches]
    streams = [torch.cuda.Stream() for _ in caches]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(caches[i].attend(q))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize("dim,group,block,length", [
    (64, 1, 32, 2560), (64, 1, 32, 2561), (64, 3, 16, 2600), (128, 1, 64, 1025), (128, 2, 16, 1100),
    (64, 7, 32, 1792), (64, 7, 32, 1793), (128, 8, 64, 768), (128, 16, 32, 769), (128, 16, 64, 14000),
    (64, 16, 64, 52000), (128, 40, 16, 2000)])
def test_splits(dim, group, block, length):
    """Lengths from which the keys are split, and splits of more tiles than the fewest."""
    b = Both(1, 1, dim, length + 20, block, "f16", seed=length)
    k, kn = rows(b.rng, (1, length, 1, dim), "f16")
    b.c.append(k, k)
    b.r.append(kn, kn)
    q, qn = rows(b.rng, (1, 1, group, dim), "f16", 2.0)
    near(b.c.attend(q), b.r, qn, "f16")


@pytest.mark.parametrize("dim,group,block,dtype", [(64, 20, 16, "f32"), (128, 20, 64, "bf16"), (40, 22, 32, "f16")])
def test_many_columns_of_several_pairs_of_tiles(dim, group, block, dtype):
    b = Both(2, 4, dim, 330, block, dtype, seed=dim)
    b.append(321, counts=[190, 321])
    q, qn = rows(b.rng, (2, 150, 4 * group, dim), dtype, 2.0)
    near(b.c.attend(q, counts=ints([150, 141])), b.r, qn, dtype, [150, 141])


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "f16"), (20, "bf16")])
def test_long_reads_of_sequences_of_different_lengths(dim, dtype):
    b = Both(5, 2, dim, 1700, 32, dtype, seed=dim)
    k, kn = rows(b.rng, (5, 1700, 2, dim), dtype)
    lens = [0, 1, 700, 1664, 1700]
    b.c.append(k, k, counts=ints(lens))
    b.r.append(kn, kn, lens)
    b.same(1700)
    b.same(1600, [0, 5, 690, -70, 200])


def test_results_of_other_orders_and_given_ones():
    rng = np.random.default_rng(25)
    c = QuantisedCache(2, 3, 64, 200)
    k, q = rows(rng, (2, 150, 3, 64))[0], rows(rng, (2, 20, 6, 64))[0]
    c.append(k, k)
    want = c.attend(q)
    swapped = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(c.attend(swapped), want) and c.attend(swapped).is_contiguous()
    assert torch.equal(c.attend(q[:, :1].expand(2, 20, 6, 64))[:, :1], c.attend(q[:, :1].repeat(1, 20, 1, 1))[:, :1])
    out = torch.empty(2, 6, 20, 64, device="cuda").transpose(1, 2)
    assert c.attend(q, out=out) is out and torch.equal(out, want)
    both = c.read(170)
    mine = torch.full((2, 3, 170, 64), 7.0, device="cuda").transpose(1, 2)
    for got in (c.read(170, k=mine), c.read(170, v=mine)):
        assert all(torch.equal(a, b) for a, b in zip(got, both))
