"""Attention over the 8-bit cache against 64 bits, element by element: results
are those of f32 sums or better and are rounded to their type once, whatever the
type of the rows and however the values' scales lie."""
import numpy as np
import pytest
import torch

from tests.test_gpu_qcache import EPS, Both, ints, rows

pytestmark = pytest.mark.gpu


def spacing(x, dtype):
    """Distance of neighbouring numbers of dtype around |x| (the larger one where x is next to a power of two)."""
    bits, least = {"f32": (23, -126), "bf16": (7, -126), "f16": (10, -14)}[dtype]
    e = np.frexp(np.abs(x) * (1 + 2.0 ** -bits))[1] - 1
    return 2.0 ** (np.maximum(e, least) - bits)


def check(b, got, q, dtype, counts=None, scale=None, every=1, seqs=None):
    """Each row of got against 64 bits, of the sequences `seqs` (all), every `every`-th query.

    A result is off by half a step of its type, and before that (EPS = 2^-24, p the probabilities, o the result, n the
    keys, all as 64 bits have them) by
      - the query as fixed point: half a step, 1.01 EPS of its largest component, for each of a key's components;
        8 EPS of the score's size for the roundings on its way to an exponent (the scale, log2 e and their product, the
        unit of the sums, its product with the key's scale, the sums to f32, the difference to the maximum and the
        maximum's own), 2 EPS for exp2; a change of the scores by e_j moves o by sum p_j |v_j - o| e_j at most;
      - the probabilities as fixed point: half a step, 1.01 EPS of the largest product p_j * (largest |v|
        of the block) of the (up to 128) keys taken together, for each of them;
      - f32 sums: 4 EPS of sum p_j |v_j| for every 64 keys, 16 times that for joins and the factors of a tile."""
    D, r = q.shape[-1], b.r
    scale = D ** -0.5 if scale is None else scale
    got = got.double().cpu().numpy()
    group = q.shape[2] // r.heads
    worst = 0.0
    for s in range(q.shape[0]) if seqs is None else seqs:
        c = q.shape[1] if counts is None else min(max(int(counts[s]), 0), q.shape[1])
        n = r.length(s)
        assert not got[s, c:].any() and not got[s, :max(c - n, 0)].any()
        for h in range(q.shape[2]):
            k, v = (x[s][h // group].values().astype(np.float64) for x in (r.k, r.v))
            if not n:
                continue
            top = np.repeat(r.v[s][h // group].s * 127, r.v[0][0].block)[:n]
            for i in sorted({*range(max(c - n, 0), c, every), max(c - 1, 0)} - set(range(max(c - n, 0)))):
                if i >= c:
                    continue
                see = n - c + i + 1
                sc = k[:see] @ q[s, i, h] * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                o = p @ v[:see]
                e = abs(scale) * 1.01 * EPS * np.abs(q[s, i, h]).max() * np.abs(k[:see]).sum(1) + 8 * EPS * np.abs(sc) + 2 * EPS
                off = (p * e) @ np.abs(v[:see] - o)
                prod = np.concatenate([p * top[:see], np.zeros(-see % 128)]).reshape(-1, 128)
                off = off + 1.01 * EPS * 128 * prod.max(1).sum() + 4 * EPS * (see / 64 + 16) * (p @ np.abs(v[:see]))
                over = np.abs(got[s, i, h] - o) - (spacing(o, dtype) / 2 + off)
                assert np.all(over <= 0), (s, h, i, over.max(), np.abs(off).max(), np.abs(o).max())
                worst = max(worst, (np.abs(got[s, i, h] - o) / (spacing(o, dtype) / 2 + off)).max())
    return worst


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [1.0, 300.0])
@pytest.mark.parametrize("dim,seqs,heads,group,n_q,length", [
    (64, 2, 2, 3, 4, 250), (128, 2, 1, 8, 1, 250),          # the keys split over waves
    (64, 10, 4, 4, 152, 280), (128, 10, 4, 4, 100, 260)])   # every wave all keys
def test_one_large_channel(dim, seqs, heads, group, n_q, length, size, dtype):
    """Queries with a channel of `size` times the rest keep the others' bits: five and more columns a head."""
    b = Both(seqs, heads, dim, length, 32, dtype, seed=dim + n_q)
    (k, kn), (v, vn) = (rows(b.rng, (seqs, length, heads, dim), dtype) for _ in range(2))
    k[..., 5] /= size
    b.c.append(k, v)
    b.r.append(k.double().cpu().numpy(), vn)
    q = rows(b.rng, (seqs, n_q, heads * group, dim), dtype, 2.0)[0]
    q[..., 5] *= size
    got = b.c.attend(q)
    print(f"    worst {check(b, got, q.double().cpu().numpy(), dtype, every=37, seqs=[0, seqs - 1]):.3f}", flush=True)


@pytest.mark.parametrize("dtype,big,small", [("f32", 1e20, 1.0), ("bf16", 1e20, 1.0), ("f32", 1e5, 1e-30), ("f32", 1e4, 1.0),
                                             ("bf16", 1e3, 1.0), ("f16", 1e3, 1e-4)])
@pytest.mark.parametrize("hidden", [False, True])
@pytest.mark.parametrize("dim,seqs,heads,group,block", [(64, 1, 1, 1, 16), (128, 1, 1, 2, 32), (64, 1, 2, 5, 32),
                                                        (64, 10, 4, 4, 16), (64, 10, 4, 4, 32), (128, 10, 4, 4, 16)])
def test_scales_far_apart(dim, seqs, heads, group, block, hidden, dtype, big, small):
    """Blocks of large and of small values side by side: rows that do not see the large ones yet and, `hidden`, rows whose
    scores keep them out, are as exact as if those were not there."""
    n = 152
    b = Both(seqs, heads, dim, n, block, dtype, seed=block + dim)
    (k, _), (v, _), (q, _) = (rows(b.rng, (seqs, n, h, dim), dtype) for h in (heads, heads, heads * group))
    large = (torch.arange(n, device="cuda") // block % 3 == 1)[:, None, None]
    v *= torch.where(large, big, small).to(v.dtype)
    if hidden:
        q[..., 0] = 8.0
        k[..., 0] = torch.where(large, -25.0 * dim ** 0.5, 0.0)[..., 0].to(k.dtype)
    b.c.append(k, v)
    b.r.append(k.double().cpu().numpy(), v.double().cpu().numpy())
    got = b.c.attend(q)
    every = 1 if seqs == 1 else 13
    print(f"    worst {check(b, got, q.double().cpu().numpy(), dtype, every=every, seqs=[seqs - 1]):.3f}", flush=True)


@pytest.mark.parametrize("dim,seqs,heads,group", [(64, 1, 1, 1), (128, 1, 1, 2), (64, 10, 4, 4), (128, 10, 4, 4)])
def test_blocks_of_zeros_that_take_the_probability(dim, seqs, heads, group):
    """Values of 0 at scores 60 above the rest: what the rest leaves in a result is as exact as ever."""
    n = 152
    b = Both(seqs, heads, dim, n, 16, seed=dim)
    (k, _), (v, _), (q, _) = (rows(b.rng, (seqs, n, h, dim)) for h in (heads, heads, heads * group))
    zero = (torch.arange(n, device="cuda") // 16 % 3 == 1)[:, None, None]
    v *= torch.where(zero, 0.0, 1.0)
    q[..., 0] = 8.0
    k[..., 0] = torch.where(zero, 7.5 * dim ** 0.5, 0.0)[..., 0]
    b.c.append(k, v)
    b.r.append(k.double().cpu().numpy(), v.double().cpu().numpy())
    check(b, b.c.attend(q), q.double().cpu().numpy(), "f32", every=1 if seqs == 1 else 13, seqs=[seqs - 1])


def test_padding_behind_a_prompt_takes_no_time():
    """Queries that are padding take none of the keys: one token each of long sequences, padded, against whole prompts."""
    n = 2000
    b = Both(16, 16, 64, n, 32, seed=7)
    k, q = (rows(b.rng, (16, n, 16, 64))[0] for _ in range(2))
    b.c.append(k, k)
    one = ints([1] * 16)
    out = torch.empty_like(q)

    def ms(counts):
        best = 1e9
        for _ in range(5):
            t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            t[0].record()
            b.c.attend(q, counts=counts, out=out)
            t[1].record()
            torch.cuda.synchronize()
            best = min(best, t[0].elapsed_time(t[1]))
        return best

    whole, padded = ms(None), ms(one)
    print(f"    whole {1e3 * whole:.0f} us, one token each {1e3 * padded:.0f} us", flush=True)
    assert padded < whole / 3


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16")])
def test_padded_prompts(dim, dtype):
    seqs, heads, group, n = 10, 4, 4, 200
    b = Both(seqs, heads, dim, n, 32, dtype, seed=dim)
    lens = [0, 1, 66, 200, 63, 64, 65, 128, 129, 199]
    (k, kn), (v, vn) = (rows(b.rng, (seqs, n, heads, dim), dtype) for _ in range(2))
    b.c.append(k, v, counts=ints(lens))
    b.r.append(kn, vn, lens)
    q, qn = rows(b.rng, (seqs, n, heads * group, dim), dtype)
    for counts in (lens, [0, 1, 66, 66, 0, 1, 0, 64, 200, 3]):
        check(b, b.c.attend(q, counts=ints(counts)), qn, dtype, counts, every=23)


@pytest.mark.parametrize("dim,n_q,group", [(64, 1, 1), (128, 1, 4), (64, 7, 2)])
@pytest.mark.parametrize("scale,q_size,k_size", [(3e36, 1e-36, 0.1), (2e38, 1e-20, 1e-19), (-1e37, 1e-33, 1e-4), (1e-37, 1e30, 1e7)])
def test_scales_of_the_scores_near_the_ends_of_f32(dim, n_q, group, scale, q_size, k_size):
    b = Both(2, 2, dim, 100, 32, seed=n_q)
    (k, _), (v, vn), (q, _) = (rows(b.rng, (2, n, h, dim)) for n, h in ((90, 2), (90, 2), (n_q, 2 * group)))
    k, q = k * k_size, q * q_size
    b.c.append(k, v)
    b.r.append(k.double().cpu().numpy(), vn)
    got = b.c.attend(q, scale=scale)
    check(b, got, q.double().cpu().numpy(), "f32", scale=float(np.float32(scale)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,block,seqs,heads,group,n_q", [
    (128, 16, 10, 4, 4, 100), (128, 32, 10, 4, 4, 100), (128, 64, 10, 4, 4, 100), (80, 32, 10, 4, 5, 80), (80, 16, 10, 8, 1, 170),
    (64, 64, 300, 8, 1, 5), (64, 16, 10, 4, 4, 160), (20, 32, 12, 10, 2, 100)])
def test_many_columns_of_every_form(dim, block, seqs, heads, group, n_q, dtype):
    """Enough blocks of 16 columns that every wave takes all keys of its own; lengths that end in a pair of tiles' first
    and second tile and in a block's middle, sequences and queries of different numbers."""
    blocks = seqs * heads * -(-n_q * group // 16)
    assert n_q * group > 4 and blocks >= (1400 if dim <= 64 else 800)
    n = 300
    b = Both(seqs, heads, dim, n, block, dtype, seed=dim + block)
    lens = b.rng.integers(0, n + 1, seqs)
    lens[:5] = [n, 128 + 64, 128 + 65, 40, 1]
    counts = np.minimum(b.rng.integers(0, n_q + 1, seqs), lens)
    counts[:3] = np.minimum(n_q, lens[:3])
    (k, kn), (v, vn) = (rows(b.rng, (seqs, n, heads, dim), dtype) for _ in range(2))
    b.c.append(k, v, counts=ints(lens))
    b.r.append(kn, vn, lens)
    q, qn = rows(b.rng, (seqs, n_q, heads * group, dim), dtype, 2.0)
    got = b.c.attend(q, counts=ints(counts))
    check(b, got, qn, dtype, counts, every=31, seqs=[0, 1, 2, 3, 4, 7, seqs - 1])
