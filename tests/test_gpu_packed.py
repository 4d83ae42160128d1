"""Causal attention over packed prompts on the GPU, row by row against 64 bits."""
import numpy as np
import pytest
import torch

from rusttorch_amd._lib import Gpt2Error
from rusttorch_amd.attention import packed_attention
from tests.fourbit_ref import attention
from tests.test_gpu_fourbit import TYPES, ints, near, rows

pytestmark = pytest.mark.gpu


def prob_step(dtype):
    """What a probability is rounded by, relative: bf16's half step, f16's, three bf16 parts'."""
    return {"f32": 2.0 ** -24, "bf16": 2.0 ** -9, "f16": 2.0 ** -12}[dtype]


def want_of(q, k, v, offsets, scale, dtype):
    out, off = np.zeros(q.shape), np.zeros(q.shape)
    group = q.shape[1] // k.shape[1]
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        for h in range(q.shape[1]):
            out[lo:hi, h], off[lo:hi, h], *_ = attention(q[lo:hi, h], k[lo:hi, h // group], v[lo:hi, h // group],
                                                        np.arange(hi - lo) + 1, scale, prob_step(dtype),
                                                        # (f16: 2^6 times the probability, in steps of 2^-24 at least)
                                                        2.0 ** -31 if dtype == "f16" else 2.0 ** -125)
    return out, off


def check(lengths, heads, kv, dim, dtype="f32", before=0, behind=0, scale=None, seed=0, size=1.0):
    print(f"[gpu] packed {lengths}, {heads} heads over {kv} of {dim}, {dtype}, {before} rows before, {behind} behind", flush=True)
    rng = np.random.default_rng(seed)
    offsets = np.cumsum([before, *lengths])
    n = int(offsets[-1]) + behind
    (q, qn), (k, kn), (v, vn) = (rows(rng, (n, h, dim), dtype, size) for h in (heads, kv, kv))
    out = torch.full_like(q, 7.0)
    got = packed_attention(q, k, v, ints(offsets), scale=scale, out=out)
    assert got is out
    want, off = want_of(qn, kn, vn, offsets, dim ** -0.5 if scale is None else scale, dtype)
    near(got, want, off, dtype)
    assert torch.equal(got, packed_attention(q, k, v, ints(offsets), scale=scale))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 80, 24, 1, 33])
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2), (5, 1)])
def test_sequences_of_many_lengths(dim, dtype, heads, kv):
    check([1], heads, kv, dim, dtype, seed=1)
    check([1, 2, 31, 32, 33, 0, 63, 64, 65, 0, 127, 128, 129], heads, kv, dim, dtype, before=3, behind=2, seed=2)
    check([300], heads, kv, dim, dtype, behind=200, seed=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_long_ones(dtype):
    check([1500, 3, 700], 2, 1, 64, dtype, seed=4)
    check([1100], 3, 1, 128, dtype, seed=5)


def test_many_sequences():
    rng = np.random.default_rng(6)
    check(list(rng.integers(0, 5, 300)), 2, 2, 64, seed=7, behind=1)
    check(list(rng.integers(0, 40, 70)), 4, 1, 32, "bf16", seed=8, before=10, behind=500)
    check([0] * 100, 3, 3, 64, behind=9)
    check([0], 1, 1, 64, behind=1)


def test_groups_that_are_large():
    for heads in (16, 100, 128, 130, 260):
        check([9, 0, 70], heads, 1, 64, "bf16", seed=heads)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scales(dtype):
    for scale in (-0.2, 0.0, 1e-30, 3.0):
        check([150, 20], 2, 2, 64, dtype, scale=scale, seed=9)
    if dtype != "f16":
        check([150], 2, 1, 64, dtype, scale=1e-20, size=1e10, seed=10)
        check([150], 2, 1, 64, dtype, scale=1e28, size=1e-14, seed=11)
    else:
        check([150], 2, 1, 64, dtype, scale=1e-6, size=1e3, seed=10)
        check([150], 2, 1, 64, dtype, scale=1e6, size=1e-3, seed=11)


def test_many_small_probabilities_of_f16():
    """One key that stands out by 2^20 among many: what the others weigh together counts."""
    n = 3000
    q = torch.ones(n, 1, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(n, 1, 64, dtype=torch.float16, device="cuda")
    k[0] = 1.0
    v = torch.ones(n, 1, 64, dtype=torch.float16, device="cuda")
    v[0] = 0
    scale = 20 * np.log(2) / 64
    got = packed_attention(q, k, v, ints([0, n]), scale=scale).double().cpu().numpy()
    others = np.arange(n) * 2.0 ** -20
    want = np.broadcast_to((others / (1 + others))[:, None, None], got.shape)
    # (a probability of 2^-20 of the largest is 2^-14, 2^-20 or so of steps of 2^-24: off by 2^-5 at most)
    near(torch.from_numpy(got), want, want * 2.0 ** -5, "f16")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_finite_reaches_those_that_see_it(dim, dtype):
    n = 200
    offsets = [0, 150, 200]
    for bad in (float("nan"), float("inf"), -float("inf")):
        g = torch.Generator().manual_seed(1)
        q, k, v = (torch.randn(n, 2, dim, generator=g).to(TYPES[dtype]).cuda() for _ in range(3))
        plain = packed_attention(q, k, v, ints(offsets))
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        v2[40, 0, 5], v2[149, 1, 0], k2[90, 1, 3], q2[170, 0, 2] = bad, bad, bad, bad
        got = packed_attention(q2, k2, v2, ints(offsets))
        free = torch.ones_like(got, dtype=torch.bool)
        free[40:150, 0, 5] = free[149, 1, 0] = False
        free[90:150, 1] = free[170, 0] = False
        assert torch.equal(got[free], plain[free])
        assert not torch.isfinite(got[40:150, 0, 5]).any() and not torch.isfinite(got[149, 1, 0])
        assert torch.isnan(got[170, 0]).all()
        if bad != bad:
            assert torch.isnan(got[90:150, 1]).all()
        else:   # (a score of -infinity takes no part; one of infinity is all there is)
            assert (torch.isnan(got[90:150, 1]).all(-1) | torch.isfinite(got[90:150, 1, 1:]).all(-1)).all()
        # rows of no sequence, whatever they hold
        k2[:], v2[:], q2[:] = k, v, q
        for x in (q2, k2, v2):
            x[:40], x[120:] = bad, bad
        got = packed_attention(q2, k2, v2, ints([40, 60, 60, 120]))
        assert torch.isfinite(got).all() and (got[:40] == 0).all() and (got[120:] == 0).all()


def test_rows_in_any_strides():
    rng = np.random.default_rng(12)
    for dtype in ("f32", "bf16", "f16"):
        for dim in (64, 72):
            offsets = ints([0, 50, 130])
            qkv, _ = rows(rng, (130, 4 + 2 + 2, dim), dtype)       # as one projection leaves them
            odd, _ = rows(rng, (3, 130, 6, dim + 3), dtype)
            for q, k, v in ((qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]), (odd[0, :, :4, 1:dim + 1], odd[1, :, ::3, 3:], odd[2, :, 4:, :dim]),
                            (qkv.transpose(0, 1).contiguous().transpose(0, 1)[:, :4], qkv[:, :1].expand(130, 2, dim), qkv[:, 2:4])):
                want = packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), offsets)
                assert torch.equal(packed_attention(q, k, v, offsets), want)
                out = torch.full((130, 4, dim + 5), 7.0, dtype=q.dtype, device="cuda")
                packed_attention(q, k, v, offsets, out=out[..., 2:dim + 2])
                assert torch.equal(out[..., 2:dim + 2], want) and (out[..., :2] == 7).all() and (out[..., dim + 2:] == 7).all()


def test_offsets_out_of_range_are_clamped():
    g = torch.Generator().manual_seed(3)
    q = torch.randn(100, 2, 64, generator=g).cuda()
    want = packed_attention(q, q, q, ints([0, 30, 100]))
    assert torch.equal(packed_attention(q, q, q, ints([-7, 30, 2 ** 31 - 1])), want)
    want = packed_attention(q, q, q, ints([0, 100]))
    assert torch.equal(packed_attention(q, q, q, ints([-2 ** 31, 100, 3 * 10 ** 6])), want)


def test_offsets_that_descend():
    """One counts as the largest before it: its sequence has no row, and no row belongs to two."""
    g = torch.Generator().manual_seed(5)
    q = torch.randn(300, 2, 64, generator=g).cuda()
    for given, meant in (([0, 100, 50, 200], [0, 100, 100, 200]), ([120, 7, 7, 130], [120, 120, 120, 130]), ([300, 0, 0, 0], [300] * 4),
                         ([50, 300, 0, 300] * 40, [50] + [300] * 159), ([0, 10, -5, 20] + [3] * 100 + [40], [0, 10, 10, 20] + [20] * 100 + [40])):
        assert torch.equal(packed_attention(q, q, q, ints(given)), packed_attention(q, q, q, ints(meant))), given


def test_rows_past_32_bits():
    """8200 sequences of 64 rows, 32 heads of 128: the last ones' rows lie more than 2^31 elements in."""
    n, rng = 8200 * 64, torch.Generator(device="cuda").manual_seed(1)
    some = torch.randn(640, 32 + 2 * 8, 128, generator=rng, device="cuda").bfloat16()
    qkv = torch.zeros(n, 48, 128, dtype=torch.bfloat16, device="cuda")
    qkv[-640:] = some
    offsets = torch.arange(0, n + 64, 64, dtype=torch.int32, device="cuda")
    got = packed_attention(qkv[:, :32], qkv[:, 32:40], qkv[:, 40:], offsets)
    assert n * 48 * 128 > 2 ** 31 and torch.equal(got[-640:], packed_attention(some[:, :32], some[:, 32:40], some[:, 40:], offsets[:11]))
    assert (got[:-640] == 0).all()


def test_captured_and_replayed():
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(300, 4, 64, generator=g).cuda().bfloat16() for _ in range(3))
    offsets = ints([0, 100, 300])
    packed_attention(q, k, v, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = packed_attention(q, k, v, offsets)
    for lens in ([0, 100, 300], [0, 299, 299], [5, 17, 200], [0, 0, 0]):
        offsets.copy_(ints(lens))
        q.copy_(torch.randn(300, 4, 64, generator=g).bfloat16())
        graph.replay()
        want = packed_attention(q, k, v, offsets)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_on_another_stream():
    side = torch.cuda.Stream()
    x = torch.randn(200, 2, 64, device="cuda")
    want = packed_attention(x * 2, x, x, ints([0, 200]))
    offsets = ints([0, 200])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = packed_attention(x * 2, x, x, offsets)
    side.synchronize()
    assert torch.equal(got, want)


def test_prompts_then_tokens_over_the_cache():
    """As a program uses them: packed prompts, their keys and values into the cache, then attention over it: with
    values the cache holds exactly, the last positions' results are the prompt's."""
    from rusttorch_amd.q4cache import FourBitCache

    lengths, H, KV, D = [70, 1, 129], 4, 2, 64
    offsets = np.cumsum([0, *lengths])
    rng = np.random.default_rng(2)
    numbers = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    k, v = (torch.from_numpy(rng.choice(np.r_[numbers, -numbers], (200, KV, D))).float().cuda() for _ in range(2))
    k[:, :, ::32], v[:, :, ::32] = 6, -6   # (every group's largest is 6: the scale is 1)
    q, qn = rows(rng, (200, H, D))
    out = packed_attention(q, k, v, ints(offsets))
    c = FourBitCache(3, KV, D, 150)
    at = torch.from_numpy(np.minimum(offsets[:-1, None] + np.arange(129), 199)).cuda()
    c.append(k[at], v[at], counts=ints(lengths))
    assert torch.equal(c.read(129)[0][2], k[71:]) and torch.equal(c.read(129)[1][2], v[71:])
    for n in (1, 40):
        last = torch.from_numpy(np.clip(offsets[1:, None] - np.minimum(n, lengths)[:, None] + np.arange(n), 0, 199)).cuda()
        got = c.attend(q[last], counts=ints(np.minimum(n, lengths)))
        want, off = want_of(qn, k.double().cpu().numpy(), v.double().cpu().numpy(), offsets, D ** -0.5, "f32")
        for s in range(3):
            m = min(n, lengths[s])
            rows_s = slice(offsets[s + 1] - m, offsets[s + 1])
            near(got[s, :m], want[rows_s], off[rows_s], "f32")
            near(out[rows_s], want[rows_s], off[rows_s], "f32")


def test_refuses():
    x, o = torch.zeros(10, 2, 64, device="cuda"), ints([0, 10])
    for call, what in [
        (lambda: packed_attention(x, x[:9], x, o), "k must be"), (lambda: packed_attention(x, x, x[:, :1], o), "v must be"),
        (lambda: packed_attention(x, x[..., :32], x, o), "k must be"), (lambda: packed_attention(x, x, x.half(), o), "must be torch.float32"),
        (lambda: packed_attention(x, x, x.cpu(), o), "v is on"), (lambda: packed_attention(x, x, x, o.long()), "contiguous int32"),
        (lambda: packed_attention(x, x, x, o[:1]), "n \\+ 1"), (lambda: packed_attention(x, x, x, o.cpu()), "offsets is on"),
        (lambda: packed_attention(x, x, x, ints([0, 1, 2, 3])[::2]), "contiguous"),
        (lambda: packed_attention(x[:, :1].expand(10, 3, 64), x, x, o), "not a multiple"),
        (lambda: packed_attention(x, x, x, o, scale=float("inf")), "finite"), (lambda: packed_attention(x, x, x, o, out=x[:5]), "out must be"),
        (lambda: packed_attention(x.transpose(0, 2).contiguous().transpose(0, 2), x, x, o), "last dimension"),
        (lambda: packed_attention(x, x, x.clone().requires_grad_(), o), "requires a gradient"),
        (lambda: packed_attention(torch.zeros(4, 1, 129, device="cuda"), torch.zeros(4, 1, 129, device="cuda"),
                                  torch.zeros(4, 1, 129, device="cuda"), o), "head_dim 129"),
    ]:
        with pytest.raises(Gpt2Error, match=what):
            call()
    assert packed_attention(x[:0], x[:0], x[:0], ints([0, 0])).shape == (0, 2, 64)


def test_refuses_heads_of_no_channel():
    x = torch.zeros(4, 1, 0, device="cuda")
    with pytest.raises(Gpt2Error, match="head_dim 0"):
        packed_attention(x, x, x, ints([0, 4]))
