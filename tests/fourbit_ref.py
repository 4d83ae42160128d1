"""The 4-bit key/value cache in numpy, written from its definition (values of 64
bits), causal attention over rows, and how far f32 sums may be off."""
import numpy as np

NUMBERS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
U = 2.0 ** -24  # half a step of f32, relative


def held(x):
    """What x [..., dim] (float64 holding f32 values) is held as, 32 channels at a time."""
    out = np.zeros_like(x)
    for c in range(0, x.shape[-1], 32):
        part = x[..., c:c + 32]
        top = np.abs(part).max(-1, keepdims=True)
        fine = np.isfinite(top)
        mantissa, e = np.frexp(np.where(fine, top, 1.0))  # top = mantissa 2^e, mantissa in [0.5, 1)
        e = np.clip(e - 1 + (mantissa * 2 > 1.75) - 2, -100, 125)
        scale = np.exp2(e.astype(np.float64))
        a = np.abs(np.where(fine, part, 0.0)) / scale
        code = np.zeros(part.shape, int)
        for i in range(7):  # between numbers i and i + 1: to the even one
            border = (NUMBERS[i] + NUMBERS[i + 1]) / 2
            code += (a >= border) if i % 2 else (a > border)
        value = np.copysign(NUMBERS[code] * scale, part)
        out[..., c:c + 32] = np.where(fine, value, np.nan)
    return out


def attention(q, k, v, see, scale, prob=0.0, least=2.0 ** -125):
    """q [n, D], k, v [m, D], see [n] (keys of each) -> (out, what it may be off by before the results are rounded,
    probabilities [n, m], what each row's may be off by, relative). prob: the relative rounding of a probability; least: what may be lost of one that is tiny
    beside the largest (f32's numbers end at 2^-126, below which a probability and a part of one are 0).

    A score's error: D products (exact, or of f32 numbers) summed in f32, 2 D + 8 steps of rounding of the sum of
    their magnitudes at most, and the scale's own; a probability's: twice that of its score, as the largest score's
    enters too, and 2^-21 for the exponential. Then the sum over the keys, m + 8 steps of rounding in the products
    and as many in the sum of the probabilities."""
    n, m = len(q), len(k)
    out, off, probs, rel = np.zeros((n, v.shape[1])), np.zeros((n, v.shape[1])), np.zeros((n, m)), np.zeros(n)
    for i in range(n):
        s = max(int(see[i]), 0)
        if s == 0:
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            score = k[:s] @ q[i] * scale
            p = np.exp(score - score.max())
            p = p / p.sum()
            far = (np.abs(k[:s]) @ np.abs(q[i])).max() * abs(scale) * (2 * k.shape[1] + 8) * U
            out[i], probs[i, :s] = p @ v[:s], p
            rel[i] = 2 * far + 2.0 ** -21 + 2 * (s + 8) * U
            off[i] = p @ np.abs(v[:s]) * (rel[i] + 2 * prob) + np.abs(v[:s]).sum(0) * least
    return out, off, probs, rel


class Cache:
    def __init__(self, n_seq, n_head, dim, capacity):
        self.cap, self.dim = capacity, dim
        self.k = [[np.zeros((0, dim)) for _ in range(n_head)] for _ in range(n_seq)]
        self.v = [[np.zeros((0, dim)) for _ in range(n_head)] for _ in range(n_seq)]
        self.w = [[np.zeros(0) for _ in range(n_head)] for _ in range(n_seq)]
        self.w_off = [[np.zeros(0) for _ in range(n_head)] for _ in range(n_seq)]  # what they may be off by

    def length(self, s):
        return len(self.k[s][0])

    def append(self, k, v, counts=None, start=None):
        """k, v [n_seq, T, n_head, D]; returns the sequences refused."""
        refused = []
        for s in range(len(self.k)):
            n = k.shape[1] if counts is None else min(max(int(counts[s]), 0), k.shape[1])
            at = self.length(s) if start is None else int(start[s])
            if at < 0 or at > self.length(s) or at + n > self.cap:
                refused.append(s)
                continue
            for h in range(len(self.k[s])):
                for side, x in ((self.k, k), (self.v, v)):
                    side[s][h] = np.concatenate([side[s][h][:at], held(x[s, :n, h].astype(np.float64))])
                for side in (self.w, self.w_off):
                    side[s][h] = np.concatenate([side[s][h][:at], np.zeros(n)])
        return refused

    def read(self, n, first=None):
        out = []
        for side in (self.k, self.v):
            x = np.zeros((len(side), n, len(side[0]), self.dim))
            for s, heads in enumerate(side):
                f = 0 if first is None else int(first[s])
                for h, rows in enumerate(heads):
                    lo, hi = max(f, 0), min(f + n, len(rows))
                    if lo < hi:
                        x[s, lo - f:hi - f, h] = rows[lo:hi]
            out.append(x)
        return out

    def attend(self, q, counts=None, scale=None, prob=0.0, weigh=None):
        """q [n_seq, T, heads, D] -> (out, what it may be off by before it is rounded)."""
        n_seq, T, H, D = q.shape
        group = H // len(self.k[0])
        scale = D ** -0.5 if scale is None else scale
        out, off = np.zeros(q.shape), np.zeros(q.shape)
        for s in range(n_seq):
            c = T if counts is None else min(max(int(counts[s]), 0), T)
            see = self.length(s) - c + np.arange(c) + 1
            if weigh is not None:
                for w in self.w[s] + self.w_off[s]:
                    w *= weigh
            for h in range(H):
                k, v = self.k[s][h // group], self.v[s][h // group]
                out[s, :c, h], off[s, :c, h], p, rel = attention(q[s, :c, h].astype(np.float64), k, v, see, scale, prob)
                if weigh is not None and c:
                    self.w[s][h // group] += p.sum(0)
                    # (f32 sums of so many, and two steps more)
                    self.w_off[s][h // group] += rel @ p + (c * group + 4) * U * self.w[s][h // group]
        return out, off

    def evict(self, keep, recent):
        """Which tokens are kept [n_seq, n_head, keep], -1 where there is none."""
        kept = np.full((len(self.k), len(self.k[0]), keep), -1)
        for s in range(len(self.k)):
            for h in range(len(self.k[s])):
                n = len(self.k[s][h])
                which = np.arange(n)
                if n > keep:
                    old = n - recent
                    w = np.where(np.isnan(self.w[s][h][:old]), np.inf, self.w[s][h][:old])
                    nan = np.isnan(self.w[s][h][:old])
                    order = sorted(range(old), key=lambda t: (not nan[t], -w[t], t))[:keep - recent]
                    which = np.array(sorted(order) + list(range(old, n)))
                kept[s, h, :len(which)] = which
                for side in (self.k, self.v, self.w, self.w_off):
                    side[s][h] = side[s][h][which]
        return kept
