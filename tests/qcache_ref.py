"""The 8-bit key/value cache in numpy, written from its definition: what a
sequence's tokens are held as (values of 64 bits), and attention over them."""
import numpy as np

TINY = 127 * 2.0 ** -126


def token_scale(x):
    """f32 scale of a token's values x [..., D] (float64 holding f32 values)."""
    a = np.max(np.abs(x), axis=-1)
    with np.errstate(invalid="ignore"):
        s = (a / 127).astype(np.float32).astype(np.float64)
    s = np.where(a < TINY, 0.0, s)
    return np.where(np.isfinite(x).all(axis=-1), s, np.nan)


def quantise(x, s):
    """Codes of values x [n, D] under scale s (scalar)."""
    if not s > 0:
        return np.zeros_like(x)
    return np.rint(x / s)


class Head:
    """Keys (or values) of one head of one sequence."""

    def __init__(self, dim, block):
        self.block, self.n = block, 0
        self.x = np.zeros((0, dim))     # what the tokens are quantised from
        self.ts = np.zeros(0)           # their own scales
        self.codes = np.zeros((0, dim))
        self.s = np.zeros(0)            # per block

    def cut(self, at):
        b = max(at - 1, 0) // self.block     # the block of the last token left
        if 0 < at < self.n and b < (self.n - 1) // self.block:
            lo = b * self.block
            s = self.s[b]
            self.x[lo:at] = (self.codes[lo:at].astype(np.float32) * np.float32(s)).astype(np.float64)
            for t in range(lo, at):
                full = np.max(np.abs(self.codes[t])) == 127
                self.ts[t] = s if full or np.isnan(s) else token_scale(self.x[t])
        self.x, self.ts, self.codes, self.n = self.x[:at], self.ts[:at], self.codes[:at], at
        self.s = self.s[:-(-at // self.block)]
        self._blocks(b * self.block)

    def append(self, x):
        lo = self.n // self.block * self.block
        self.x = np.concatenate([self.x, x.astype(np.float64)])
        self.ts = np.concatenate([self.ts, token_scale(x.astype(np.float64))])
        self.n = len(self.x)
        self._blocks(lo)

    def _blocks(self, lo):
        self.codes = np.concatenate([self.codes[:lo], np.zeros((self.n - lo, self.x.shape[1]))])
        self.s = np.concatenate([self.s[:lo // self.block], np.zeros(-(-self.n // self.block) - lo // self.block)])
        for a in range(lo, self.n, self.block):
            e = min(a + self.block, self.n)
            ts = self.ts[a:e]
            s = np.nan if np.isnan(ts).any() else ts.max()
            self.s[a // self.block] = s
            self.codes[a:e] = quantise(self.x[a:e], s)

    def values(self):
        """[n, D] as read back in f32 (code times scale, rounded once)."""
        s = np.repeat(self.s, self.block)[:self.n, None]
        with np.errstate(invalid="ignore"):
            return (self.codes.astype(np.float32) * s.astype(np.float32)).astype(np.float32)


class Cache:
    def __init__(self, n_seq, n_head, dim, capacity, block):
        self.cap, self.heads = capacity, n_head
        self.k = [[Head(dim, block) for _ in range(n_head)] for _ in range(n_seq)]
        self.v = [[Head(dim, block) for _ in range(n_head)] for _ in range(n_seq)]

    def length(self, s):
        return self.k[s][0].n

    def append(self, k, v, counts=None, start=None):
        """k, v float arrays [n_seq, T, n_head, D]; returns the sequences refused."""
        refused = []
        for s in range(len(self.k)):
            n = k.shape[1] if counts is None else min(max(int(counts[s]), 0), k.shape[1])
            at = self.length(s) if start is None else int(start[s])
            if at < 0 or at > self.length(s) or at + n > self.cap:
                refused.append(s)
                continue
            for h in range(self.heads):
                for held, x in ((self.k[s][h], k), (self.v[s][h], v)):
                    if at < held.n:
                        held.cut(at)
                    if n:
                        held.append(x[s, :n, h])
        return refused

    def read(self, n, first=None):
        out = []
        for side in (self.k, self.v):
            x = np.zeros((len(side), n, self.heads, side[0][0].x.shape[1]), np.float32)
            for s, heads in enumerate(side):
                f = 0 if first is None else int(first[s])
                for h, held in enumerate(heads):
                    lo, hi = max(f, 0), min(f + n, held.n)
                    if lo < hi:
                        x[s, lo - f:hi - f, h] = held.values()[lo:hi]
            out.append(x)
        return out

    def attend(self, q, counts=None, scale=None):
        """q [n_seq, T, heads, D] -> (out, what bounds its error: see test_gpu_qcache), float64."""
        n_seq, T, H, D = q.shape
        scale = D ** -0.5 if scale is None else scale
        out, bound = np.zeros(q.shape), []
        group = H // self.heads
        q = q.astype(np.float64)
        for s in range(n_seq):
            c = T if counts is None else min(max(int(counts[s]), 0), T)
            n = self.length(s)
            for h in range(H):
                k, v = self.k[s][h // group].values().astype(np.float64), self.v[s][h // group].values().astype(np.float64)
                for i in range(c):
                    see = n - c + i + 1
                    if see <= 0:
                        continue
                    with np.errstate(invalid="ignore", over="ignore"):
                        sc = k[:see] @ q[s, i, h] * scale
                        p = np.exp(sc - sc.max())
                        out[s, i, h] = p @ v[:see] / p.sum()
        return out
