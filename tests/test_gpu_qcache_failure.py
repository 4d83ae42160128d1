"""A pass over an 8-bit model cache that fails: the cache holds what it held and can be used again.
RTG_TEST_FORWARD_FAIL=1 makes forward_cached report a failure once a pass's kernels are on their way."""
import numpy as np
import pytest

from rusttorch_amd import synth
from rusttorch_amd.gpt2 import Gpt2Error
from tests.qcache_ref import Cache
from tests.test_gpu_qcache_model import ODD, SMALL, WIDE, Exact, model

pytestmark = pytest.mark.gpu


class Held(Cache):
    """A layer's cache that holds the codes that the GPU's holds, once they are known to be the same but for values
    that lie next to a border between two codes: their last bits decide, and one code of a value moves logits by more
    than all else (1.8e-3 for one value of two layers of 25 heads; 2e-6 with the same codes).

    Few do: the GPU's keys and values are off by some 1e-6 of a block's largest, 127 * 1e-6 of a code, so that one in
    some 4000 lies near enough. Behind a failed pass a code that fell the other way moves the next layer's dropped keys
    and values by some 1e-4, one of which may have set the scale that the last block left is read back with: 127 * 1e-4
    = 1.3 % of that block's values may then fall either way."""

    def take(self, read):
        for h in range(self.heads):
            for held, values in ((self.k[0][h], False), (self.v[0][h], True)):
                s = np.repeat(held.s, held.block)[:held.n, None]
                codes = np.rint(read(h, values).astype(float) / s)
                off = np.abs(codes - held.codes)
                few = 2 + off.size / 1000 + 0.02 * held.block * off.shape[1]
                assert off.max() <= 1 and off.sum() <= few, (h, values, off.max(), off.sum())
                held.codes = codes

    def append(self, k, v, counts=None, start=None):
        super().append(k, v, counts, start)
        if self.read_gpu:
            self.take(self.read_gpu)


class Reference(Exact):
    def __init__(self, sd, sh, block, cache, seq):
        super().__init__(sd, sh, block)
        self.kv = [Held(1, sh.n_head, sh.n_embd // sh.n_head, sh.n_positions, block) for _ in range(sh.n_layer)]
        self.cache, self.seq = cache, seq
        self.reading(True)

    def reading(self, on):
        for i, kv in enumerate(self.kv):
            kv.read_gpu = (lambda h, values, i=i: self.cache.read(i, h, self.seq, values)) if on else None

    def failed(self, ids):
        """A pass whose tokens are dropped again, its last block's tokens read back."""
        kept = self.past
        self.reading(False)
        self.forward(ids)
        self.past = kept
        for kv in self.kv:
            none = np.zeros((1, 0, kv.heads, kv.k[0][0].x.shape[1]))
            kv.append(none, none, start=[kept])
        self.reading(True)


@pytest.mark.parametrize("sh,storage,batch,block,kept,failed,then", [
    (SMALL, "f32", 1, 32, 45, (60,), (33, 1)), (SMALL, "bf16", 2, 16, 41, (40, 90), (1, 1, 50)),
    (SMALL, "f32", 3, 64, 70, (1, 70), (40, 1)), (WIDE, "bf16", 1, 32, 33, (35,), (1, 40)),
    (SMALL, "f32", 1, 32, 64, (50,), (40,)), (SMALL, "f32", 2, 32, 40, (50, 1), (1,)), (ODD, "f32", 1, 16, 30, (10, 2), (1, 9))])
def test_a_failed_pass_leaves_the_cache_usable(monkeypatch, sh, storage, batch, block, kept, failed, then):
    m, sd = model(sh, storage)
    print(f"[gpu] failed pass: batch {batch} block {block}, {kept} tokens kept, {failed} fail, {then}", flush=True)
    ids = np.stack([synth.make_tokens(kept + sum(then), sh.vocab_size, stream=40 + b) for b in range(batch)])
    other = np.stack([synth.make_tokens(sh.n_positions, sh.vocab_size, stream=70 + b) for b in range(batch)])
    c = m.new_cache(batch, bits=8, block=block)
    refs = {b: Reference(sd, sh, block, c, b) for b in {0, batch - 1}}

    def same(n, at):
        got = m.forward_cached_batched(ids[:, at:at + n], c)
        for b, r in refs.items():
            want = r.forward(ids[b, at:at + n])
            # (the framework's tolerance of logits)
            assert np.max(np.abs(got[b] - want) - (1e-3 + 1e-4 * np.abs(want))) <= 0, (b, at)
        assert c.len() == at + n

    same(kept, 0)
    before = c.read(1, sh.n_head - 1, batch - 1)
    for n in failed:
        monkeypatch.setenv("RTG_TEST_FORWARD_FAIL", "1")
        with pytest.raises(Gpt2Error, match="RTG_TEST_FORWARD_FAIL"):
            m.forward_cached_batched(other[:, :n], c)
        monkeypatch.delenv("RTG_TEST_FORWARD_FAIL")
        assert c.len() == kept
        full = kept // block * block
        assert np.array_equal(c.read(1, sh.n_head - 1, batch - 1)[:full], before[:full])
        for b, r in refs.items():
            r.failed(other[b, :n])
    at = kept
    for n in then:
        same(n, at)
        at += n
    c.clear()
    plain = m.new_cache(batch, bits=8, block=block)
    assert np.array_equal(*(m.forward_cached_batched(ids[:, :30], k) for k in (c, plain)))
    m.close()
