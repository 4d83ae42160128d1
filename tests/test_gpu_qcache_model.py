"""GPT-2 over an 8-bit cache (rtg_cache_new_quantised): what the first layer's
cache holds is what its f32 counterpart's values quantise to, bit for bit, and
the logits are those of a forward in 64 bits whose attention reads keys and
values rounded to 8 bits the same way."""
import numpy as np
import pytest

from rusttorch_amd import synth
from rusttorch_amd.gpt2 import Gpt2Config, Gpt2Error, Gpt2Model
from tests import ref64
from tests.qcache_ref import Cache, Head

pytestmark = pytest.mark.gpu

SMALL = synth.ModelShape(515, 160, 768, 2, 12)
WIDE = synth.ModelShape(515, 160, 1600, 2, 25)
TINY = synth.ModelShape(61, 70, 24, 2, 3)     # head_dim 8, no batched step
ODD = synth.ModelShape(61, 70, 160, 2, 4)     # head_dim 40


def model(sh, storage="f32"):
    cfg = Gpt2Config(sh.vocab_size, sh.n_positions, sh.n_embd, sh.n_layer, sh.n_head, sh.layer_norm_epsilon)
    sd = synth.make_weights(sh, bf16=storage == "bf16")
    return Gpt2Model.from_state_dict(sd, cfg, storage=storage), sd


class Exact:
    """The forward in 64 bits of one sequence over an 8-bit cache."""

    def __init__(self, sd, sh, block):
        self.g = {k: np.asarray(v, np.float64) for k, v in sd.items()}
        self.sh, self.past = sh, 0
        self.kv = [Cache(1, sh.n_head, sh.n_embd // sh.n_head, sh.n_positions, block) for _ in range(sh.n_layer)]

    def forward(self, ids):
        g, sh = self.g, self.sh
        T, d, H = len(ids), sh.n_embd, sh.n_head
        x = g["wte.weight"][ids] + g["wpe.weight"][self.past:self.past + T]
        for i in range(sh.n_layer):
            p = f"h.{i}."
            h = ref64.layer_norm(x, g[p + "ln_1.weight"], g[p + "ln_1.bias"], sh.layer_norm_epsilon)
            q, k, v = ((h @ g[p + "attn.c_attn.weight"] + g[p + "attn.c_attn.bias"])[:, j * d:(j + 1) * d]
                       .reshape(1, T, H, d // H) for j in range(3))
            self.kv[i].append(k.astype(np.float32), v.astype(np.float32))
            x = x + self.kv[i].attend(q)[0].reshape(T, d) @ g[p + "attn.c_proj.weight"] + g[p + "attn.c_proj.bias"]
            h = ref64.layer_norm(x, g[p + "ln_2.weight"], g[p + "ln_2.bias"], sh.layer_norm_epsilon)
            f = ref64.gelu_new(h @ g[p + "mlp.c_fc.weight"] + g[p + "mlp.c_fc.bias"])
            x = x + f @ g[p + "mlp.c_proj.weight"] + g[p + "mlp.c_proj.bias"]
        self.past += T
        return ref64.layer_norm(x, g["ln_f.weight"], g["ln_f.bias"], sh.layer_norm_epsilon) @ g["wte.weight"].T


@pytest.mark.parametrize("sh,storage,batch,block,chunks", [
    (SMALL, "f32", 1, 32, (45, 1, 1, 1, 1, 33)), (SMALL, "f32", 3, 16, (40, 1, 1, 1, 1, 2)),
    (SMALL, "bf16", 2, 64, (70, 1, 1)), (WIDE, "bf16", 1, 32, (33, 1, 1, 1)), (SMALL, "f32", 20, 32, (5, 1, 1)),
    (TINY, "f32", 2, 16, (30, 1, 1, 17)), (ODD, "f32", 1, 32, (40, 1, 3)), (SMALL, "f32", 40, 32, (2, 1))])
def test_logits_and_cache(sh, storage, batch, block, chunks):
    m, sd = model(sh, storage)
    print(f"[gpu] quantised cache {sh} {storage} batch {batch} block {block} chunks {chunks}", flush=True)
    total = sum(chunks)
    ids = np.stack([synth.make_tokens(total, sh.vocab_size, stream=90 + b) for b in range(batch)])
    c, f = m.new_cache(batch, bits=8, block=block), m.new_cache(batch)
    refs = {b: Exact(sd, sh, block) for b in {0, batch - 1}}
    at = 0
    for n in chunks:
        got = m.forward_cached_batched(ids[:, at:at + n], c)
        m.forward_cached_batched(ids[:, at:at + n], f, want_logits=False)
        for b, r in refs.items():
            want = r.forward(ids[b, at:at + n])
            # the framework's tolerance of logits; a key or value that falls on the other side of a border between
            # two codes for its last bits moves a score by up to |q| * amax / 127 / sqrt(hd), some 1e-3, of one key in many
            excess = np.max(np.abs(got[b] - want) - (1e-3 + 1e-4 * np.abs(want)))
            assert excess <= 0, (b, at, excess)
        at += n
        assert c.len() == f.len() == at
    hd = sh.n_embd // sh.n_head
    for b in refs:
        for head in {0, sh.n_head - 1}:
            for values in (False, True):
                got, raw = c.read(0, head, b, values), f.read(0, head, b, values)
                h = Head(hd, block)
                h.append(raw)
                # (an f32 cache's single tokens and f32 weights' prompts of up to 32 rows run other kernels, whose keys and
                # values differ in their last bits)
                step = np.repeat(h.s, block)[:at, None]
                off = np.abs(got - h.values())
                assert got.shape == (at, hd) and np.all(off <= step * 1.01)
                if batch > 1 and storage == "bf16":
                    assert not off.any()
    c.close()
    f.close()
    m.close()


@pytest.mark.parametrize("storage,batch,n", [("f32", 1, 50), ("f32", 4, 33), ("bf16", 2, 64)])
def test_generation_is_the_callers_own_loop(storage, batch, n):
    m, _ = model(SMALL, storage)
    prompts = np.stack([synth.make_tokens(n, SMALL.vocab_size, stream=60 + b) for b in range(batch)])
    for _ in range(2):      # (the second time in a pooled cache, replaying its graph)
        out, t = m.generate_cached_batched(prompts, 20, timing=True, bits=8, block=16)
        assert t["decode_steps"] == 19 and out.shape == (batch, n + 20)
        c = m.new_cache(batch, bits=8, block=16)
        logits, ids = m.forward_cached_batched(prompts, c)[:, -1], [prompts]
        for _ in range(20):
            top = np.sort(logits, -1)
            assert np.all(top[:, -1] - top[:, -2] > 1e-6)     # (no near tie for sums of another order to turn)
            ids.append(np.argmax(logits, -1)[:, None])
            logits = m.forward_cached_batched(ids[-1], c)[:, 0]
        assert np.array_equal(out, np.concatenate(ids, 1))
        c.close()
    plain = m.generate_cached_batched(prompts, 20)
    assert plain.shape == out.shape and np.array_equal(plain[:, :n], out[:, :n])
    m.close()


def test_a_cleared_cache_is_as_new():
    m, _ = model(SMALL)
    ids = synth.make_tokens(80, SMALL.vocab_size, stream=3)
    c, d = m.new_cache(bits=8), m.new_cache(bits=8)
    m.forward_cached(ids[:77], c)
    m.forward_cached(ids[:1], c)
    c.clear()
    assert c.is_empty() and c.read(0, 0).shape == (0, 64)
    for a, b in ((40, 41), (41, 42), (42, 80)):
        x, y = (m.forward_cached(ids[a:b] if a > 40 else ids[:41], k) for k in (c, d))
        assert np.array_equal(x, y)
    assert np.array_equal(c.read(1, 5, values=True), d.read(1, 5, values=True))


def test_refusals():
    m, _ = model(TINY)
    with pytest.raises(Gpt2Error, match="block 24 is not supported"):
        m.new_cache(bits=8, block=24)
    with pytest.raises(Gpt2Error, match="block 1 is not supported"):
        m.generate_cached_batched([[1, 2]], 3, bits=8, block=1)
    with pytest.raises(ValueError, match="bits must be"):
        m.new_cache(bits=4)
    with pytest.raises(ValueError, match="bits must be"):
        m.generate_cached_batched([[1, 2]], 3, bits=16)
    with pytest.raises(Gpt2Error, match="batch must be >= 1"):
        m.new_cache(0, bits=8)
    c = m.new_cache(bits=8)
    with pytest.raises(Gpt2Error, match="exceeds max position 70"):
        m.forward_cached(np.zeros(71, int), c)
    import ctypes as C
    from rusttorch_amd import _lib
    ids = np.zeros(2, np.uint32)
    with pytest.raises(Gpt2Error, match="does not take a quantised cache"):
        _lib.check(_lib.load().rtg_forward_cached_noalloc(m._h, c._h, ids.ctypes.data_as(C.c_void_p), 2, None))
    assert c.len() == 0


@pytest.mark.parametrize("sh,block,chunks", [
    (synth.ModelShape(61, 4200, 24, 2, 3), 32, (4094, 1, 1, 1, 1)),      # head_dim 8, the per-launch step
    (synth.ModelShape(61, 2800, 768, 1, 12), 64, (2623, 1, 1))])         # the batched step
def test_steps_over_a_context_whose_keys_are_split(sh, block, chunks):
    """The workgroup that writes the new token is not the one that reads the first keys, and joins what both have."""
    test_logits_and_cache(sh, "f32", 1, block, chunks)
