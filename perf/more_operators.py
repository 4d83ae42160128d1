"""Performance cases of attention over packed prompts, of the 4-bit key/value cache and of its eviction.

The cache holds, for each sequence, key/value head and token, keys and values apart, every 32 consecutive channels
as numbers of 4 bits (sign, two bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) times a power of two:

  2^e the largest power of two not above the 32 values' largest |x|, and one more where that is over 1.75 * 2^e
  scale = 2^(e - 2), at least 2^-100 and at most 2^125
  the nearest of the numbers to x / scale, ties to the even code, at most 6;      it reads back as number * scale

A case:

  op       prompt   causal attention of packed sequences, each over itself
           attend   attention of the last `tokens` positions of each sequence over the cache
           weigh    the same, and the weight that each key gets: its probabilities summed over queries and a head's group
           evict    sequences written anew with the weights their keys have got so far, cut to `keep` tokens (the last
                    `recent` and those of the largest weight, in their order), and what is left read back
  seqs, heads, kv_heads, dim, dtype (of keys, values, queries, results)
  past     tokens in a sequence before the last `tokens` (the longest sequence's)
  tokens   new tokens or queries of a sequence (the longest sequence's)
  keep, recent
  ragged   sequences of different lengths; padded to the longest's where they lie in a batch
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _case(name, op, seqs, heads, kv_heads, dim, dtype, past, tokens, ragged, keep=0, recent=0):
    return dict(name=name, op=op, seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, past=past,
                tokens=tokens, keep=keep, recent=recent, ragged=ragged)


_LISTED = [
    # a short question to a 12-head model, alone: the smallest call
    _case("prompt_b1_t30", "prompt", 1, 12, 12, 64, "f32", 0, 30, False),
    # a batch of documents of a 20-head model, packed
    _case("prompt_b16_t1023", "prompt", 16, 20, 20, 64, "f32", 0, 1023, True),
    # requests with their histories, grouped heads
    _case("prompt_b8_t1500_bf16", "prompt", 8, 32, 8, 128, "bf16", 0, 1500, True),
    # one long document
    _case("prompt_b1_t4001_f16", "prompt", 1, 16, 16, 64, "f16", 0, 4001, False),
    # the next token of an interactive session
    _case("attend_step_b1_p45", "attend", 1, 12, 12, 64, "f32", 45, 1, False),
    # a decode step of sixteen requests to the widest model near the end of its context
    _case("attend_step_b16_p960", "attend", 16, 25, 25, 64, "f32", 960, 1, True),
    # a decode step over long documents, grouped heads
    _case("attend_step_b8_p32000_bf16", "attend", 8, 32, 8, 128, "bf16", 32000, 1, True),
    # the next piece of a long document, grouped heads
    _case("attend_chunk_b1_p12000_bf16", "attend", 1, 32, 8, 128, "bf16", 12001, 2047, False),
    # a decode step that keeps count of which keys are looked at
    _case("weigh_step_b8_p16000_f16", "weigh", 8, 32, 8, 128, "f16", 16000, 1, True),
    # the last positions of four prompts judge their keys, before the cache is cut to a budget
    _case("weigh_window_b4_p5000", "weigh", 4, 12, 12, 64, "f32", 5000, 32, True),
    # one conversation cut to a small budget
    _case("evict_b1_p700", "evict", 1, 12, 12, 64, "f32", 700, 0, False, 256, 32),
    # long documents cut to a tenth, grouped heads
    _case("evict_b4_p20000_bf16", "evict", 4, 32, 8, 128, "bf16", 20000, 0, True, 2048, 64),
]


def listed():
    return [dict(c) for c in _LISTED]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: [max(work(c)[k] for c in _LISTED if c["op"] == op) for k in ("bytes", "flops")]
            for op in ("prompt", "attend", "weigh", "evict")}
    while True:
        op = rng.choice(["prompt", "prompt", "attend", "attend", "weigh", "evict"])
        heads, kv_heads, dim = rng.choice([(12, 12, 64), (16, 16, 64), (20, 20, 64), (25, 25, 64), (32, 8, 128),
                                           (16, 2, 128), (12, 4, 64), (8, 8, 80), (14, 2, 64), (6, 6, 32)])
        c = _case("", op, _log_int(rng, 1, 32), heads, kv_heads, dim, rng.choice(["f32", "f32", "bf16", "f16"]),
                  0 if op == "prompt" else _log_int(rng, 1, 40000), 1, rng.random() < 0.6)
        if op == "prompt":
            c["tokens"] = _log_int(rng, 2, 4500)
        elif op == "evict":
            c["tokens"], c["keep"] = 0, max(1, int(c["past"] * rng.uniform(0.05, 0.7)))
            c["recent"] = rng.randint(0, min(64, c["keep"]))
        elif rng.random() < 0.5:
            c["tokens"] = _log_int(rng, 2, 2000 if op == "attend" else 64)
        del c["name"]
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and _scores(c) <= 6e8:
            return c


def _scores(case):
    """Scores that the plain form of a case holds at once."""
    return case["seqs"] * case["heads"] * case["tokens"] * (case["past"] + case["tokens"])


# -- inputs --


def _lengths(case, seed):
    """Tokens of each sequence before the last ones, and those (or queries) of each."""
    n, past, tokens = case["seqs"], case["past"], case["tokens"]
    g = torch.Generator().manual_seed(seed)
    if not case["ragged"]:
        return torch.full((n,), past), torch.full((n,), tokens)
    if case["op"] == "prompt":
        # the same lengths in another order: as many rows for every seed
        spread = (tokens * (0.3 + 0.7 * torch.arange(1, n + 1) / n)).ceil().long()
        return torch.zeros_like(spread), spread[torch.randperm(n, generator=g)].clamp_(max=tokens)
    before = (past * (0.5 + 0.5 * torch.rand(n, generator=g))).round().long()
    new = (tokens * (0.3 + 0.7 * torch.rand(n, generator=g))).ceil().long()
    before[0], new[0] = past, tokens
    return before, new


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _inputs(case, seed):
    """Keys, values and queries, lengths before and new tokens [seqs], weights of the keys so far.

    prompt: rows [all tokens, heads, dim], one sequence behind the other; a few rows behind the last where ragged.
    Others: keys and values [seqs, past + tokens, kv_heads, dim], queries [seqs, tokens, heads, dim]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, (before, new) = _DTYPES[case["dtype"]], _lengths(case, seed)
    if case["op"] == "prompt":
        rows = int(new.sum()) + (5 if case["ragged"] else 0)
        lead = (rows,)
    else:
        lead = (case["seqs"], case["past"] + case["tokens"])
    shape = (*lead, case["kv_heads"], case["dim"])
    # channels of a head differ in size, keys more than values, as projections of normed states do
    size_k = (1 + 2 * torch.rand(shape[-2:], generator=g, device="cuda")).to(dtype)
    size_v = (0.5 + torch.rand(shape[-2:], generator=g, device="cuda")).to(dtype)
    k, v = _normal(shape, g, dtype).mul_(size_k), _normal(shape, g, dtype).mul_(size_v)
    n_q = lead if case["op"] == "prompt" else (case["seqs"], case["tokens"])
    q = _normal((*n_q, case["heads"], case["dim"]), g, dtype)
    w = None
    if case["op"] == "evict":
        # a few keys get most of the weight, many none at all
        w = torch.randn((case["seqs"], case["kv_heads"], case["past"]), generator=g, device="cuda")
        w = torch.where(w < -0.7, 0.0, torch.exp(3 * w))
    return k, v, q, before, new, w


def prepare(case, seed):
    k, v, q, before, new, w = _inputs(case, seed)
    op, length = case["op"], before + new
    state = {"case": case}
    if op == "prompt":
        state.update(q=q, k=k, v=v, offsets=torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).int().cuda())
        return state
    state["counts"] = new.int().cuda() if case["ragged"] else None
    state["before"], state["new"] = before.cuda(), new.cuda()
    if op == "evict":
        state.update(k=k, v=v, w=w, counts=before.int().cuda(), start=torch.zeros(case["seqs"], dtype=torch.int32, device="cuda"))
    else:
        state["q"] = q
    if own:
        from rusttorch_amd.q4cache import FourBitCache

        cache = FourBitCache(case["seqs"], case["kv_heads"], case["dim"], k.shape[1])
        if op != "evict":
            cache.append(k, v, counts=length.int().cuda())
        state["cache"] = cache
    elif op != "evict":
        state["codes_k"], state["exp_k"] = _quantise(k)
        state["codes_v"], state["exp_v"] = _quantise(v)
    return state


# -- the plain form --


def _quantise(x):
    """Twice the numbers (int8) [..., groups, 32] of x [..., dim], and the scales' exponents (int8) [..., groups]."""
    dim = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -dim % 32)).unflatten(-1, (-1, 32))
    top, e = torch.frexp(x.abs().amax(-1))
    e = (e - 3 + (top > 0.875)).clamp(-100, 125)
    y = torch.ldexp(x, -e[..., None])
    a = y.abs()
    # steps of a half below 2, of one below 4, of two behind
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp(-6, 6)
    return (2 * y).to(torch.int8), e.to(torch.int8)


def _dequantise(codes, e, dim):
    """f32 values [..., dim]."""
    return torch.ldexp(codes.float(), e[..., None].int() - 1).flatten(-2)[..., :dim]


def _attend(q, k, v, length, count, scale, weigh=False):
    """q [seqs, tokens, heads, dim] against k, v [seqs, rows, kv_heads, dim] in 32 bits: results, weights of the keys."""
    n, tokens, heads, dim = q.shape
    rows, kv_heads = k.shape[1:3]
    group = heads // kv_heads
    # [seqs * kv_heads, group * tokens, dim]: the queries of one key/value head side by side
    qs = q.float().reshape(n, tokens, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n * kv_heads, group * tokens, dim)
    ks = k.float().permute(0, 2, 3, 1).reshape(n * kv_heads, dim, rows).contiguous()
    vs = v.float().permute(0, 2, 1, 3).reshape(n * kv_heads, rows, dim).contiguous()
    s = torch.matmul(qs * scale, ks).reshape(n, kv_heads, group, tokens, rows)
    at = (length - count)[:, None] + torch.arange(tokens, device=q.device)
    inside = torch.arange(tokens, device=q.device) < count[:, None]
    seen = (torch.arange(rows, device=q.device) <= at[:, :, None])[:, None, None]
    s = torch.where(seen, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-37)
    o = torch.matmul(p.reshape(n * kv_heads, group * tokens, rows), vs).reshape(n, kv_heads, group, tokens, dim)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, tokens, heads, dim)
    w = torch.where(inside[:, None, None, :, None], p, 0.0).sum((2, 3)) if weigh else None
    return torch.where(inside[:, :, None, None], o, 0.0).to(q.dtype), w


def _prompt(state):
    case, offsets, rows = state["case"], state["offsets"].long(), len(state["q"])
    tokens = case["tokens"]
    count = offsets[1:] - offsets[:-1]
    # every sequence padded to the longest, and the results taken back to their rows
    at = (offsets[:-1, None] + torch.arange(tokens, device=offsets.device)).clamp_(max=rows - 1)
    o, _ = _attend(state["q"][at], state["k"][at], state["v"][at], count, count, 1 / math.sqrt(case["dim"]))
    row = torch.arange(rows, device=offsets.device)
    seq = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp_(max=case["seqs"] - 1)
    out = o[seq, (row - offsets[seq]).clamp_(max=tokens - 1)]
    return torch.where((row < offsets[-1])[:, None, None], out, 0.0).to(o.dtype)


def _evict(state):
    """Which tokens are kept [seqs, kv_heads, keep] (-1: none), and their values [seqs, keep, kv_heads, dim]."""
    case, length, w = state["case"], state["before"][:, None, None], state["w"]
    keep, recent, dim = case["keep"], case["recent"], case["dim"]
    at = torch.arange(case["past"], device=w.device)
    # the recent ones before all others, what is behind the sequence last; a stable sort takes ties by their index
    rank = torch.where(at >= length - recent, float("inf"), w)
    rank = torch.where(at < length, rank, float("-inf"))
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.where(kept < length, kept, case["past"]).sort(-1).values
    none = kept == case["past"]
    rows = kept.clamp(max=case["past"] - 1).transpose(1, 2)
    seq = torch.arange(case["seqs"], device=w.device)[:, None, None]
    head = torch.arange(case["kv_heads"], device=w.device)
    out = {"kept": torch.where(none, -1, kept).int()}
    for name in ("k", "v"):
        codes, e = _quantise(state[name])
        x = _dequantise(codes[seq, rows, head], e[seq, rows, head], dim)
        out[name] = torch.where(none.transpose(1, 2)[..., None], 0.0, x).to(state[name].dtype)
    return out


def run(state):
    case, dtype = state["case"], _DTYPES[state["case"]["dtype"]]
    if own:
        if case["op"] == "prompt":
            from rusttorch_amd.attention import packed_attention

            return {"out": packed_attention(state["q"], state["k"], state["v"], state["offsets"])}
        cache = state["cache"]
        if case["op"] == "attend":
            return {"out": cache.attend(state["q"], counts=state["counts"])}
        if case["op"] == "weigh":
            out = cache.attend(state["q"], counts=state["counts"], weigh=0.0)
            return {"out": out, "weights": cache.weights(case["past"] + case["tokens"])}
        cache.append(state["k"], state["v"], counts=state["counts"], start=state["start"])
        cache.add_weights(state["w"])
        kept = cache.evict(case["keep"], recent=case["recent"])
        k, v = cache.read(case["keep"], dtype=dtype)
        return {"kept": kept, "k": k, "v": v}
    if case["op"] == "prompt":
        return {"out": _prompt(state)}
    if case["op"] == "evict":
        return _evict(state)
    k = _dequantise(state["codes_k"], state["exp_k"], case["dim"])
    v = _dequantise(state["codes_v"], state["exp_v"], case["dim"])
    out, w = _attend(state["q"], k, v, state["before"] + state["new"], state["new"], 1 / math.sqrt(case["dim"]),
                     case["op"] == "weigh")
    return {"out": out} if w is None else {"out": out, "weights": w}


# -- what a pass cannot do without --


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    n, T, H, kv, D = case["seqs"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    share = 0.75 if case["ragged"] else 1.0  # the mean length over the longest
    held = D / 2 + (D + 31) // 32  # codes and scales of one token and head, keys or values
    if case["op"] == "prompt":
        mean, square = (0.65, 0.463) if case["ragged"] else (1.0, 1.0)  # of uniform lengths 0.3 to 1
        rows, pairs = n * T * mean, n * T * (T * square + mean) / 2
        return {"bytes": float(rows * D * es * 2 * (H + kv)), "flops": float(pairs * H * 4 * D)}
    if case["op"] == "evict":
        rows, left = n * kv * case["past"] * share, n * kv * case["keep"]
        # rows in, codes out, their weights; of the kept ones codes moved and values out
        return {"bytes": float(rows * (2 * D * es + 2 * held + 4) + left * (4 * held + 2 * D * es + 4)),
                "flops": float(rows * 2 * D * 3)}
    queries = n * T * (0.65 if case["ragged"] and T > 1 else 1.0)
    keys = case["past"] * share + (T + 1) / 2
    length = case["past"] * share + T
    weights = n * kv * length * 4 if case["op"] == "weigh" else 0
    return {"bytes": float(n * kv * length * 2 * held + 2 * queries * H * D * es + weights),
            "flops": float(queries * H * keys * 4 * D)}


# -- the same in 64 bits --


def _held(x):
    """What x [rows, kv_heads, dim] is held as, in 64 bits."""
    rows, heads, dim = x.shape
    y = torch.zeros(rows, heads, -(-dim // 32) * 32, dtype=torch.float64, device=x.device)
    y[..., :dim] = x.double()
    y = y.reshape(rows, heads, -1, 32)
    top = y.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(top.clamp_min(2.0 ** -140)))
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))  # (log2 may round)
    e = torch.where(top > 1.75 * torch.exp2(e), e + 1, e)
    scale = torch.exp2((e - 2).clamp(-100, 125))
    a, code = y.abs() / scale, torch.zeros_like(y, dtype=torch.int64)
    for i, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a >= border) if i % 2 else (a > border)
    number = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)[code]
    return (torch.where(y < 0, -number, number) * scale).reshape(rows, heads, -1)[..., :dim]


def exact(case, seed):
    k, v, q, before, new, w = _inputs(case, seed)
    op, heads, kv_heads, dim = case["op"], case["heads"], case["kv_heads"], case["dim"]
    before, new = before.tolist(), new.tolist()
    group, zeros = heads // kv_heads, lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")
    if op == "prompt":
        out, at = zeros(len(q), heads, dim), 0
    else:
        out = zeros(case["seqs"], case["tokens"], heads, dim)
    weights = zeros(case["seqs"], kv_heads, case["past"] + case["tokens"])
    kept = torch.full((case["seqs"], kv_heads, case["keep"]), -1, dtype=torch.int32, device="cuda")
    left = [zeros(case["seqs"], case["keep"], kv_heads, dim) for _ in range(2)]
    for s in range(case["seqs"]):
        n, length = new[s], before[s] + new[s]
        if op == "prompt":
            qs, ks, vs, to = q[at:at + n].double(), k[at:at + n].double(), v[at:at + n].double(), out[at:at + n]
            at += n
        else:
            qs, ks, vs, to = q[s, :n].double(), _held(k[s, :length]), _held(v[s, :length]), out[s]
        if op == "evict":
            old = max(0, length - case["recent"])
            some = max(0, min(length, case["keep"]) - (length - old))
            for h in range(kv_heads):
                order = torch.sort(w[s, h, :old].double(), dim=-1, descending=True, stable=True).indices[:some]
                which = torch.cat([order, torch.arange(length - min(length - old, case["keep"]), length, device="cuda")]).sort().values
                kept[s, h, :len(which)] = which.int()
                for to, x in zip(left, (ks, vs)):
                    to[s, :len(which), h] = x[which, h]
            continue
        hidden = torch.arange(length, device="cuda") > torch.arange(before[s], length, device="cuda")[:, None]
        for h in range(heads):
            score = qs[:, h] @ ks[:, h // group].t().contiguous() / math.sqrt(dim)
            p = torch.softmax(score.masked_fill_(hidden, float("-inf")), -1)
            to[:n, h] = p @ vs[:, h // group].contiguous()
            weights[s, h // group, :length] += p.sum(0)
    if op == "evict":
        return {"kept": kept, "k": left[0], "v": left[1]}
    return {"out": out, "weights": weights} if op == "weigh" else {"out": out}
