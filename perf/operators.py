"""Performance cases of the 8-bit key/value cache: writing it, reading it back, attention over it.

The cache holds, for each sequence and key/value head, codes of 8 bits with one scale for each block of
`block` consecutive tokens, keys and values apart:

  s = f32(max |x| over the block's tokens so far / 127)        (0 where that maximum is below 127 * 2^-126)
  code = the nearest integer to x / s, ties to even;           it reads back as code * s

The block that is not full yet is quantised from its tokens' unrounded values.

A case:

  op       write    tokens appended to the sequences, then every value of the blocks that this touched read back
           read     every sequence read back whole
           attend   attention of the last `tokens` positions of each sequence over the cache
  seqs, heads, kv_heads, dim, block, dtype (of keys, values, queries, results)
  past     tokens in a sequence before the new ones (the longest sequence's)
  tokens   new tokens (write) or queries (attend) of a sequence
  ragged   sequences of different lengths and different numbers of new tokens, padded to `tokens`
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _case(name, op, seqs, heads, kv_heads, dim, block, dtype, past, tokens, ragged):
    return dict(name=name, op=op, seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim, block=block, dtype=dtype,
                past=past, tokens=tokens, ragged=ragged)


_LISTED = [
    # the prompts of eight requests to a 12-head model written at once
    _case("write_prompts_b8_p1000", "write", 8, 12, 12, 64, 32, "f32", 0, 1000, False),
    # one token for each of sixteen sequences of a 25-head model: the write of a decode step, lengths differ
    _case("write_step_b16", "write", 16, 25, 25, 64, 32, "f32", 900, 1, True),
    # the next pieces of prompts read piecewise, of different lengths, behind what is there; grouped heads
    _case("write_chunk_b4_bf16", "write", 4, 32, 8, 128, 64, "bf16", 3001, 517, True),
    # a session's cache read back for a check or a move: short
    _case("read_b1_p333", "read", 1, 12, 12, 64, 32, "f32", 333, 0, False),
    # long documents read back, for a cache in another form
    _case("read_b4_p20000_bf16", "read", 4, 32, 8, 128, 64, "bf16", 20000, 0, True),
    # the smallest call: the next token of an interactive session
    _case("attend_step_b1_p45", "attend", 1, 12, 12, 64, 32, "f32", 45, 1, False),
    # a decode step of sixteen requests to the widest model near the end of its context
    _case("attend_step_b16_p960", "attend", 16, 25, 25, 64, 32, "f32", 960, 1, True),
    # a decode step over long documents, grouped heads
    _case("attend_step_b8_p32000_bf16", "attend", 8, 32, 8, 128, 64, "bf16", 32000, 1, True),
    # one long document, a few sequences' worth of work only: the length has to be split
    _case("attend_step_b1_p50001_f16", "attend", 1, 16, 16, 64, 16, "f16", 50001, 1, False),
    # a few tokens at once behind a conversation (a short question, or drafted tokens to be judged)
    _case("attend_five_b6_p700", "attend", 6, 16, 16, 64, 16, "f32", 700, 5, True),
    # whole documents of a 20-head model in one batch
    _case("attend_prompts_b16_p1023", "attend", 16, 20, 20, 64, 32, "f32", 0, 1023, False),
    # the next piece of a long document, grouped heads
    _case("attend_chunk_b1_p12000_bf16", "attend", 1, 32, 8, 128, 64, "bf16", 12001, 2047, False),
]


def listed():
    return [dict(c) for c in _LISTED]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: [max(work(c)[k] for c in _LISTED if c["op"] == op) for k in ("bytes", "flops")]
            for op in ("write", "read", "attend")}
    while True:
        op = rng.choice(["write", "read", "attend", "attend"])
        heads, kv_heads, dim = rng.choice([(12, 12, 64), (16, 16, 64), (20, 20, 64), (25, 25, 64), (32, 8, 128),
                                           (16, 2, 128), (12, 4, 64), (8, 8, 80), (14, 2, 64), (6, 6, 32)])
        step = rng.random() < 0.5
        c = _case("", op, _log_int(rng, 1, 32), heads, kv_heads, dim, rng.choice([16, 32, 64]),
                  rng.choice(["f32", "f32", "bf16", "f16"]), _log_int(rng, 1, 40000),
                  0 if op == "read" else 1 if step else _log_int(rng, 2, 2000), rng.random() < 0.6)
        del c["name"]
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and _scores(c) <= 4e8:
            return c


def _scores(case):
    """Scores that the plain form of a case holds at once."""
    return case["seqs"] * case["heads"] * case["tokens"] * (case["past"] + case["tokens"])


# -- inputs --


def _lengths(case, seed):
    """Tokens of each sequence before the new ones, and new tokens (or queries) of each."""
    n, past, tokens = case["seqs"], case["past"], case["tokens"]
    g = torch.Generator().manual_seed(seed)
    if not case["ragged"]:
        return torch.full((n,), past), torch.full((n,), tokens)
    before = (past * (0.5 + 0.5 * torch.rand(n, generator=g))).round().long()
    new = (tokens * (0.3 + 0.7 * torch.rand(n, generator=g))).ceil().long()
    before[0], new[0] = past, tokens
    return before, new


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _inputs(case, seed):
    """Keys and values [seqs, past + tokens, kv_heads, dim] as they were written (a sequence's tokens first, padding
    behind), queries [seqs, tokens, heads, dim], lengths before and new tokens [seqs]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, (before, new) = _DTYPES[case["dtype"]], _lengths(case, seed)
    shape = (case["seqs"], case["past"] + case["tokens"], case["kv_heads"], case["dim"])
    # channels of a head differ in size, keys more than values, as projections of normed states do
    size_k = (1 + 2 * torch.rand(shape[2:], generator=g, device="cuda")).to(dtype)
    size_v = (0.5 + torch.rand(shape[2:], generator=g, device="cuda")).to(dtype)
    k, v = _normal(shape, g, dtype).mul_(size_k), _normal(shape, g, dtype).mul_(size_v)
    q = _normal((case["seqs"], case["tokens"], case["heads"], case["dim"]), g, dtype)
    return k, v, q, before.cuda(), new.cuda()


def _rows(x, first, n):
    """Rows first[s] .. first[s] + n of x [seqs, rows, ...] for each s; clamped to the last row."""
    at = (first[:, None] + torch.arange(n, device=x.device)).clamp_(max=x.shape[1] - 1)
    return x[torch.arange(x.shape[0], device=x.device)[:, None], at]


def prepare(case, seed):
    k, v, q, before, new = _inputs(case, seed)
    state = {"case": case, "counts": new.int() if case["ragged"] else None, "before": before, "new": new}
    block, length = case["block"], before + new
    if case["op"] == "write":
        # the new tokens, contiguous as a projection leaves them, and the unrounded start of the block they go on in
        state["start"] = before.int()
        state["first"] = (before // block * block).int()
        state["k"], state["v"] = _rows(k, before, case["tokens"]), _rows(v, before, case["tokens"])
        state["open_k"], state["open_v"] = _rows(k, before // block * block, block), _rows(v, before // block * block, block)
    if case["op"] == "attend":
        state["q"] = q
    if own:
        from rusttorch_amd.qcache import QuantisedCache

        cache = QuantisedCache(case["seqs"], case["kv_heads"], case["dim"], k.shape[1], block=block)
        cache.append(k, v, counts=(before if case["op"] == "write" else length).int())
        state["cache"] = cache
    elif case["op"] != "write":
        state["codes_k"], state["scale_k"] = _quantise(k, length, block)
        state["codes_v"], state["scale_v"] = _quantise(v, length, block)
    return state


# -- the plain form --


def _quantise(x, length, block):
    """Codes int8 [seqs, rows, heads, dim] and scales [seqs, blocks, heads] of the first length[s] rows of x, rows
    rounded up to whole blocks."""
    n, rows, heads, dim = x.shape
    blocks = -(-rows // block)
    inside = torch.arange(rows, device=x.device) < length[:, None]
    x = torch.where(inside[:, :, None, None], x.float(), torch.zeros((), device=x.device))
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, blocks * block - rows)).reshape(n, blocks, block, heads, dim)
    amax = x.abs().amax((2, 4))
    scale = torch.where(amax < 127 * 2.0 ** -126, 0.0, amax.double() / 127).float()
    # (64 bits: a quotient next to a border between two codes must fall on the right side of it)
    codes = x.double().div_(torch.where(scale == 0, 1.0, scale.double())[:, :, None, :, None]).round_()
    codes.mul_(scale[:, :, None, :, None] != 0)
    return codes.to(torch.int8).reshape(n, blocks * block, heads, dim), scale


def _dequantise(codes, scale, block):
    """f32 values of codes [seqs, rows, heads, dim]."""
    n, rows, heads, dim = codes.shape
    return (codes.reshape(n, rows // block, block, heads, dim).float() * scale[:, :, None, :, None]).reshape(codes.shape)


def _touched(case):
    """Rows that hold every block a write can touch."""
    return case["tokens"] + case["block"] - 1 if case["past"] else case["tokens"]


def _write_back(new, opened, before, count, case):
    """What the blocks touched by a write read back as: `opened` holds the open block's unrounded rows."""
    block, inside = case["block"], before % case["block"]
    rows = torch.arange(_touched(case), device=new.device)
    behind = rows - inside[:, None]
    seq = torch.arange(case["seqs"], device=new.device)[:, None]
    x = torch.where((behind >= 0)[:, :, None, None], new[seq, behind.clamp(0, case["tokens"] - 1)],
                    opened[seq, rows.clamp(max=block - 1).expand_as(behind)])
    codes, scale = _quantise(x, inside + count, block)
    return _dequantise(codes, scale, block)[:, :len(rows)].to(new.dtype)


def _attend(q, k, v, length, count, scale):
    """q [seqs, tokens, heads, dim] against k, v [seqs, rows, kv_heads, dim] in 32 bits."""
    n, tokens, heads, dim = q.shape
    rows, kv_heads = k.shape[1:3]
    group = heads // kv_heads
    # [seqs * kv_heads, group * tokens, dim]: the queries of one key/value head side by side
    qs = q.float().reshape(n, tokens, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n * kv_heads, group * tokens, dim)
    ks = k.permute(0, 2, 3, 1).reshape(n * kv_heads, dim, rows).contiguous()
    vs = v.permute(0, 2, 1, 3).reshape(n * kv_heads, rows, dim).contiguous()
    s = torch.matmul(qs * scale, ks).reshape(n, kv_heads, group, tokens, rows)
    at = (length - count)[:, None] + torch.arange(tokens, device=q.device)
    seen = (torch.arange(rows, device=q.device) <= at[:, :, None])[:, None, None]
    s = torch.where(seen, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-37)
    o = torch.matmul(p.reshape(n * kv_heads, group * tokens, rows), vs).reshape(n, kv_heads, group, tokens, dim)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, tokens, heads, dim)
    padding = torch.arange(tokens, device=q.device) >= count[:, None]
    return torch.where(padding[:, :, None, None], 0.0, o).to(q.dtype)


def run(state):
    case = state["case"]
    if own:
        cache = state["cache"]
        if case["op"] == "write":
            cache.append(state["k"], state["v"], counts=state["counts"], start=state["start"])
            k, v = cache.read(_touched(case), first=state["first"], dtype=state["k"].dtype)
            return {"k": k, "v": v}
        if case["op"] == "read":
            k, v = cache.read(case["past"], dtype=_DTYPES[case["dtype"]])
            return {"k": k, "v": v}
        return {"out": cache.attend(state["q"], counts=state["counts"])}
    if case["op"] == "write":
        return {"k": _write_back(state["k"], state["open_k"], state["before"], state["new"], case),
                "v": _write_back(state["v"], state["open_v"], state["before"], state["new"], case)}
    k = _dequantise(state["codes_k"], state["scale_k"], case["block"])
    v = _dequantise(state["codes_v"], state["scale_v"], case["block"])
    if case["op"] == "read":
        dtype = _DTYPES[case["dtype"]]
        return {"k": k[:, :case["past"]].to(dtype), "v": v[:, :case["past"]].to(dtype)}
    return {"out": _attend(state["q"], k, v, state["before"] + state["new"], state["new"], 1 / math.sqrt(case["dim"]))}


# -- what a pass cannot do without --


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    n, T, kv, D, block = case["seqs"], case["tokens"], case["kv_heads"], case["dim"], case["block"]
    share = 0.75 if case["ragged"] else 1.0  # the mean length over the longest
    held = 2 * D + 8 / block  # codes and scales of one token and head
    if case["op"] == "write":
        rows = n * kv * T * (0.65 if case["ragged"] and T > 1 else 1.0)
        # the new rows in, codes and scales out, the values read back
        return {"bytes": float(rows * (2 * D * es + held) + n * kv * _touched(case) * 2 * D * es),
                "flops": float(rows * 2 * D * 3)}
    if case["op"] == "read":
        rows = n * kv * case["past"]
        return {"bytes": float(rows * (share * held + 2 * D * es)), "flops": float(rows * share * 2 * D)}
    queries = n * T * (0.65 if case["ragged"] and T > 1 else 1.0)
    keys = case["past"] * share + (T + 1) / 2
    return {"bytes": float(n * kv * (case["past"] * share + T) * held + 2 * queries * case["heads"] * D * es),
            "flops": float(queries * case["heads"] * keys * 4 * D)}


# -- the same in 64 bits --


def exact(case, seed):
    k, v, q, before, new = _inputs(case, seed)
    block, heads, kv_heads, dim = case["block"], case["heads"], case["kv_heads"], case["dim"]
    before, new = before.tolist(), new.tolist()

    def held(x):
        """Values [rows, kv_heads, dim] that a sequence's rows x are held as."""
        parts = []
        for b in x.double().split(block):
            top = b.abs().amax((0, 2), keepdim=True)
            s = (top / 127).float().double()
            s = torch.where(top < 127 * 2.0 ** -126, torch.zeros_like(s), s)
            parts.append(torch.where(s > 0, torch.round(b / s.clamp_min(2.0 ** -149)) * s, torch.zeros_like(b)))
        return torch.cat(parts) if parts else x.double()

    outs = []
    for s in range(case["seqs"]):
        length = before[s] + new[s]
        if case["op"] == "write":
            first, rows = before[s] // block * block, _touched(case)
        else:
            first, rows = 0, case["past"]
        ks, vs = held(k[s, first:length]), held(v[s, first:length])
        if case["op"] != "attend":
            pad = (0, 0, 0, 0, 0, rows - (length - first))
            outs.append((torch.nn.functional.pad(ks, pad), torch.nn.functional.pad(vs, pad)))
            continue
        o = torch.zeros(case["tokens"], heads, dim, dtype=torch.float64, device="cuda")
        hidden = torch.arange(length, device="cuda") > torch.arange(before[s], length, device="cuda")[:, None]
        for h in range(heads):
            g = h // (heads // kv_heads)
            score = q[s, :new[s], h].double() @ ks[:, g].t().contiguous() / math.sqrt(dim)
            p = torch.softmax(score.masked_fill_(hidden, float("-inf")), -1)
            o[:new[s], h] = p @ vs[:, g].contiguous()
        outs.append(o)
    if case["op"] == "attend":
        return {"out": torch.stack(outs)}
    return {"k": torch.stack([o[0] for o in outs]), "v": torch.stack([o[1] for o in outs])}
