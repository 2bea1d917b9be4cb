"""A paged key/value cache, operator by operator, as cases that can be timed: new tokens'
keys and values written into pages (as they are, or in 8 bits), pages read back into rows,
and attention of a chunk of new tokens over the pages, from one token to a whole prompt.

The pages: `k`, `v` [pages, page_size, kv_heads, head_dim] in the stream type, or in e4m3
beside one power of two a token and head, `k_scale`, `v_scale` [pages, kv_heads, page_size]
e8m0. Token p of sequence b lies in slot p % page_size of page `table[b, p // page_size]`;
entries of `table` behind a sequence's last page mean nothing. A chunk is T tokens a row, of
which row b's first `lens[b]` are real; they stand at positions `start[b]` and on.

    write     a row of e4m3 has the scale 2^e, e the least with amax <= 448 * 2^e, and holds
              round(x / 2^e); a row with a NaN or an infinity reads back as NaN
    read      x = page value * scale, zeros behind a sequence's end
    attention o_i = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j over keys j <= start + i (and
              j >= start + i - window), query head h on KV head h // (heads / kv_heads);
              zeros for the chunk's rows from `lens[b]` on

`listed()` are the fixed cases, `draw` makes more of the same ranges, `prepare` makes what a
program holds before the call, `run` is one call, in plain torch operations or, where `own`
is true, through `svod_b200.ops`. `exact` computes the same in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # The keys and values of one decoding step of a busy server: latency alone counts.
        dict(name="write_step_bf16", op="write", dtype="bfloat16", quantized=False, batch=32, tokens=1, shortest=100,
             longest=4000, kv_heads=8, head_dim=128, page=16, ragged=False),
        # A batch of prompts of unequal length going into an 8-bit cache.
        dict(name="write_prompts_e4m3", op="write", dtype="bfloat16", quantized=True, batch=8, tokens=2048, shortest=0,
             longest=0, kv_heads=8, head_dim=128, page=64, ragged=True),
        # The next chunks of a few conversations, one head to a query head, small heads.
        dict(name="write_chunks_f16", op="write", dtype="float16", quantized=False, batch=5, tokens=333, shortest=17,
             longest=1900, kv_heads=12, head_dim=64, page=32, ragged=True),
        # A shared instruction's pages copied out into rows.
        dict(name="read_prefix_bf16", op="read", dtype="bfloat16", quantized=False, batch=1, shortest=413, longest=413,
             kv_heads=8, head_dim=128, page=16),
        # Long conversations read back from 8 bits, to move them to another layout or machine.
        dict(name="read_long_e4m3", op="read", dtype="bfloat16", quantized=True, batch=6, shortest=3000, longest=16384,
             kv_heads=8, head_dim=128, page=64),
        # One conversation's next token: the smallest call.
        dict(name="decode_one_bf16", op="attention", dtype="bfloat16", quantized=False, batch=1, tokens=1, shortest=776,
             longest=776, heads=16, kv_heads=8, head_dim=128, page=16, window=0, ragged=False),
        # A wide batch's next tokens over small pages.
        dict(name="decode_wide_bf16", op="attention", dtype="bfloat16", quantized=False, batch=64, tokens=1, shortest=64,
             longest=4095, heads=16, kv_heads=8, head_dim=128, page=16, window=0, ragged=False),
        # Long conversations' next tokens over an 8-bit cache.
        dict(name="decode_long_e4m3", op="attention", dtype="bfloat16", quantized=True, batch=16, tokens=1, shortest=8000,
             longest=32767, heads=16, kv_heads=8, head_dim=128, page=64, window=0, ragged=False),
        # Five drafted tokens a row to be checked, three query heads to a KV head.
        dict(name="draft_f16", op="attention", dtype="float16", quantized=False, batch=24, tokens=5, shortest=100,
             longest=2500, heads=12, kv_heads=4, head_dim=64, page=32, window=0, ragged=False),
        # Chunks of prompts of unequal length behind what the cache holds already.
        dict(name="chunks_bf16", op="attention", dtype="bfloat16", quantized=False, batch=6, tokens=512, shortest=0,
             longest=6000, heads=16, kv_heads=8, head_dim=128, page=16, window=0, ragged=True),
        # The next chunk of two long documents, windowed, over an 8-bit cache.
        dict(name="chunks_window_e4m3", op="attention", dtype="bfloat16", quantized=True, batch=2, tokens=1000,
             shortest=12000, longest=16000, heads=16, kv_heads=8, head_dim=128, page=64, window=4096, ragged=False),
        # Whole prompts at once, nothing held before: the largest case.
        dict(name="prompts_f16", op="attention", dtype="float16", quantized=False, batch=4, tokens=4096, shortest=0,
             longest=0, heads=16, kv_heads=8, head_dim=128, page=128, window=0, ragged=False),
    ]


def _spread(rng, low, high):
    """A whole number between `low` and `high`, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    case = dict(op=rng.choice(["write", "read", "attention", "attention"]), dtype=rng.choice(list(DTYPES)),
                quantized=rng.random() < 0.5, head_dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]))
    if case["op"] == "read":
        batch = _spread(rng, 1, 32)
        longest = _spread(rng, 50, min(16384, 60000 // batch))
        return case | dict(batch=batch, shortest=rng.randint(1, longest), longest=longest, kv_heads=rng.choice([4, 8, 12]))
    if case["op"] == "write":
        tokens = rng.choice([1, _spread(rng, 2, 2048)])
        batch = _spread(rng, 1, min(64, 12000 // tokens))
        longest = rng.choice([0, _spread(rng, 16, 4000)])
        return case | dict(batch=batch, tokens=tokens, shortest=rng.randint(0, longest), longest=longest,
                           kv_heads=rng.choice([4, 8, 12]), ragged=tokens > 1 and rng.random() < 0.5)
    kv_heads, group = rng.choice([(8, 2), (4, 3), (2, 8), (12, 1), (5, 4)])
    tokens = rng.choice([1, rng.randint(2, 9), _spread(rng, 10, 2048)])
    batch = _spread(rng, 1, max(1, min(48, 6000 // tokens)))
    longest = rng.choice([0, _spread(rng, 30, min(30000, 150000 // batch))])
    longest = max(longest, 1) if tokens == 1 else longest
    window = rng.choice([0, 0, _spread(rng, 64, 4096)])
    # the scores of the plain form, in 32 bits, stay within a few GB
    while batch * tokens * (tokens + longest) * kv_heads * group > 6e8:
        batch, longest = max(1, batch // 2), longest // 2
        tokens = tokens if batch > 1 else max(1, tokens // 2)
    return case | dict(batch=batch, tokens=tokens, shortest=rng.randint(0, longest), longest=longest, heads=kv_heads * group,
                       kv_heads=kv_heads, window=window, ragged=tokens > 1 and rng.random() < 0.5)


def _numbers(low, high, count):
    """`count` whole numbers spread evenly from `low` to `high`."""
    return [high] if count == 1 else [low + (high - low) * i // (count - 1) for i in range(count)]


def _lengths(case):
    """(tokens held before the call, new tokens) of each row, in an order of their own."""
    held = _numbers(case["shortest"], case["longest"], case["batch"])
    if case["op"] == "read":
        return held, [0] * case["batch"]
    new = _numbers(max(1, case["tokens"] // 4), case["tokens"], case["batch"]) if case["ragged"] else [case["tokens"]] * case["batch"]
    return held, new[::-1]


def work(case):
    held, new = _lengths(case)
    size = 2 * case["kv_heads"] * case["head_dim"]                     # values of a token's keys and values
    stored = size * (1 if case["quantized"] else 2) + (2 * case["kv_heads"] if case["quantized"] else 0)
    if case["op"] == "write":
        return {"bytes": sum(new) * (2 * size + stored), "flops": sum(new) * size * (3 if case["quantized"] else 0)}
    if case["op"] == "read":
        return {"bytes": sum(held) * stored + case["batch"] * case["longest"] * 2 * size,
                "flops": sum(held) * size if case["quantized"] else 0}
    seen = pairs = 0
    for h, n in zip(held, new):
        w = case["window"] or h + n
        first = max(0, h - w)
        seen += h + n - first
        # query i sees min(h + i, w) + 1 keys
        full = min(n, max(0, w - h))
        pairs += sum(range(h + 1, h + full + 1)) + (n - full) * (w + 1)
    rows = case["batch"] * case["tokens"] * case["heads"] * case["head_dim"]
    return {"bytes": seen * stored + 4 * rows, "flops": 4 * pairs * case["heads"] * case["head_dim"]}


def _quantise(x):
    """(e4m3 values, e8m0 scales) of rows `[..., D]`."""
    amax = x.float().abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)                             # amax = mantissa * 2^exponent, 0.5 <= mantissa < 1
    exponent = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)    # 448 = 0.875 * 2^9
    code = torch.where(amax > 0, (exponent + 127).clamp(0, 254), 127)
    code = torch.where(torch.isfinite(amax), code, 255)
    scaled = torch.ldexp(x.float(), (127 - code)[..., None].to(torch.int32))
    values = torch.where(code[..., None] == 255, 0.0, scaled).to(torch.float8_e4m3fn)
    return values, code.to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    batch, page, hk, d = case["batch"], case["page"], case["kv_heads"], case["head_dim"]
    held, new = _lengths(case)
    order = torch.randperm(batch, generator=gen, device="cuda").tolist()
    held, new = [held[i] for i in order], [new[i] for i in order]
    width = max(1, -(-(case["longest"] + case.get("tokens", 0)) // page))
    used = [-(-(h + n) // page) for h, n in zip(held, new)]
    pages = sum(used) + max(2, sum(used) // 8)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    # pages in the order in which a server's free list hands them out after some hours
    free = torch.randperm(pages, generator=gen, device="cuda")[:sum(used)].to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = free[at:at + n]
        at += n
    state = dict(case=case, table=table, start=torch.tensor(held, dtype=torch.int32, device="cuda"),
                 lens=torch.tensor(new, dtype=torch.int32, device="cuda") if case.get("ragged") else None,
                 k_scale=None, v_scale=None)
    # keys have a few loud channels, as projections do; every slot holds something, stale or not
    loud = torch.ones(d, device="cuda")
    loud[torch.randint(0, d, (max(1, d // 32),), generator=gen, device="cuda")] = 4.0
    for name, scale in (("k", loud), ("v", 1.0)):
        x = normal(pages, page, hk, d, scale=scale)
        if case["quantized"]:
            x, s = _quantise(x)
            state[name + "_scale"] = s.transpose(1, 2).contiguous()
        state[name] = x
        if case["op"] == "write":
            state["new_" + name] = normal(batch, case["tokens"], hk, d, scale=scale)
    if case["op"] == "attention":
        state["q"] = normal(batch, case["tokens"], case["heads"], d)
    return state


def run(state):
    case = state["case"]
    if own:
        from svod_b200 import ops
        cache = ops.PagedCache(state["k"], state["v"], state["k_scale"], state["v_scale"])
        if case["op"] == "write":
            ops.cache_write(state["new_k"], state["new_v"], cache, state["table"], state["start"], state["lens"])
            return _cache_of(state)
        if case["op"] == "read":
            return ops.cache_read(cache, state["table"], state["start"], case["longest"], DTYPES[case["dtype"]])
        window = (case["window"], 0) if case["window"] else None
        return ops.attention_paged(state["q"], cache, state["table"], state["start"], state["lens"],
                                   ops.Attn(causal=True, window=window))
    if case["op"] == "write":
        return _plain_write(state)
    if case["op"] == "read":
        k, v = _plain_read(state, case["longest"])
        here = torch.arange(case["longest"], device=k.device) < state["start"][:, None]
        dtype = DTYPES[case["dtype"]]
        return tuple(torch.where(here[..., None, None], x, 0.0).to(dtype) for x in (k, v))
    return _plain_attention(state)


def _cache_of(state):
    return {n: state[n] for n in ("k", "v", "k_scale", "v_scale") if state[n] is not None}


def _plain_write(state):
    table, start, lens, page = state["table"], state["start"], state["lens"], state["case"]["page"]
    batch, tokens = state["new_k"].shape[:2]
    i = torch.arange(tokens, device=table.device)
    real = i < (lens[:, None] if lens is not None else torch.full_like(start, tokens)[:, None])
    rows = torch.arange(batch, device=table.device)[:, None].expand(batch, tokens)[real]
    pos = (start[:, None] + i)[real].long()
    at, slot = table[rows, pos // page].long(), pos % page
    for name in ("k", "v"):
        x = state["new_" + name][real]
        if state["k_scale"] is None:
            state[name][at, slot] = x
        else:
            x, s = _quantise(x)
            state[name].view(torch.uint8)[at, slot] = x.view(torch.uint8)
            state[name + "_scale"].view(torch.uint8)[at, :, slot] = s.view(torch.uint8)
    return _cache_of(state)


def _plain_read(state, length):
    """(k, v) [B, length, kv_heads, D] f32 of what lies under the table, whatever it is."""
    case = state["case"]
    table = state["table"].clamp(min=0).long()
    got = []
    for name in ("k", "v"):
        x = state[name].view(torch.uint8)[table].view(state[name].dtype).float() if case["quantized"] else state[name][table].float()
        if case["quantized"]:
            x = x * state[name + "_scale"].view(torch.uint8)[table].view(torch.float8_e8m0fnu).float().transpose(2, 3)[..., None]
        got.append(x.flatten(1, 2)[:, :length])
    return got


def _plain_attention(state):
    case, q, start = state["case"], state["q"].float(), state["start"].long()
    batch, tokens, heads, d = q.shape
    hk = case["kv_heads"]
    lens = state["lens"].long() if state["lens"] is not None else torch.full_like(start, tokens)
    k, v = _plain_read(state, case["longest"] + tokens)
    i = torch.arange(tokens, device=q.device)
    j = torch.arange(k.shape[1], device=q.device)
    pos = start[:, None] + i
    seen = (j <= pos[..., None]) & (i < lens[:, None])[..., None]
    if case["window"]:
        seen = seen & (j >= pos[..., None] - case["window"])
    v = torch.where((j < (start + lens)[:, None])[..., None, None], v, 0.0)
    k = torch.where((j < (start + lens)[:, None])[..., None, None], k, 0.0)
    # [B, Hkv, group * T, D] . [B, Hkv, D, Tk]
    qg = q.view(batch, tokens, hk, heads // hk, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, d)
    s = torch.matmul(qg, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    s = s.view(batch, hk, heads // hk, tokens, -1).masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    del s
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, hk, -1, p.shape[-1]), v.permute(0, 2, 1, 3)).view(batch, hk, heads // hk, tokens, d)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, tokens, heads, d).to(DTYPES[case["dtype"]])


def exact(case, seed):
    """What `run` returns, token by token and in 64 bits."""
    state = prepare(case, seed)
    page, hk, d = case["page"], case["kv_heads"], case["head_dim"]
    table, start = state["table"].cpu(), state["start"].tolist()
    new = state["lens"].tolist() if state["lens"] is not None else [case.get("tokens", 0)] * case["batch"]

    def e4m3(x):
        """The nearest e4m3 value of each, in 64 bits: steps of 2^-9 up to 2^-6, of an eighth of the octave above."""
        octave = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
        step = torch.exp2(octave - 3)
        return torch.round(x / step) * step

    def rows(b, name, first, last):
        """Tokens [first, last) of sequence b, [n, Hkv, D] in 64 bits."""
        p = torch.arange(first, last, device="cuda")
        at = table[b].cuda()[p // page].long()
        if not case["quantized"]:
            return state[name][at, p % page].double()
        s = state[name + "_scale"].view(torch.uint8)[at, :, p % page].double()
        return state[name].view(torch.uint8)[at, p % page].view(torch.float8_e4m3fn).double() * torch.exp2(s - 127)[..., None]

    if case["op"] == "write":
        out = {n: x.double() for n, x in _cache_of(state).items()}
        for b in range(case["batch"]):
            p = torch.arange(start[b], start[b] + new[b], device="cuda")
            at = table[b].cuda()[p // page].long()
            for name in ("k", "v"):
                x = state["new_" + name][b, :new[b]].double()
                if case["quantized"]:
                    amax = x.abs().amax(-1)
                    e = torch.ceil(torch.log2(amax / 448.0))
                    e = e + (amax > 448.0 * torch.exp2(e)).double() - (amax <= 448.0 * torch.exp2(e - 1)).double()
                    out[name + "_scale"][at, :, p % page] = torch.exp2(e)
                    x = e4m3(x / torch.exp2(e)[..., None])
                out[name][at, p % page] = x
        return out
    if case["op"] == "read":
        got = [torch.zeros(case["batch"], case["longest"], hk, d, dtype=torch.float64, device="cuda") for _ in "kv"]
        for b in range(case["batch"]):
            for x, name in zip(got, "kv"):
                x[b, :start[b]] = rows(b, name, 0, start[b])
        return tuple(got)
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // hk
    for b in range(case["batch"]):
        n, h0 = new[b], start[b]
        first = max(0, h0 - case["window"]) if case["window"] else 0
        k, v = rows(b, "k", first, h0 + n), rows(b, "v", first, h0 + n)
        i = torch.arange(h0, h0 + n, device="cuda")[:, None]
        j = torch.arange(first, h0 + n, device="cuda")
        hidden = j > i
        if case["window"]:
            hidden |= j < i - case["window"]
        for h in range(case["heads"]):
            s = state["q"][b, :n, h].double() @ k[:, h // group].T / math.sqrt(d)
            out[b, :n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[:, h // group]
    return out
