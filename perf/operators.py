"""Timed cases of the 4-bit key/value cache: the block tables of a serving step, writing keys and
values into the cache (and reading them back), and attention over it.

`run` computes an operator in its plain form (elementary torch operations, 32 bits), or, where the
module's `own` is true, through this package's calls."""

import math
import random

import torch

own = False

GROUP = 64  # channels that share a scale and a minimum
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    def tables(name, requests, prefills, kv_max, q, page, lens):
        return {"name": name, "op": "tables", "requests": requests, "prefills": prefills, "kv_max": kv_max, "q": q,
                "page": page, "spread": True, "lens": lens}

    def write(name, tokens, kv_heads, head_dim, page, dtype, fused):
        return {"name": name, "op": "write", "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
                "dtype": dtype, "fused": fused}

    def attend(name, requests, prefills, kv_max, q, heads, kv_heads, head_dim, page, dtype, window, spread, lens):
        return {"name": name, "op": "attend", "requests": requests, "prefills": prefills, "kv_max": kv_max, "q": q,
                "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype,
                "window": window, "spread": spread, "lens": lens}

    return [
        # One decode step of a small batch: a page table update that must cost no more than a launch.
        tables("tables_decode_8", 8, 0, 4096, 1, 16, 11),
        # A serving step of 1024 requests, 24 of them with a chunk of their prompt.
        tables("tables_mixed_1024", 1024, 24, 16384, 1024, 64, 12),
        # The keys and values of one decode step of 48 requests.
        write("write_decode_48", 48, 8, 128, 64, "bf16", True),
        # A prompt chunk of 8192 tokens, k and v as views of the fused q/k/v projection's output.
        write("write_prompt_8192", 8192, 8, 128, 64, "bf16", True),
        # An odd number of tokens and heads of a small f16 model.
        write("write_odd_f16", 5003, 5, 64, 16, "f16", False),
        # One user, short conversation: latency.
        attend("attend_one_517", 1, 0, 517, 1, 16, 2, 128, 16, "bf16", 0, False, 21),
        # Decode step of 64 requests of ragged lengths, 4 query heads a key head.
        attend("attend_decode_64", 64, 0, 16384, 1, 32, 8, 128, 64, "bf16", 0, True, 22),
        # One user with a long context.
        attend("attend_long_131072", 1, 0, 131071, 1, 64, 8, 128, 64, "bf16", 0, False, 23),
        # Multi-head attention (a key head for each query head), head dimension 64, f16.
        attend("attend_heads_f16", 24, 0, 4001, 1, 20, 20, 64, 32, "f16", 0, True, 24),
        # Four drafted tokens verified for each of 16 requests; head dimension 256.
        attend("attend_draft_256", 16, 16, 8192, 4, 16, 2, 256, 64, "bf16", 0, True, 25),
        # A prompt chunk over its own and 4096 earlier tokens.
        attend("attend_prompt_4096", 1, 1, 8192, 4096, 32, 8, 128, 64, "bf16", 0, False, 26),
        # A mixed step: 3 prompt chunks beside 29 decoding requests, sliding window.
        attend("attend_mixed_window", 32, 3, 6000, 777, 32, 4, 128, 16, "bf16", 2048, True, 27),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    page = rng.choice([16, 32, 64, 128])
    op = rng.choice(["tables", "write", "attend", "attend", "attend"])
    lens = rng.randrange(1 << 30)
    if op == "tables":
        requests = spread(1, 2048)
        prefills = rng.choice([0, rng.randrange(0, min(requests, 24) + 1)])
        return {"op": op, "requests": requests, "prefills": prefills, "kv_max": spread(64, 16384), "q": spread(2, 1024),
                "page": page, "spread": True, "lens": lens}
    head_dim = rng.choice([64, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "write":
        kv_heads = spread(1, 16)
        return {"op": op, "tokens": spread(1, 8192 * 8 * 128 // (kv_heads * head_dim)), "kv_heads": kv_heads,
                "head_dim": head_dim, "page": page, "dtype": dtype, "fused": rng.random() < 0.6}
    kv_heads = spread(1, 16)
    group = rng.choice([1, 2, 4, 5, 7, 8, 8, 16])
    window = rng.choice([0, 0, 0, spread(16, 4096)])
    kind = rng.choice(["decode", "decode", "draft", "prompt", "mixed"])
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype,
            "window": window, "spread": rng.random() < 0.7, "lens": lens}
    if kind in ("decode", "draft"):
        requests = spread(1, 128)
        room = 64 * 16384 * 8 * 128 // (requests * kv_heads * head_dim)
        case.update(requests=requests, kv_max=spread(8, max(16, min(131072, room // 2))))
        case.update(prefills=0, q=1) if kind == "decode" else case.update(prefills=requests, q=rng.randrange(2, 9))
        return case
    # rows * keys * heads * channels below half of attend_prompt_4096's
    room = 4096 * 8192 * 32 * 128 // (2 * kv_heads * group * head_dim)
    q = spread(16, 2048)
    kv_max = max(q, min(spread(64, 16384), room // q))
    if kind == "prompt":
        case.update(requests=1, prefills=1, kv_max=kv_max, q=q)
    else:
        case.update(requests=spread(2, 32), prefills=1, kv_max=min(kv_max, 8192), q=min(q, 1024, kv_max))
    return case


def _lens(case):
    """(key/value lengths with the step's tokens, the step's tokens) of each request."""
    r = random.Random(case["lens"])
    kv, new = [], []
    for b in range(case["requests"]):
        length = case["kv_max"]
        if case["spread"] and b > 0:
            length = int(round(math.exp(r.uniform(math.log(max(1.0, length / 16)), math.log(length)))))
        n = 1
        if b < case["prefills"]:
            n = case["q"]
            if case["spread"] and b > 0 and n >= 16:
                n = r.randint(n // 2, n)
        length = max(length, 1)
        kv.append(length)
        new.append(min(n, length))
    order = list(range(len(kv)))
    r.shuffle(order)
    return [kv[i] for i in order], [new[i] for i in order]


def _group_bytes(head_dim):
    """Bytes of one head's key (or value) of one token: 4 bits a channel, two f16 a group."""
    return head_dim // 2 + 4 * (head_dim // GROUP)


def work(case):
    if case["op"] == "tables":
        kv, new = _lens(case)
        p = case["page"]
        grown = sum(-(-a // p) - -(-(a - n) // p) for a, n in zip(kv, new))
        return {"bytes": 8 * len(kv) + 8 * len(kv) + 12 * sum(new) + 8 * grown, "flops": 0}
    if case["op"] == "write":
        n = case["tokens"] * case["kv_heads"]
        # k and v in, the cache written and read, k and v out
        return {"bytes": 2 * n * (2 * case["head_dim"] + 2 * _group_bytes(case["head_dim"]) + 2 * case["head_dim"]),
                "flops": 0}
    kv, new = _lens(case)
    w = case["window"]
    read = pairs = 0
    for length, n in zip(kv, new):
        for_row = (lambda p: min(p + 1, w)) if w else (lambda p: p + 1)
        first = length - n
        read += length - (max(0, first + 1 - w) if w else 0)
        pairs += sum(for_row(first + i) for i in range(n))
    d, h = case["head_dim"], case["heads"]
    return {"bytes": read * case["kv_heads"] * 2 * _group_bytes(d) + 4 * sum(new) * h * d, "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _keys_values(tokens, kv_heads, head_dim, dtype, g):
    """Keys with a few strong channels and an offset of each channel (as rotated projections have),
    values without."""
    f = dict(generator=g, device="cuda")
    gain = 1.0 + 3.0 * (torch.rand((kv_heads, head_dim), **f) < 0.05)
    shift = 0.5 * torch.randn((kv_heads, head_dim), **f)
    k = (torch.randn((tokens, kv_heads, head_dim), **f) * gain + shift).to(dtype)
    v = torch.randn((tokens, kv_heads, head_dim), **f).to(dtype)
    return k, v


def _pages(case, kv, g):
    """A pool's free pages in random order and each request's table filled from it."""
    p = case["page"]
    width = -(-max(kv) // p)
    counts = [-(-n // p) for n in kv]
    total = sum(counts)
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    return table, total


def _slots(table, kv, page):
    """The cache place of every position of every request, back to back."""
    out = []
    for b, n in enumerate(kv):
        pos = torch.arange(n, device="cuda")
        out.append(table[b].long()[pos // page] * page + pos % page)
    return torch.cat(out)


def prepare(case, seed):
    g = _generator(seed)
    if own:
        import sushi_b200 as sx
    if case["op"] == "tables":
        kv, new = _lens(case)
        p = case["page"]
        ctx = [a - n for a, n in zip(kv, new)]
        width = -(-max(kv) // p)
        have = [-(-c // p) for c in ctx]
        spare = sum(-(-a // p) for a in kv) - sum(have) + 64
        perm = torch.randperm(sum(have) + spare, generator=g, device="cuda").to(torch.int32)
        counts = torch.tensor(have, device="cuda")
        first = torch.cumsum(counts, 0) - counts
        col = torch.arange(width, device="cuda")
        held = col[None, :] < counts[:, None]
        at = (first[:, None] + col[None, :]).clamp(max=perm.numel() - 1)
        table = torch.where(held, perm[at], torch.full_like(perm[at], -1))
        i32 = dict(dtype=torch.int32, device="cuda")
        return {"case": case, "ctx": torch.tensor(ctx, **i32), "new": torch.tensor(new, **i32), "table": table,
                "free": perm[sum(have):].contiguous(), "count": torch.tensor([spare], **i32), "tokens": sum(new)}
    dt = _DT[case["dtype"]]
    if case["op"] == "write":
        t, h, d, p = case["tokens"], case["kv_heads"], case["head_dim"], case["page"]
        k, v = _keys_values(t, h, d, dt, g)
        if case["fused"]:  # views of a [tokens, (queries + keys + values)] projection output
            qkv = torch.cat([torch.zeros((t, 2 * h, d), dtype=dt, device="cuda"), k, v], 1)
            k, v = qkv[:, 2 * h:3 * h], qkv[:, 3 * h:]
        pages = -(-t // p) + 3
        perm = torch.randperm(pages, generator=g, device="cuda")
        pos = torch.arange(t, device="cuda")
        slots = perm[pos // p] * p + pos % p
        state = {"case": case, "k": k, "v": v, "slots": slots}
        if own:
            state["cache"] = sx.Kv4Cache(pages, h, d, p)
        else:
            state["held"] = _empty_plain(pages * p, h, d)
        return state
    kv, new = _lens(case)
    table, pages = _pages(case, kv, g)
    h, d, p = case["kv_heads"], case["head_dim"], case["page"]
    k, v = _keys_values(sum(kv), h, d, dt, g)
    slots = _slots(table, kv, p)
    q = torch.randn((sum(new), case["heads"], d), generator=g, device="cuda").to(dt)
    i32 = dict(dtype=torch.int32, device="cuda")
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    state = {"case": case, "q": q, "table": table, "kv": kv, "new": new, "kv_lens": torch.tensor(kv, **i32),
             "cu_q": torch.tensor(cu, **i32), "max_q": max(new), "scale": d ** -0.5}
    if own:
        state["cache"] = sx.Kv4Cache(pages, h, d, p)
        sx.kv4_write(state["cache"], k, v, slots)
    else:
        state["held"] = _empty_plain(pages * p, h, d)
        _plain_write(state["held"], k, v, slots)
    return state


# ------------------------------------------------------------------ the plain forms
def _empty_plain(places, kv_heads, head_dim):
    code = dict(dtype=torch.uint8, device="cuda")
    par = dict(dtype=torch.float16, device="cuda")
    g = head_dim // GROUP
    return [(torch.zeros((places, kv_heads, head_dim), **code), torch.zeros((places, kv_heads, g), **par),
             torch.zeros((places, kv_heads, g), **par)) for _ in range(2)]


def _plain_write(held, k, v, slots):
    for (codes, scale, low), x in zip(held, (k, v)):
        t, h, d = x.shape
        y = x.float().reshape(t, h, d // GROUP, GROUP)
        lo, hi = y.amin(-1), y.amax(-1)
        m = lo.half()
        s = ((hi - lo) * (1.0 / 15.0)).half()
        sf = s.float()[..., None]
        c = torch.round((y - m.float()[..., None]) / torch.where(sf > 0, sf, torch.ones_like(sf)))
        c = torch.where(sf > 0, c.clamp(0.0, 15.0), torch.zeros_like(c))
        codes[slots] = c.to(torch.uint8).reshape(t, h, d)
        scale[slots] = s
        low[slots] = m


def _plain_read(held, slots):
    out = []
    for codes, scale, low in held:
        c = codes[slots]
        t, h, d = c.shape
        c = c.float().reshape(t, h, d // GROUP, GROUP)
        out.append((c * scale[slots].float()[..., None] + low[slots].float()[..., None]).reshape(t, h, d))
    return out


def _plain_tables(st):
    p, ctx, new, table = st["case"]["page"], st["ctx"].long(), st["new"].long(), st["table"]
    width = table.shape[1]
    kv = ctx + new
    have = (ctx + p - 1) // p
    need = torch.clamp((kv + p - 1) // p, max=width)
    grow = torch.clamp(need - have, min=0)
    start = torch.cumsum(grow, 0) - grow
    col = torch.arange(width, device=table.device)[None, :]
    at = st["count"].long() - 1 - start[:, None] - (col - have[:, None])
    page = torch.where(at >= 0, st["free"][at.clamp(0, st["free"].numel() - 1)], torch.full_like(table, -1))
    table = torch.where((col >= have[:, None]) & (col < need[:, None]), page, table)
    ends = torch.cumsum(new, 0)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    i = torch.arange(st["tokens"], device=table.device)
    b = torch.searchsorted(ends, i, right=True)
    pos = ctx[b] + i - cu[b]
    page = table[b, (pos // p).clamp(max=width - 1)].long()
    slots = torch.where((page >= 0) & (pos // p < width), page * p + pos % p, torch.full_like(pos, -1))
    left = st["count"] - grow.sum().int()
    return [table, kv.int(), cu.int(), slots, pos.int(), left]


def _plain_attend(st):
    case, q = st["case"], st["q"]
    h, hk, d, p, w = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["window"]
    table, scale = st["table"], st["scale"]
    if max(st["new"]) == 1:  # every request has one row: one padded batch
        b, longest = len(st["kv"]), max(st["kv"])
        pos = torch.arange(longest, device=q.device)
        page = table[:, pos // p].long().clamp(min=0)
        k, v = (x.reshape(b, longest, hk, d).permute(0, 2, 1, 3)
                for x in _plain_read(st["held"], (page * p + pos % p).reshape(-1)))
        s = torch.matmul(q.float().reshape(b, hk, h // hk, d), k.transpose(-1, -2)) * scale
        n = st["kv_lens"].long()[:, None]
        seen = pos[None, :] < n
        if w:
            seen = seen & (pos[None, :] >= n - w)
        return _softmax_product(s, seen[:, None, None, :], v).reshape(b, h, d).to(q.dtype)
    out, at = [], 0
    for b, (length, n) in enumerate(zip(st["kv"], st["new"])):
        pos = torch.arange(length, device=q.device)
        k, v = (x.permute(1, 0, 2)[:, None] for x in _plain_read(st["held"], table[b].long()[pos // p] * p + pos % p))
        row = torch.arange(length - n, length, device=q.device)[:, None]
        seen = pos[None, :] <= row
        if w:
            seen = seen & (pos[None, :] > row - w)
        rows = q[at:at + n].float().permute(1, 0, 2).reshape(hk, h // hk, n, d)
        o = _softmax_product(torch.matmul(rows, k.transpose(-1, -2)) * scale, seen, v)
        out.append(o.reshape(h, n, d).permute(1, 0, 2))
        at += n
    return torch.cat(out).to(q.dtype)


def _softmax_product(s, seen, v):
    s = s.masked_fill(~seen, float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return torch.matmul(e, v) / e.sum(-1, keepdim=True)


def run(state):
    op = state["case"]["op"]
    if own:
        import sushi_b200 as sx

        if op == "tables":
            t = sx.block_tables(state["ctx"], state["new"], state["table"], state["free"], state["count"],
                                state["case"]["page"], state["tokens"])
            return [state["table"], t.kv_lens, t.cu_q, t.slots, t.positions, t.free_left]
        if op == "write":
            sx.kv4_write(state["cache"], state["k"], state["v"], state["slots"])
            return list(sx.kv4_read(state["cache"], state["slots"], state["k"].dtype))
        return sx.kv4_attention(state["q"], state["cache"], state["table"], state["kv_lens"], state["cu_q"],
                                state["max_q"], scale=state["scale"], window=state["case"]["window"])
    if op == "tables":
        return _plain_tables(state)
    if op == "write":
        _plain_write(state["held"], state["k"], state["v"], state["slots"])
        return [x.to(state["k"].dtype) for x in _plain_read(state["held"], state["slots"])]
    return _plain_attend(state)


# ------------------------------------------------------------------ the definition in 64 bits
def _held64(x):
    """What the cache holds for x [tokens, heads, channels], from the format's definition."""
    t, h, d = x.shape
    y = x.double().reshape(t, h, d // GROUP, GROUP)
    low = y.amin(-1, keepdim=True)
    step = ((y.amax(-1, keepdim=True) - low) / 15).half().double()
    low = low.half().double()
    code = torch.where(step > 0, torch.round((y - low) / torch.where(step > 0, step, 1.0)).clamp(0, 15), 0.0)
    return (code * step + low).reshape(t, h, d)


def exact(case, seed):
    g = _generator(seed)
    if case["op"] == "tables":
        return None  # whole numbers
    dt = _DT[case["dtype"]]
    h, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "write":
        k, v = _keys_values(case["tokens"], h, d, dt, g)
        return [_held64(k), _held64(v)]
    kv, new = _lens(case)
    _pages(case, kv, g)
    k, v = _keys_values(sum(kv), h, d, dt, g)
    q = torch.randn((sum(new), case["heads"], d), generator=g, device="cuda").to(dt)
    group = case["heads"] // h
    out = torch.empty((sum(new), case["heads"], d), dtype=torch.float64, device="cuda")
    at = row = 0
    for length, n in zip(kv, new):
        held_k, held_v = _held64(k[at:at + length]), _held64(v[at:at + length])
        key = torch.arange(length, device="cuda")
        for head in range(case["heads"]):
            ks, vs = held_k[:, head // group], held_v[:, head // group]
            for r0 in range(0, n, 1024):
                r1 = min(n, r0 + 1024)
                at_row = torch.arange(length - n + r0, length - n + r1, device="cuda")
                hidden = key[None, :] > at_row[:, None]
                if case["window"]:
                    hidden |= key[None, :] <= at_row[:, None] - case["window"]
                s = (q[row + r0:row + r1, head].double() @ ks.T) * d ** -0.5
                out[row + r0:row + r1, head] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ vs
        at += length
        row += n
    return out
