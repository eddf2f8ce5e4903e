"""Plain 64-bit statements of the 4-bit key/value cache's operators, for the tests."""

import math

import numpy as np
import torch

GROUP = 64


def held(x):
    """(held values f64, steps f64, distance of (x - m)/s from the nearest tie) of x [T, H, D]: the
    group's parameters by the format's f32 formula, the codes by a division in 64 bits."""
    t, h, d = x.shape
    y32 = x.float().clamp(-57344.0, 57344.0).reshape(t, h, d // GROUP, GROUP)
    lo, hi = y32.amin(-1, keepdim=True), y32.amax(-1, keepdim=True)
    step = ((hi - lo) * np.float32(1.0 / 15.0).item()).half().double()
    low = lo.half().double()
    r = (y32.double() - low) / torch.where(step > 0, step, torch.ones_like(step))
    code = torch.where(step > 0, torch.round(r).clamp(0, 15), torch.zeros_like(r))
    tie = (r - torch.floor(r) - 0.5).abs()
    v = code * step + low
    bad = ~torch.isfinite(x.float().reshape(t, h, d // GROUP, GROUP)).all(-1, keepdim=True)
    v = torch.where(bad, torch.full_like(v, math.nan), v)
    full = lambda a: a.expand(t, h, d // GROUP, GROUP).reshape(t, h, d)
    return v.reshape(t, h, d), full(step), tie.reshape(t, h, d)


def attention(q, k, v, scale, window=0):
    """One request: q [n, H, D] at the last n positions of k, v [L, Hk, D] (held values, f64) ->
    (out [n, H, D], bound [n, H, D] on a kernel's error before its final rounding).

    The bound: operands of the products are rounded to 11 bits (relative error u = 2^-11: the
    probability times the step, and in the tile kernel the held key and value), so a score is off by
    at most scale * u * sum |q||k| =: e, a probability's weight by 2 e relatively, and the value sum
    by (2 e + 2 u) * max |v| (f32 sums add less than u/8 at these lengths)."""
    n, heads, d = q.shape
    length, hk, _ = k.shape
    u = 2.0 ** -11
    out = torch.zeros((n, heads, d), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    pos = torch.arange(length - n, length, device=q.device)[:, None]
    key = torch.arange(length, device=q.device)[None, :]
    seen = key <= pos
    if window:
        seen = seen & (key > pos - window)
    if length == 0 or n == 0:
        return out, bound
    any_seen = seen.any(-1)
    for h in range(heads):
        kh, vh, qh = k[:, h // (heads // hk)], v[:, h // (heads // hk)], q[:, h].double()
        s = (qh @ kh.T * scale).masked_fill(~seen, -math.inf)
        s = torch.where(any_seen[:, None], s, torch.zeros_like(s))
        p = torch.softmax(s, -1) * seen
        out[:, h] = torch.where(any_seen[:, None], p @ vh, torch.zeros_like(qh))
        e = ((qh.abs() @ kh.abs().T) * seen).amax(-1) * abs(scale) * u
        bound[:, h] = ((2 * e + 2.25 * u) * vh.abs().max())[:, None]
    return out, bound


def rounding(dtype):
    return {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]


def block_tables(ctx, new, table, free, count, page, tokens):
    """Plain loops over the requests: (table, kv_lens, cu_q, slots, positions, free_left)."""
    table = [list(r) for r in table]
    width, top = len(table[0]), count
    kv, cu, slots, positions = [], [0], [], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        kv.append(c + n)
        cu.append(cu[-1] + n)
        for col in range(-(-c // page), min(-(-(c + n) // page), width)):
            top -= 1
            table[b][col] = free[top] if top >= 0 else -1
        for pos in range(c, c + n):
            positions.append(pos)
            pg = table[b][pos // page] if pos // page < width else -1
            slots.append(pg * page + pos % page if pg >= 0 else -1)
    pad = max(0, tokens - len(slots))
    return table, kv, cu, (slots + [-1] * pad)[:tokens], (positions + [0] * pad)[:tokens], top
