"""The 4-bit key/value cache on the GPU against plain 64-bit statements (tests/kv4_ref.py)."""

import math
import random

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu


def sx():
    import sushi_b200

    return sushi_b200


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ block tables
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("requests,top", [(1, 1), (1, 700), (3, 40), (33, 300), (257, 90), (1025, 40)])
def test_block_tables_match_the_loops(page, requests, top):
    r = random.Random(requests * 1000 + page)
    ctx = [r.choice([0, 0, 1, page - 1, page, page + 1, r.randrange(top)]) for _ in range(requests)]
    new = [r.choice([0, 1, 1, 1, page, page + 1, r.randrange(top)]) for _ in range(requests)]
    ctx[-1] = -5 if requests > 30 else ctx[-1]
    width = max(1, max(-(-(max(c, 0) + n) // page) for c, n in zip(ctx, new)) - (1 if requests == 33 else 0))
    need = sum(max(0, min(-(-(max(c, 0) + n) // page), width) - -(-max(c, 0) // page)) for c, n in zip(ctx, new))
    count = need // 2 if requests == 257 else need + 3  # a stack that runs short
    ids = list(range(need + 3 + requests * width))
    r.shuffle(ids)
    free = ids[:need + 3]
    table = [[ids[need + 3 + b * width + j] if j * page < max(ctx[b], 0) else -7 for j in range(width)] for b in range(requests)]
    tokens = sum(new) + (5 if requests != 3 else -min(2, sum(new)))  # room to spare, or too little
    want = ref.block_tables(ctx, new, table, free, count, page, tokens)
    wide = torch.full((requests, width + 3), -9, dtype=torch.int32, device="cuda")  # rows wider than the table
    wide[:, :width] = i32(table)
    got = sx().block_tables(i32(ctx), i32(new), wide[:, :width], i32(free), i32([count]), page, tokens)
    assert wide[:, :width].tolist() == want[0]
    assert (wide[:, width:] == -9).all()
    assert got.kv_lens.tolist() == want[1] and got.cu_q.tolist() == want[2]
    assert got.slots.tolist() == want[3] and got.positions.tolist() == want[4]
    assert got.free_left.tolist() == [want[5]]
    before = wide.clone()  # a step can be prepared again
    again = sx().block_tables(i32(ctx), i32(new), wide[:, :width], i32(free), i32([count]), page, tokens)
    assert torch.equal(before, wide) and all(torch.equal(a, b) for a, b in zip(got, again))


def test_block_tables_of_the_most_requests():
    n = 16384
    ctx = i32([b % 97 for b in range(n)])
    new = i32([(b * 7) % 5 for b in range(n)])
    table = torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
    table[:, :7] = torch.arange(7, device="cuda", dtype=torch.int32)
    free = torch.arange(100, 100 + n, device="cuda", dtype=torch.int32)
    total = int(new.sum())
    want = ref.block_tables(ctx.tolist(), new.tolist(), table.tolist(), free.tolist(), n, 16, total)
    got = sx().block_tables(ctx, new, table, free, i32([n]), 16, total)
    assert table.tolist() == want[0] and got.slots.tolist() == want[3] and got.free_left.item() == want[5]
    assert got.cu_q.tolist() == want[2] and got.positions.tolist() == want[4]


# ------------------------------------------------------------------ write and read
def check_held(got, x):
    """got f32 against the 64-bit statement: 2^-23 relative where the code is clear of a tie (the
    product and the sum round once each in 24 bits), else at most a step off."""
    want, step, tie = ref.held(x)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    err = (got.double() - want).abs()
    fine = (err <= 2.0 ** -23 * (want.abs() + 16 * step)) | nan
    near = (tie < 1e-5) & (err <= 1.001 * step)
    assert (fine | near).all(), (err[~(fine | near)][:8], want[~(fine | near)][:8])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,page,layout", [(1, 1, 16, "plain"), (37, 3, 16, "fused"), (130, 2, 64, "plain"),
                                                      (65, 5, 256, "odd"), (257, 1, 32, "heads")])
def test_write_then_read(d, dtype, tokens, heads, page, layout):
    g = gen(d + tokens)
    k, v = (torch.randn((tokens, heads, d), generator=g, device="cuda") * 3 + 1 for _ in range(2))
    k[:, :, 1] *= 20
    v[0] = 0.25  # a constant group: step 0
    if tokens > 2:
        v[1, 0, :d // 2] = 1e-7  # tiny steps: below f16's smallest normal
        v[1, 0, d // 2:] = torch.linspace(-3e-6, 3e-6, d // 2, device="cuda")
        k[2] = torch.arange(d, device="cuda") % 31 - 15.0  # codes at and between ties
    k, v = k.to(dtype), v.to(dtype)
    if layout == "fused":
        both = torch.cat([k, v, k], 1)
        a, b = both[:, :heads], both[:, heads:2 * heads]
    elif layout == "odd":  # rows that do not start on 16 bytes
        wide = torch.empty((2, tokens, heads, d + 1), dtype=dtype, device="cuda")
        wide[0, :, :, 1:], wide[1, :, :, 1:] = k, v
        a, b = wide[0, :, :, 1:], wide[1, :, :, 1:]
    elif layout == "heads":  # heads outermost
        a, b = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    else:
        a, b = k, v
    pages = -(-tokens // page) + 2
    c = sx().Kv4Cache(pages, heads, d, page)
    c.pool.fill_(0xff)
    perm = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    sx().kv4_write(c, a, b, perm)
    gk, gv = sx().kv4_read(c, perm, torch.float32)
    check_held(gk, k)
    check_held(gv, v)
    for dt in (torch.bfloat16, torch.float16):
        hk, hv = sx().kv4_read(c, perm, dt)
        assert torch.equal(hk, gk.to(dt)) and torch.equal(hv, gv.to(dt))


def test_write_skips_and_read_zeroes_places_outside_the_pool():
    c = sx().Kv4Cache(3, 2, 64, 16)
    c.pool.fill_(0x5a)
    before = c.pool.clone()
    x = torch.randn((5, 2, 64), device="cuda").to(torch.bfloat16)
    out = torch.tensor([-1, 48, 1 << 40, -(1 << 40), 49], device="cuda")
    sx().kv4_write(c, x, x, out)
    assert torch.equal(c.pool, before)
    k, v = sx().kv4_read(c, out)
    assert not k.any() and not v.any()
    sx().kv4_write(c, x, x, torch.tensor([-1, 47, -1, 0, 17], device="cuda"))
    k, _ = sx().kv4_read(c, torch.tensor([47, 0, 17], device="cuda"), torch.float32)
    check_held(k, x[[1, 3, 4]])


def test_write_of_extreme_values():
    x = torch.randn((6, 1, 128), device="cuda")
    x[0, 0, 3] = math.inf
    x[1, 0, 70] = -math.inf
    x[2, 0, 5] = math.nan
    x[3, 0, 0], x[3, 0, 1] = 3e38, -3e38  # finite, past the format's largest
    x[4, 0, :] = 65504.0
    x = x.to(torch.bfloat16)
    c = sx().Kv4Cache(1, 1, 128, 16)
    s = torch.arange(6, device="cuda")
    sx().kv4_write(c, x, x, s)
    k, v = sx().kv4_read(c, s, torch.float32)
    check_held(k, x)
    check_held(v, x)
    assert torch.isnan(k[0, 0, :64]).all() and torch.isfinite(k[0, 0, 64:]).all()


# ------------------------------------------------------------------ attention
class Step:
    """A filled cache and one call's inputs.  Unwritten places hold NaN parameters."""

    def __init__(self, seed, d, dtype, heads, kv_heads, page, lens, window=0, spare=2, qgain=1.0):
        g = gen(seed)
        self.d, self.dtype, self.heads, self.window = d, dtype, heads, window
        self.lens = lens  # (kv_len, q_len) of each request
        width = max(1, max(-(-n // page) for n, _ in lens))
        counts = [-(-n // page) for n, _ in lens]
        pages = sum(counts) + spare
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        at, slots = 0, []
        for b, (n, _) in enumerate(lens):
            self.table[b, :counts[b]] = perm[at:at + counts[b]]
            at += counts[b]
            pos = torch.arange(n, device="cuda")
            slots.append(self.table[b].long()[pos // page] * page + pos % page if n else pos)
        total = sum(n for n, _ in lens)
        f = dict(generator=g, device="cuda")
        self.k = (torch.randn((total, kv_heads, d), **f) * 1.5 + 0.5 * torch.randn((kv_heads, d), **f)).to(dtype)
        self.v = (torch.randn((total, kv_heads, d), **f) + 0.5).to(dtype)
        self.rows = sum(n for _, n in lens)
        self.q = (qgain * torch.randn((self.rows, heads, d), **f)).to(dtype)
        self.cache = sx().Kv4Cache(pages, kv_heads, d, page)
        self.cache.pool.fill_(0xff)
        self.slots = torch.cat(slots)
        if total:
            sx().kv4_write(self.cache, self.k, self.v, self.slots)
        cu = [0]
        for _, n in lens:
            cu.append(cu[-1] + n)
        self.cu, self.kv_lens = i32(cu), i32([n for n, _ in lens])
        self.max_q = max(1, max(n for _, n in lens))

    def run(self, q=None, **kw):
        kw.setdefault("window", self.window)
        return sx().kv4_attention(self.q if q is None else q, self.cache, self.table, self.kv_lens, self.cu, self.max_q, **kw)

    def want(self, scale=None):
        scale = self.d ** -0.5 if scale is None else scale
        k, v = ref.held(self.k)[0], ref.held(self.v)[0]
        outs, bounds, at, row = [], [], 0, 0
        for n, r in self.lens:
            # rows before position 0 (q_len > kv_len) see nothing
            o, b = ref.attention(self.q[row:row + r], k[at:at + n], v[at:at + n], scale, self.window)
            outs.append(o)
            bounds.append(b)
            at += n
            row += r
        return torch.cat(outs), torch.cat(bounds)

    def check(self, got, scale=None):
        want, bound = self.want(scale)
        err = (got.double() - want).abs()
        tol = bound + ref.rounding(self.dtype) * (want.abs() + bound)
        assert torch.isfinite(got).all()
        assert (err <= tol).all(), f"worst {(err - tol).max().item()} of {want.abs().max().item()}"


LENS = {
    "one": [(1, 1)],
    "single": [(n, 1) for n in (1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 128, 129, 255, 257, 400)],
    "empty": [(0, 1), (5, 0), (0, 0), (7, 9), (3, 1), (0, 3), (64, 1)],
    "draft": [(9, 2), (64, 4), (65, 3), (130, 8), (1, 1), (77, 5), (3, 3)],
    "mixed": [(300, 1), (200, 200), (129, 1), (260, 37), (64, 64), (500, 130), (17, 1)],
    "long": [(5000, 1), (333, 1)],
}


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 4, 7])
def test_attention_of_long_units(d, group):
    """Units of many tiles a CTA, whole and shared, so that every ring goes round several times."""
    st = Step(d + group, d, torch.bfloat16, 8 * group, 8, 64, [(4100, 700), (900, 900), (2500, 300)])
    first = st.run()
    st.check(first)
    assert torch.equal(st.run(), first)
    assert sx().device_error() == 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("heads,kv_heads,page,window", [(1, 1, 16, 0), (8, 2, 64, 0), (7, 1, 32, 50), (32, 2, 128, 0),
                                                        (40, 1, 16, 0), (12, 4, 256, 16)])
def test_attention(d, dtype, lens, heads, kv_heads, page, window):
    st = Step(7 * d + heads, d, dtype, heads, kv_heads, page, LENS[lens], window)
    st.check(st.run())
    assert sx().device_error() == 0


@pytest.mark.parametrize("window", [1, 2, 16, 64, 65, 1 << 20, (1 << 31) - 1])
def test_attention_windows(window):
    st = Step(window, 128, torch.bfloat16, 8, 2, 16, [(1, 1), (64, 1), (65, 2), (200, 150), (513, 1), (129, 129)], window)
    st.check(st.run())


@pytest.mark.parametrize("lens", [[(20000, 1)], [(9000, 1), (3, 1), (4100, 1)], [(12000, 3), (2, 2)], [(8200, 70), (100, 1)]])
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (16, 8)])
def test_attention_split_over_long_caches(lens, heads, kv_heads):
    st = Step(len(lens), 128, torch.bfloat16, heads, kv_heads, 64, lens)
    first = st.run()
    st.check(first)
    for _ in range(3):  # the split's sums are joined in one order: the same bits every time
        assert torch.equal(st.run(), first)


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.5])
def test_attention_scales(scale):
    st = Step(3, 64, torch.float16, 4, 2, 16, [(100, 1), (40, 40), (64, 2)])
    st.check(st.run(scale=scale), scale)


@pytest.mark.parametrize("gain", [1e-5, 300.0])
@pytest.mark.parametrize("n", [1, 80])
def test_attention_of_small_and_large_queries(gain, n):
    # 300: the softmax is nearly one-hot and scores reach the thousands
    st = Step(5, 128, torch.bfloat16, 8, 2, 32, [(300, n), (90, 1)], qgain=gain)
    st.check(st.run())


def test_attention_of_strided_queries_and_tables():
    st = Step(11, 128, torch.bfloat16, 8, 2, 64, [(300, 1), (70, 20), (64, 3)])
    want = st.run()
    fused = torch.cat([st.q, st.q[:, :4]], 1)  # [tokens, q + k + v heads]
    assert torch.equal(st.run(fused[:, :8]), want)
    odd = torch.zeros((st.rows, 8, 129), dtype=st.dtype, device="cuda")
    odd[:, :, 1:] = st.q
    assert torch.equal(st.run(odd[:, :, 1:]), want)  # rows that do not start on 16 bytes
    outer = st.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(st.run(outer), want)
    wide = torch.full((st.table.shape[0], st.table.shape[1] + 5), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, :st.table.shape[1]] = st.table
    st.table = wide[:, :st.table.shape[1]]
    assert torch.equal(st.run(), want)
    st.table = wide  # page ids past the lengths are never used
    assert torch.equal(st.run(), want)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_passes_over_pages_outside_the_pool(n):
    st = Step(13, 128, torch.bfloat16, 8, 2, 16, [(200, n)])
    st.table[0, 3], st.table[0, 6] = -1, 1 << 30
    k, v = ref.held(st.k)[0], ref.held(st.v)[0]
    keep = torch.tensor([p // 16 not in (3, 6) for p in range(200)], device="cuda")
    got = st.run()
    for i in range(n):
        end = 200 - n + i + 1
        o, b = ref.attention(st.q[i:i + 1], k[:end][keep[:end]], v[:end][keep[:end]], 128 ** -0.5)
        assert ((got[i:i + 1].double() - o).abs() <= b + ref.rounding(st.dtype) * (o.abs() + b)).all()
    st.table[:] = -1
    assert not st.run().any()


@pytest.mark.parametrize("n", [1, 30])
def test_attention_of_a_table_narrower_than_the_length(n):
    st = Step(17, 64, torch.bfloat16, 4, 2, 16, [(100, n)])
    k, v = ref.held(st.k)[0], ref.held(st.v)[0]
    st.table = st.table[:, :4].contiguous()  # 64 of the 100 positions
    got = st.run()
    for i in range(n):
        end = min(64, 100 - n + i + 1)
        o, b = ref.attention(st.q[i:i + 1], k[:end], v[:end], 64 ** -0.5)
        assert ((got[i:i + 1].double() - o).abs() <= b + ref.rounding(st.dtype) * (o.abs() + b)).all()


def test_rows_past_the_requests_are_zero():
    st = Step(19, 128, torch.bfloat16, 8, 2, 64, [(100, 1), (50, 1)])
    q = torch.cat([st.q, torch.full_like(st.q, math.nan)])
    out = torch.full_like(q, 7.0)
    st.run(q, out=out)
    st.check(out[:2])
    assert not out[2:].any()


@pytest.mark.parametrize("n", [1, 25])
def test_nan_and_infinity_reach_only_the_rows_that_see_them(n):
    st = Step(23, 128, torch.bfloat16, 8, 2, 16, [(100, n), (60, n)])
    clean = st.run()
    k = st.k[90:91].clone()
    k[0, 1, 5] = math.inf
    sx().kv4_write(st.cache, k, st.v[90:91], st.slots[90:91])
    got = st.run()
    first = n - 10 if n > 10 else 0  # rows at positions >= 90 of request 0 see it, in the heads of key head 1
    assert torch.isnan(got[first:n, 4:]).all()
    assert torch.equal(got[:first], clean[:first]) and torch.equal(got[:n, :4], clean[:n, :4])
    assert torch.equal(got[n:], clean[n:])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 3, 130])
def test_nan_values_reach_only_the_rows_that_see_them(d, n):
    st = Step(24, d, torch.bfloat16, 4, 2, 16, [(300, n), (60, 1)])
    clean = st.run()
    at = 299 if n == 3 else 290
    v = st.v[at:at + 1].clone()
    v[0, 1, d - 3] = math.nan
    sx().kv4_write(st.cache, st.k[at:at + 1], v, st.slots[at:at + 1])
    got = st.run()
    first = max(0, at - (300 - n))
    group = slice(d - 64, d)  # the channels of the NaN's group, in the heads of key head 1
    assert torch.isnan(got[first:n, 2:, group]).all()
    assert torch.equal(got[:first], clean[:first]) and torch.equal(got[:n, :2], clean[:n, :2])
    assert torch.equal(got[:n, :, :d - 64], clean[:n, :, :d - 64])
    assert torch.equal(got[n:], clean[n:])


def test_values_of_any_magnitude():
    """Steps far below and above 1, and growing along the keys (the streaming kernel's reference follows them)."""
    for scale in (1e-3, 1.0, 2000.0):
        for n in (1, 40):
            st = Step(25, 128, torch.bfloat16, 8, 2, 16, [(500, n)])
            ramp = torch.logspace(-2, 1, 500, device="cuda")[:, None, None] * scale
            st.v = (st.v.float() * ramp).to(torch.bfloat16)
            sx().kv4_write(st.cache, st.k, st.v, st.slots)
            st.check(st.run())


def test_attention_past_32_bit_offsets():
    """Pages whose bytes lie past 2^31 and 2^32 of a 5 GB pool."""
    pages = 68000
    c = sx().Kv4Cache(pages, 8, 128, 64)
    assert c.pool.numel() > 1 << 32
    g = gen(29)
    n = 300
    ids = torch.tensor([pages - 1, 0, pages // 2 + 1, pages - 2, 3], device="cuda")
    pos = torch.arange(n, device="cuda")
    slots = ids[pos // 64] * 64 + pos % 64
    k, v = (torch.randn((n, 8, 128), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    sx().kv4_write(c, k, v, slots)
    check_held(sx().kv4_read(c, slots, torch.float32)[0], k)
    for rows in (1, 40):
        q = torch.randn((rows, 16, 128), generator=g, device="cuda").to(torch.bfloat16)
        got = sx().kv4_attention(q, c, ids.int()[None], i32([n]), i32([0, rows]), rows)
        o, b = ref.attention(q, ref.held(k)[0], ref.held(v)[0], 128 ** -0.5)
        assert ((got.double() - o).abs() <= b + 2.0 ** -8 * (o.abs() + b)).all()


def test_one_workspace_for_calls_of_other_sizes():
    steps = [Step(31, 128, torch.bfloat16, 8, 2, 64, l) for l in ([(9000, 1)], [(300, 60), (5000, 2)], [(40, 1)] * 50, [(7000, 33)])]
    alone = [st.run() for st in steps]
    need = max(sx().kv4_attention_workspace_bytes(st.cache, len(st.lens), st.rows, 8, st.max_q) for st in steps)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")  # whatever it held before
    for _ in range(2):
        for st, want in zip(steps, alone):
            assert torch.equal(st.run(workspace=ws), want)


def test_attention_on_another_stream_and_in_a_graph():
    st = Step(37, 128, torch.bfloat16, 8, 2, 64, [(3000, 1), (500, 40), (90, 2)])
    want = st.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [st.run() for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(x, want) for x in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rec = st.run()
    assert torch.equal(st.run(), want)  # eager calls between recording and replay
    for _ in range(2):
        rec.zero_()
        graph.replay()
        assert torch.equal(rec, want)
    fresh = Step(38, 128, torch.bfloat16, 8, 2, 64, [(3000, 1), (500, 40), (90, 2)])
    st.q.copy_(fresh.q)  # new inputs in the recorded buffers
    graph.replay()
    assert torch.equal(rec, st.run())


def test_a_whole_step_of_block_tables_write_and_attention():
    """Requests grow over several steps through the public calls; the last step against the whole history."""
    heads, kv_heads, d, page, dt = 8, 2, 128, 16, torch.bfloat16
    g = gen(41)
    c = sx().Kv4Cache(64, kv_heads, d, page)
    c.pool.fill_(0xff)
    free, count = torch.randperm(64, generator=g, device="cuda").int(), i32([64])
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    ctx = i32([0, 0, 0])
    hist = [([], []) for _ in range(3)]
    for new in ([40, 17, 0], [1, 1, 90], [1, 1, 1], [1, 0, 1], [30, 1, 1]):
        t = sx().block_tables(ctx, i32(new), table, free, count, page, sum(new))
        k, v = (torch.randn((sum(new), kv_heads, d), generator=g, device="cuda").to(dt) for _ in range(2))
        q = torch.randn((sum(new), heads, d), generator=g, device="cuda").to(dt)
        sx().kv4_write(c, k, v, t.slots)
        got = sx().kv4_attention(q, c, table, t.kv_lens, t.cu_q, max(new))
        at = 0
        for b, n in enumerate(new):
            hist[b][0].append(k[at:at + n])
            hist[b][1].append(v[at:at + n])
            o, e = ref.attention(q[at:at + n], ref.held(torch.cat(hist[b][0]))[0], ref.held(torch.cat(hist[b][1]))[0], d ** -0.5)
            assert ((got[at:at + n].double() - o).abs() <= e + 2.0 ** -8 * (o.abs() + e)).all()
            at += n
        ctx, count = t.kv_lens, t.free_left
    assert count.item() == 64 - sum(-(-sum(x.shape[0] for x in h[0]) // page) for h in hist)


def test_refusals_by_name():
    st = Step(43, 128, torch.bfloat16, 8, 2, 64, [(100, 1)])
    E = sx().Exl3Error
    with pytest.raises(E, match="SX_ERR_BAD_DTYPE"):
        st.run(st.q.float())
    with pytest.raises(E, match="SX_ERR_BAD_SHAPE"):
        st.run(st.q[:, :7])
    with pytest.raises(E, match="SX_ERR_BAD_SHAPE"):
        st.run(st.q[:, :, :64])
    with pytest.raises(E, match="SX_ERR_BAD_SHAPE"):
        st.run(out=torch.empty((1, 8, 64), dtype=st.dtype, device="cuda"))
    with pytest.raises(E, match="SX_ERR_BAD_SHAPE"):
        st.run(window=-1)
    with pytest.raises(E, match="SX_ERR_WORKSPACE_TOO_SMALL"):
        st.run(workspace=torch.zeros(0, dtype=torch.uint8, device="cuda").new_zeros(8))
    with pytest.raises(E, match="SX_ERR_BAD_DTYPE"):
        sx().kv4_write(st.cache, st.k, st.v.half(), st.slots)
    with pytest.raises(E, match="SX_ERR_BAD_DTYPE"):
        sx().kv4_write(st.cache, st.k, st.v, st.slots.int())
    with pytest.raises(E, match="SX_ERR_BAD_SHAPE"):
        sx().kv4_write(st.cache, st.k[:5], st.v, st.slots)
    with pytest.raises(E, match="SX_ERR_BAD_SHAPE"):
        sx().kv4_write(st.cache, st.k, st.v, st.slots[:5])
    with pytest.raises(E, match="SX_ERR_BAD_DTYPE"):
        sx().kv4_read(st.cache, st.slots, torch.int32)


def test_the_example_layer():
    """Prompt, decode and graph steps of an EXL3 attention layer; a decoded row against the same row of a
    whole prompt: bf16 activations through two projections and both attention kernels, each rounded
    to 2^-8, four roundings deep."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "kv4_layer.py")
    spec = importlib.util.spec_from_file_location("kv4_layer", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main() < 4 * 2.0 ** -8
    assert sx().device_error() == 0
