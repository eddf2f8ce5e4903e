"""Attention over long caches, held to bars that a lost key or a drifting sum breaks (tests/kv4_bars.py)."""

import threading

import pytest
import torch

import kv4_bars as bars
import kv4_ref as ref
from test_gpu_kv4 import Step

pytestmark = pytest.mark.gpu


def sx():
    import sushi_b200

    return sushi_b200


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


class Shared:
    """Many requests over the same pages (one cache of n keys, values without a mean), the same query
    rows in each: more units than the GPU has CTAs, so a CTA sums whole units."""

    def __init__(self, seed, n, requests, rows, heads, kv_heads, d, dtype, page=64):
        f = dict(generator=gen(seed), device="cuda")
        pages = -(-n // page)
        self.cache = sx().Kv4Cache(pages, kv_heads, d, page)
        self.k, self.v = (torch.randn((n, kv_heads, d), **f).to(dtype) for _ in range(2))
        ids = torch.randperm(pages, **f)
        pos = torch.arange(n, device="cuda")
        sx().kv4_write(self.cache, self.k, self.v, ids[pos // page] * page + pos % page)
        self.table = ids.int()[None].repeat(requests, 1)
        self.q = torch.randn((rows, heads, d), **f).to(dtype)
        self.n, self.requests, self.rows, self.heads, self.kv_heads, self.d = n, requests, rows, heads, kv_heads, d

    def run(self):
        cu = [self.rows * b for b in range(self.requests + 1)]
        return sx().kv4_attention(self.q.repeat(self.requests, 1, 1), self.cache, self.table, i32([self.n] * self.requests),
                                  i32(cu), self.rows).reshape(self.requests, self.rows, self.heads, self.d)

    def want(self):
        k, v = ref.held(self.k)[0], ref.held(self.v)[0]
        seen = torch.arange(self.n, device="cuda") <= torch.arange(self.n - self.rows, self.n, device="cuda")[:, None]
        out = []
        for h in range(self.heads):
            kh = h // (self.heads // self.kv_heads)
            s = (self.q[:, h].double() @ k[:, kh].T * self.d ** -0.5).masked_fill(~seen, float("-inf"))
            out.append(torch.softmax(s, -1) @ v[:, kh])
        return torch.stack(out, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,requests,rows,heads,kv_heads,d", [(131072, 64, 1, 16, 8, 128), (131072, 32, 1, 16, 8, 256),
                                                              (131072, 64, 1, 8, 8, 64), (65536, 96, 5, 12, 6, 128),
                                                              (131072, 48, 17, 32, 8, 128)])
def test_sums_do_not_drift_over_long_caches(n, requests, rows, heads, kv_heads, d, dtype):
    st = Shared(n + d, n, requests, rows, heads, kv_heads, d, dtype)
    assert bars.relative(st.run(), st.want()[None]) <= bars.relative_bar(dtype)


@pytest.mark.parametrize("rows,heads,kv_heads,d", [(2, 32, 8, 128), (16, 32, 8, 128), (4, 32, 8, 64), (2, 16, 4, 256), (4, 64, 8, 256)])
def test_bf16_outputs_of_few_rows_are_off_by_little_more_than_their_rounding(rows, heads, kv_heads, d):
    st = Shared(rows + d, 6000, 2, rows, heads, kv_heads, d, torch.bfloat16)
    assert bars.beyond_rounding(st.run(), st.want()[None].expand(2, -1, -1, -1)) <= bars.BEYOND_BAR[torch.bfloat16]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 3, 130])
@pytest.mark.parametrize("at", [5, 40, 291])
def test_a_nan_value_reaches_its_rows_however_little_it_weighs(d, n, at):
    """Key `at` scores 8 * 8 * sqrt(d) below the others, so its probability is 0 in 32 bits; 0 * NaN is NaN."""
    f = dict(generator=gen(d + n + at), device="cuda")
    k, v = (torch.randn((300, 1, d), **f).to(torch.bfloat16) for _ in range(2))
    k[at], v[at, 0, d - 1] = -8.0, float("nan")
    cache = sx().Kv4Cache(19, 1, d, 16)
    sx().kv4_write(cache, k, v, torch.arange(300, device="cuda"))
    q = torch.full((n, 1, d), 8.0, dtype=torch.bfloat16, device="cuda")
    got = sx().kv4_attention(q, cache, torch.arange(19, device="cuda", dtype=torch.int32)[None], i32([300]), i32([0, n]), n)[:, 0]
    first = max(0, at - (300 - n))
    assert torch.isnan(got[first:, d - 64:]).all()
    assert torch.isfinite(got[:first]).all() and torch.isfinite(got[:, :d - 64]).all()


def test_two_host_threads_on_one_stream():
    """Long caches whose units are split over the CTAs and joined, from two threads at once on the default
    stream: the bits of the calls one after another."""
    cases = [Shared(51, 30000, 1, 1, 16, 2, 128, torch.bfloat16), Shared(52, 20000, 2, 40, 16, 2, 128, torch.bfloat16)]
    want = [c.run() for c in cases]
    got, start = [[], []], threading.Barrier(2)

    def thread(i):
        start.wait()
        got[i] = [cases[i].run() for _ in range(60)]

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i in range(2):
        assert len(got[i]) == 60 and all(torch.equal(x, want[i]) for x in got[i])


# ------------------------------------------------------------------ every key counts, once
class Centred(Step):
    """A step whose values have no common mean, so that an output shows its keys and not the mean."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.v = (self.v.float() - 0.5).to(self.dtype)
        sx().kv4_write(self.cache, self.k, self.v, self.slots)


class Counted(Step):
    """A step of the count statement: zero queries, and values that say which block of keys they are of."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.q.zero_()
        self.blocks, v = [], []
        for n, _ in self.lens:
            x, block = bars.count_values(max(n, 1), self.d, "cuda")
            v.append(x[:n])
            self.blocks.append(block)
        v = torch.cat(v)[:, None].expand(-1, self.cache.kv_heads, -1).to(self.dtype)
        if len(v):
            sx().kv4_write(self.cache, self.k, v, self.slots)

    def check(self, got):
        row = 0
        for (n, r), block in zip(self.lens, self.blocks):
            if r and n >= r:
                assert block * (bars.UNIT[self.dtype] + 2.0 ** -20) < 1  # one key is more than the bar
                want = bars.counts(n, r, self.d, block, self.window, "cuda")[:, None]
                err = (got[row:row + r].double() - want).abs()
                assert (err <= bars.count_bar(want, self.dtype)).all(), (n, r, (err - bars.count_bar(want, self.dtype)).max().item())
            row += r


LONG = {
    "one": [(20000, 1)],
    "ragged": [(9000, 1), (3, 1), (4100, 1)],
    "draft": [(12000, 3), (2, 2), (5000, 8)],
    "chunk": [(8200, 70), (100, 1)],
    "mixed": [(5000, 1), (6000, 130), (4321, 5), (2500, 300), (7000, 1)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", list(LONG))
@pytest.mark.parametrize("d,heads,kv_heads,page", [(64, 8, 2, 16), (128, 8, 1, 64), (128, 16, 8, 32), (256, 4, 2, 64)])
def test_long_caches_within_the_relative_bar(d, heads, kv_heads, page, lens, dtype):
    st = Centred(61 + d, d, dtype, heads, kv_heads, page, LONG[lens])
    got, (want, _) = st.run(), st.want()
    row = 0
    for n, r in st.lens:
        if n >= 1000:
            assert bars.relative(got[row:row + r], want[row:row + r]) <= bars.relative_bar(dtype), (n, r)
        row += r


@pytest.mark.parametrize("lens", list(LONG))
@pytest.mark.parametrize("window", [0, 1, 100, 1000, 4099])
@pytest.mark.parametrize("d,heads,kv_heads,page", [(64, 8, 2, 16), (128, 1, 1, 64), (128, 40, 1, 16), (128, 16, 8, 256), (256, 4, 2, 32)])
def test_long_caches_count_every_key_once(d, heads, kv_heads, page, window, lens):
    st = Counted(67 + d, d, torch.float16, heads, kv_heads, page, LONG[lens], window)
    st.check(st.run())


@pytest.mark.parametrize("lens", [[(131071, 1)], [(100003, 2), (60000, 1)], [(99991, 40)]])
@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (16, 8)])
def test_the_longest_caches_count_every_key_once(heads, kv_heads, lens):
    st = Counted(71, 128, torch.float16, heads, kv_heads, 64, lens)
    st.check(st.run())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 2, 7, 33, 150])
def test_short_caches_count_every_key_once(rows, dtype, d):
    """Lengths around every granule, step and tile edge."""
    edges = sorted({max(rows, e + o) for e in (16, 32, 64, 128, 256, 384, 512) for o in (-1, 0, 1, 7)})
    st = Counted(73 + rows, d, dtype, 6, 2, 16, [(n, rows) for n in edges])
    st.check(st.run())


# ------------------------------------------------------------------ many requests
@pytest.mark.parametrize("requests", [64, 65, 129, 513, 1025, 16384])
@pytest.mark.parametrize("d,heads,kv_heads,chunks", [(64, 2, 1, {}), (128, 8, 2, {0: 70, 63: 33, -1: 200}), (256, 16, 1, {7: 5, -2: 90})])
@pytest.mark.parametrize("window", [0, 37])
def test_many_requests_count_every_key_once(requests, d, heads, kv_heads, chunks, window):
    """Ragged requests over one shared row of pages, some without keys or rows, a few with many rows."""
    n, page, g = 400, 16, gen(requests + d)
    lens = torch.randint(0, n + 1, (requests,), generator=g, device="cuda", dtype=torch.int32)
    rows = (torch.rand((requests,), generator=g, device="cuda") < 0.9).int()
    for at, r in chunks.items():
        rows[at], lens[at] = r, 250
    cu = torch.cat([i32([0]), torch.cumsum(rows, 0, dtype=torch.int32)])
    cache = sx().Kv4Cache(n // page, kv_heads, d, page)
    v, block = bars.count_values(n, d, "cuda")
    k = torch.randn((n, kv_heads, d), generator=g, device="cuda").half()
    ids = torch.randperm(n // page, generator=g, device="cuda")
    pos = torch.arange(n, device="cuda")
    sx().kv4_write(cache, k, v[:, None].expand(-1, kv_heads, -1).half(), ids[pos // page] * page + pos % page)
    tokens = int(cu[-1])
    q = torch.zeros((tokens + 3, heads, d), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    sx().kv4_attention(q, cache, ids.int()[None].repeat(requests, 1), lens, cu, max([1, *chunks.values()]), window=window, out=out)
    b = torch.repeat_interleave(torch.arange(requests, device="cuda"), rows.long())
    at = lens.long()[b] - rows.long()[b] + torch.arange(tokens, device="cuda") - cu.long()[b]
    want = bars.counts_at(at, d, block, window)
    assert ((out[:tokens].double() - want[:, None]).abs() <= bars.count_bar(want, torch.float16)[:, None]).all()
    assert not out[tokens:].any()
    assert sx().device_error() == 0


# ------------------------------------------------------------------ scores of any finite magnitude
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,rows", [(300, 1), (300, 3), (700, 130), (20000, 1), (9000, 40)])
@pytest.mark.parametrize("q,scale", [(1e4, None), (1e7, None), (1e20, None), (1e36, None), (3.3e38, None), (-1e30, None), (-3.3e38, -1.0),
                                     (1.0, 1e30), (1e-3, -1e20), (1e-38, None), (1e-38, 1e20), (3e38, 0.0)])
def test_scores_of_any_finite_magnitude(n, rows, d, q, scale):
    """One key points along the query, one against it, ten times as far as any other: the softmax is one of
    them, or the mean where scores are nothing."""
    f = dict(generator=gen(n + rows + d), device="cuda")
    k = (torch.rand((n, 1, d), **f) * 0.2 - 0.1).to(torch.bfloat16)
    v = torch.randn((n, 1, d), **f).to(torch.bfloat16)
    first = n - rows
    at, against = first // 3, first // 2  # seen by every row
    k[at], k[against] = 1.0, -1.0
    page = 64
    pages = -(-n // page)
    cache = sx().Kv4Cache(pages, 1, d, page)
    sx().kv4_write(cache, k, v, torch.arange(n, device="cuda"))
    qs = torch.full((rows, 6, d), q, dtype=torch.bfloat16, device="cuda")
    got = sx().kv4_attention(qs, cache, torch.arange(pages, device="cuda", dtype=torch.int32)[None], i32([n]), i32([0, rows]), rows,
                             scale=scale)
    values = ref.held(v)[0][:, 0]
    s = (d ** -0.5 if scale is None else scale) * float(qs[0, 0, 0]) * d
    if abs(s) > 1e3:
        want = values[at if s > 0 else against].expand(rows, 6, d)
        assert ((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -10) * want.abs().max()).all()
    else:
        want = (values.cumsum(0) / torch.arange(1, n + 1, device="cuda")[:, None])[first:, None]
        assert abs(s) < 1e-10 and bars.relative(got, want) <= bars.relative_bar(torch.bfloat16)
    assert sx().device_error() == 0


# ------------------------------------------------------------------ rows that see nothing
@pytest.mark.parametrize("d,heads,kv_heads", [(64, 4, 2), (128, 32, 8), (256, 16, 1)])
@pytest.mark.parametrize("lens,window", [([(0, 4000), (5000, 1)], 0), ([(10, 1700), (0, 513), (5000, 1), (0, 1)], 0),
                                         ([(0, 3)] * 500 + [(300, 2), (100, 400)], 0), ([(0, 200), (7, 1)] * 60, 9)])
def test_rows_without_keys_are_zero_and_others_count_every_key(d, heads, kv_heads, lens, window):
    """Whole requests without keys, and blocks of rows before the first key."""
    st = Counted(79 + d, d, torch.float16, heads, kv_heads, 16, lens, window)
    out = torch.full_like(st.q, 7.0)
    st.run(out=out)
    st.check(out)
    row = 0
    for n, r in lens:
        assert not out[row:row + max(0, r - n)].any()
        if n and r > n:
            want = bars.counts(n, n, d, st.blocks[lens.index((n, r))], window, "cuda")[:, None]
            assert ((out[row + r - n:row + r].double() - want).abs() <= bars.count_bar(want, torch.float16)).all()
        row += r


@pytest.mark.parametrize("rows", [3, 900])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_windows_past_a_narrow_table_see_nothing(d, rows):
    """Rows whose window lies past the table's pages are 0; the others see the window's part that has pages."""
    n, window, held = 3000, 40, 2560
    st = Counted(83 + d, d, torch.float16, 8, 2, 16, [(n, rows)], window)
    st.table = st.table[:, :held // 16].contiguous()
    out = torch.full_like(st.q, 7.0)
    st.run(out=out)
    pos = torch.arange(n - rows, n, device="cuda")
    assert not out[pos - window + 1 >= held].any()
    whole = pos < held
    want = bars.counts_at(pos[whole], d, st.blocks[0], window)[:, None]
    assert ((out[whole].double() - want).abs() <= bars.count_bar(want, torch.float16)).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("pairs", [60, 64, 68, 92, 96, 100, 128])
@pytest.mark.parametrize("widest", [0, 200])
def test_both_sides_of_the_kernel_choice(pairs, widest, d):
    """Requests of 60 to 128 pairs a key head, alone (16 columns a unit) or beside a chunk (8)."""
    st = Counted(89 + d, d, torch.float16, 8, 2, 64, [(2000, pairs // 4), (1000 + widest, max(1, widest)), (3, 1)])
    st.check(st.run())
    got = Centred(97 + d, d, torch.bfloat16, 8, 2, 64, [(2000, pairs // 4), (1500, max(1, widest))])
    out, (want, _) = got.run(), got.want()
    assert bars.relative(out, want) <= bars.relative_bar(torch.bfloat16)


@pytest.mark.parametrize("rows,heads,kv_heads,d", [(2, 32, 8, 128), (4, 32, 8, 64), (2, 16, 4, 256), (40, 32, 8, 128), (300, 4, 1, 128),
                                                   (130, 16, 8, 64), (70, 8, 4, 256), (9, 32, 2, 256)])
@pytest.mark.parametrize("n", [700, 6000])
def test_f16_outputs_are_off_by_little_more_than_their_rounding(rows, heads, kv_heads, d, n):
    st = Shared(rows + d, n, 2, rows, heads, kv_heads, d, torch.float16)
    assert bars.beyond_rounding(st.run(), st.want()[None].expand(2, -1, -1, -1)) <= bars.BEYOND_BAR[torch.float16]


@pytest.mark.parametrize("rows", [1, 120])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("gain,shift", [(1e-4, 0.0), (1.0, 30.0), (500.0, -2e4), (3e3, 1e4)])
def test_f16_values_of_any_magnitude_keep_their_bits(gain, shift, d, rows):
    """Values around 1e-4 to those near the format's largest, with and without a mean: the error of a row
    against its values' size, which is what the parts of a value are taken against."""
    st = Shared(rows + d, 3000, 2, rows, 4, 2, d, torch.float16)
    st.v = (st.v.float() * gain + shift).half()
    pages = st.table.shape[1]
    pos = torch.arange(st.n, device="cuda")
    sx().kv4_write(st.cache, st.k, st.v, st.table[0].long()[pos // 64] * 64 + pos % 64)
    want, size = st.want()[None], ref.held(st.v)[0].abs().max()
    err = (st.run().double() - want).abs()
    assert pages and (err <= 2.0 ** -11 * want.abs() + 2.0 ** -15 * size + 2.0 ** -25).all()


# ------------------------------------------------------------------ units of many tiles
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,window", [([(40000, 70)] * 4, 0), ([(9000, 70), (8257, 66)] * 12, 0), ([(20000, 9000)], 0), ([(30000, 1500)], 9500)])
def test_units_of_many_tiles_count_every_key_once(lens, window, d, dtype):
    """More tiles than an F16 call sums at a time in tensor memory, of whole units and of shared ones."""
    n = max(n for n, _ in lens)
    st = Counted(101 + d, d, dtype, 8, 4, 64, lens, window)
    got = st.run()
    if n // d < 240:  # one key shows beside the output's rounding
        st.check(got)
    assert torch.equal(got, st.run())
    st = Centred(103 + d, d, dtype, 4, 2, 64, lens[:2], window)
    got, row = st.run(), 0
    for (n, r), k, v in zip(st.lens, st.k.split([n for n, _ in st.lens]), st.v.split([n for n, _ in st.lens])):
        rows = torch.arange(0, r, max(1, r // 50), device="cuda")
        kk, vv = ref.held(k)[0], ref.held(v)[0]
        pos, key = n - r + rows[:, None], torch.arange(n, device="cuda")[None]
        seen = (key <= pos) & (key > pos - window if window else key >= 0)
        for h in range(4):
            s = (st.q[row + rows, h].double() @ kk[:, h // 2].T * d ** -0.5).masked_fill(~seen, float("-inf"))
            assert bars.relative(got[row + rows, h], torch.softmax(s, -1) @ vv[:, h // 2]) <= bars.relative_bar(dtype)
        row += r


@pytest.mark.parametrize("rows,heads,kv_heads,d", [(40, 16, 4, 128), (100, 4, 4, 64), (70, 4, 4, 256)])
def test_f16_outputs_of_many_rows_over_long_caches(rows, heads, kv_heads, d):
    """Units of hundreds of tiles a CTA: what the matrix unit cuts of its sums must not grow with them."""
    st = Shared(107 + d, 60000, 40, rows, heads, kv_heads, d, torch.float16)
    assert bars.beyond_rounding(st.run(), st.want()[None].expand(40, -1, -1, -1)) <= bars.BEYOND_BAR[torch.float16]


@pytest.mark.parametrize("rows,heads,kv_heads,d", [(1, 32, 8, 128), (2, 32, 4, 64), (1, 16, 4, 256), (40, 16, 4, 128), (3, 64, 4, 128)])
@pytest.mark.parametrize("n,requests", [(20000, 1), (131071, 1), (60000, 40)])
def test_f16_outputs_of_long_caches_with_strong_channels(n, requests, rows, heads, kv_heads, d):
    """Keys with a few channels four times the others: the weights of a granule's keys differ widely."""
    st = Shared(n + d, n, requests, rows, heads, kv_heads, d, torch.float16)
    g = gen(5)
    st.k = (st.k.float() * (1.0 + 3.0 * (torch.rand((kv_heads, d), generator=g, device="cuda") < 0.05))).half()
    pos = torch.arange(n, device="cuda")
    sx().kv4_write(st.cache, st.k, st.v, st.table[0].long()[pos // 64] * 64 + pos % 64)
    want = st.want()[None].expand(requests, -1, -1, -1)
    assert bars.beyond_rounding(st.run(), want) <= bars.BEYOND_BAR[torch.float16] * (1 if n < 1e5 or rows < 40 else 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_request_past_max_q_is_right_or_nan(d, dtype):
    """A caller that understates max_q gets no stale memory: rows of a request that only the tile kernel could take
    are NaN, the others right."""
    lens = [(900, 1), (700, 100), (0, 90), (500, 3), (64, 1)]
    st = Counted(109 + d, d, dtype, 8, 2, 16, lens)
    right, out = st.run(), torch.full_like(st.q, 7.0)
    st.max_q = 3
    st.run(out=out)
    wide = torch.zeros(st.rows, dtype=torch.bool, device="cuda")
    wide[1:191] = True
    assert torch.isnan(out[wide]).all()
    st.blocks = [b for (_, r), b in zip(lens, st.blocks) if r < 90]
    st.lens = [(n, r) for n, r in lens if r < 90]
    st.check(out[~wide])
    st.check(right[~wide])
