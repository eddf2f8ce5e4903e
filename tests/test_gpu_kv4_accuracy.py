"""Attention over long caches, held to bars that a lost key or a drifting sum breaks (tests/kv4_bars.py)."""

import threading

import pytest
import torch

import kv4_bars as bars
import kv4_ref as ref

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
    assert bars.beyond_rounding(st.run(), st.want()[None].expand(2, -1, -1, -1)) <= bars.BEYOND_BAR


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
