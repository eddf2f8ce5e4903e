"""The bars of tests/kv4_bars.py see what they are for: mistakes planted in a 64-bit attention (no GPU)."""

import pytest
import torch

import kv4_bars as bars

D = 64


def attend(q, k, v, weight):
    """Softmax attention in 64 bits; `weight` [n] multiplies each key's part (0: lost, 2: counted twice)."""
    p = torch.softmax(q @ k.T * D ** -0.5, -1) * weight
    return p @ v / p.sum(-1, keepdim=True)


def plant(n, what):
    w = torch.ones(n, dtype=torch.float64)
    if what == "a lost tenth":
        w[n // 2:n // 2 + n // 10] = 0
    elif what == "a lost tile":
        w[1280:1408] = 0
    elif what == "a lost granule":
        w[1600:1616] = 0
    elif what == "256 keys twice":
        w[512:768] = 2
    return w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [9000, 20000])
def test_the_relative_bar(n, dtype):
    g = torch.Generator()
    g.manual_seed(n)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((8, D), (n, D), (n, D)))
    want = attend(q, 1.5 * k, v, plant(n, "nothing"))
    assert bars.relative(want.to(dtype), want) <= bars.relative_bar(dtype)
    for what in ("a lost tenth", "a lost tile", "a lost granule", "256 keys twice"):
        got = attend(q, 1.5 * k, v, plant(n, what)).to(dtype)
        assert bars.relative(got, want) > bars.relative_bar(dtype), what
    assert bars.relative(v.mean(0, keepdim=True).expand(8, -1).to(dtype), want) > bars.relative_bar(dtype)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 9000), (torch.float16, 9000), (torch.float16, 100003)])
def test_the_count_bar(n, dtype):
    v, block = bars.count_values(n, D)
    v = v.double()
    want = bars.counts(n, 1, D, block)
    even = torch.ones(n, dtype=torch.float64)
    zero, k = torch.zeros((1, D), dtype=torch.float64), torch.zeros((n, D), dtype=torch.float64)
    ok = lambda got: ((got.to(dtype).double() - want).abs() <= bars.count_bar(want, dtype)).all()
    assert ok(attend(zero, k, v, even))
    for key in (0, 15, 16, n // 2, n - 1):
        for times in (0.0, 2.0):
            w = even.clone()
            w[key] = times
            assert not ok(attend(zero, k, v, w)), (key, times)
    # the last row shown one key fewer or more than its position: another row's counts
    assert not ok(bars.counts(n - 1, 1, D, block)) and not ok(bars.counts(n + 1, 1, D, block))


@pytest.mark.parametrize("window", [0, 1, 100, 5000])
def test_the_counts_are_the_definition(window):
    n, rows = 700, 9
    v, block = bars.count_values(n, D)
    for i, want in enumerate(bars.counts(n, rows, D, block, window)):
        pos = n - rows + i
        seen = v[max(0, pos - window + 1) if window else 0:pos + 1].double()
        assert torch.allclose(seen.mean(0), want, rtol=1e-14, atol=0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,rows,d", [(700, 700, 64), (20000, 9000, 128), (131071, 50, 256)])
def test_rounded_counts_are_within_the_bar(n, rows, d, dtype):
    """F16 outputs below 2^-14 round to multiples of 2^-24."""
    block = -(-n // d)
    want = bars.counts(n, rows, d, block)
    assert ((want.to(dtype).double() - want).abs() <= bars.count_bar(want, dtype)).all()
