"""The 4-bit cache's entry points on the host (no GPU): block sizes and refusals before any launch."""

import ctypes

import pytest

from sushi_b200 import _lib

FAKE = 0x10000


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def name(L, st):
    return L.sx_status_name(st).decode()


def cache(pool=FAKE, pages=4, kv_heads=2, head_dim=128, page_size=64):
    return _lib.SxKv4(pool, pages, kv_heads, head_dim, page_size)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("p", [16, 32, 64, 128, 256])
def test_block_bytes_are_four_and_a_half_bits_a_channel(L, d, p):
    assert L.sx_kv4_block_bytes(d, p) == 2 * p * d * 9 // 16


@pytest.mark.parametrize("d,p", [(0, 16), (96, 16), (512, 16), (128, 0), (128, 8), (128, 48), (128, 512), (-64, 16)])
def test_block_bytes_refuses_other_formats(L, d, p):
    assert L.sx_kv4_block_bytes(d, p) == 0


BAD_CACHES = [
    (dict(pool=None), "SX_ERR_NULL_POINTER"),
    (dict(pool=FAKE + 8), "SX_ERR_BAD_SHAPE"),
    (dict(pages=0), "SX_ERR_BAD_SHAPE"),
    (dict(kv_heads=0), "SX_ERR_BAD_SHAPE"),
    (dict(head_dim=96), "SX_ERR_BAD_SHAPE"),
    (dict(page_size=24), "SX_ERR_BAD_SHAPE"),
]


def attention(L, c=None, q=FAKE, dtype=2, tokens=3, heads=8, cu=FAKE, kv=FAKE, table=FAKE, requests=2, width=4, stride=4,
              max_q=2, scale=0.1, window=0, out=FAKE, ws=FAKE, nbytes=1 << 40):
    c = cache() if c is None else c
    return name(L, L.sx_kv4_attention(None, ctypes.byref(c), q, heads * 128, 128, dtype, tokens, heads, cu, kv, table,
                                      requests, width, stride, max_q, scale, window, out, ws, nbytes))


@pytest.mark.parametrize("kw,want", BAD_CACHES)
def test_cache_refusals(L, kw, want):
    c = cache(**kw)
    assert attention(L, c) == want
    assert name(L, L.sx_kv4_write(None, ctypes.byref(c), FAKE, 256, 128, FAKE, 256, 128, 2, 3, FAKE)) == want
    assert name(L, L.sx_kv4_read(None, ctypes.byref(c), FAKE, 3, 2, FAKE, FAKE)) == want


@pytest.mark.parametrize(
    "kw,want",
    [
        (dict(dtype=0), "SX_ERR_BAD_DTYPE"),
        (dict(dtype=9), "SX_ERR_BAD_DTYPE"),
        (dict(tokens=-1), "SX_ERR_BAD_SHAPE"),
        (dict(heads=0), "SX_ERR_BAD_SHAPE"),
        (dict(heads=7), "SX_ERR_BAD_SHAPE"),
        (dict(requests=0), "SX_ERR_BAD_SHAPE"),
        (dict(requests=16385), "SX_ERR_BAD_SHAPE"),
        (dict(width=0), "SX_ERR_BAD_SHAPE"),
        (dict(stride=3), "SX_ERR_BAD_SHAPE"),
        (dict(requests=1 << 14, width=1 << 20, stride=1 << 20), "SX_ERR_BAD_SHAPE"),
        (dict(requests=1 << 20, width=1 << 10, stride=1 << 10), "SX_ERR_BAD_SHAPE"),
        (dict(max_q=0), "SX_ERR_BAD_SHAPE"),
        (dict(window=-1), "SX_ERR_BAD_SHAPE"),
        (dict(scale=float("nan")), "SX_ERR_BAD_SHAPE"),
        (dict(scale=float("inf")), "SX_ERR_BAD_SHAPE"),
        (dict(q=None), "SX_ERR_NULL_POINTER"),
        (dict(cu=None), "SX_ERR_NULL_POINTER"),
        (dict(kv=None), "SX_ERR_NULL_POINTER"),
        (dict(table=None), "SX_ERR_NULL_POINTER"),
        (dict(out=None), "SX_ERR_NULL_POINTER"),
        (dict(ws=None), "SX_ERR_NULL_POINTER"),
        (dict(ws=FAKE + 8), "SX_ERR_BAD_SHAPE"),
        (dict(out=FAKE + 2), "SX_ERR_BAD_SHAPE"),
        (dict(nbytes=1), "SX_ERR_WORKSPACE_TOO_SMALL"),
        (dict(tokens=0, q=None), "SX_OK"),
    ],
)
def test_attention_refusals(L, kw, want):
    assert attention(L, **kw) == want


@pytest.mark.parametrize(
    "args,want",
    [
        ((None, 256, 128, FAKE, 256, 128, 2, 3, FAKE), "SX_ERR_NULL_POINTER"),
        ((FAKE, 256, 128, None, 256, 128, 2, 3, FAKE), "SX_ERR_NULL_POINTER"),
        ((FAKE, 256, 128, FAKE, 256, 128, 2, 3, None), "SX_ERR_NULL_POINTER"),
        ((FAKE, 256, 128, FAKE, 256, 128, 5, 3, FAKE), "SX_ERR_BAD_DTYPE"),
        ((FAKE, 256, 128, FAKE, 256, 128, 2, -3, FAKE), "SX_ERR_BAD_SHAPE"),
        ((None, 256, 128, None, 256, 128, 2, 0, None), "SX_OK"),
    ],
)
def test_write_refusals(L, args, want):
    c = cache()
    assert name(L, L.sx_kv4_write(None, ctypes.byref(c), *args)) == want


@pytest.mark.parametrize(
    "args,want",
    [
        ((None, 3, 2, FAKE, FAKE), "SX_ERR_NULL_POINTER"),
        ((FAKE, 3, 2, FAKE, None), "SX_ERR_NULL_POINTER"),
        ((FAKE, 3, 4, FAKE, FAKE), "SX_ERR_BAD_DTYPE"),
        ((FAKE, -1, 2, FAKE, FAKE), "SX_ERR_BAD_SHAPE"),
        ((None, 0, 2, None, None), "SX_OK"),
    ],
)
def test_read_refusals(L, args, want):
    c = cache()
    assert name(L, L.sx_kv4_read(None, ctypes.byref(c), *args)) == want


def tables(L, ctx=FAKE, new=FAKE, requests=2, page=16, table=FAKE, width=4, stride=4, free=FAKE, count=FAKE, tokens=3,
           outs=(FAKE,) * 5):
    return name(L, L.sx_block_tables(None, ctx, new, requests, page, table, width, stride, free, count, tokens, *outs))


@pytest.mark.parametrize(
    "kw,want",
    [
        (dict(ctx=None), "SX_ERR_NULL_POINTER"),
        (dict(new=None), "SX_ERR_NULL_POINTER"),
        (dict(table=None), "SX_ERR_NULL_POINTER"),
        (dict(free=None), "SX_ERR_NULL_POINTER"),
        (dict(count=None), "SX_ERR_NULL_POINTER"),
        (dict(outs=(FAKE, FAKE, None, FAKE, FAKE)), "SX_ERR_NULL_POINTER"),
        (dict(outs=(FAKE, FAKE, FAKE, FAKE, None)), "SX_ERR_NULL_POINTER"),
        (dict(requests=0), "SX_ERR_BAD_SHAPE"),
        (dict(requests=16385), "SX_ERR_BAD_SHAPE"),
        (dict(page=20), "SX_ERR_BAD_SHAPE"),
        (dict(width=0), "SX_ERR_BAD_SHAPE"),
        (dict(stride=3), "SX_ERR_BAD_SHAPE"),
        (dict(tokens=-1), "SX_ERR_BAD_SHAPE"),
    ],
)
def test_block_tables_refusals(L, kw, want):
    assert tables(L, **kw) == want


def test_the_python_calls_refuse_by_name():
    import torch

    import sushi_b200 as sx

    with pytest.raises(sx.Exl3Error, match="SX_ERR_BAD_SHAPE"):
        sx.Kv4Cache(4, 2, 96)
    with pytest.raises(sx.Exl3Error, match="SX_ERR_BAD_SHAPE"):
        sx.Kv4Cache(4, 2, 128, 24)
    with pytest.raises(sx.Exl3Error, match="SX_ERR_BAD_DTYPE"):
        sx.Kv4Cache(4, 2, 128, 16, pool=torch.zeros(4))
    with pytest.raises(sx.Exl3Error, match="SX_ERR_BAD_SHAPE"):  # a host tensor
        sx.Kv4Cache(4, 2, 128, 16, pool=torch.zeros(4 * 2 * 2304, dtype=torch.uint8))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(sx.Exl3Error, match="SX_ERR_BAD_SHAPE"):
        sx.block_tables(i, i, i.reshape(2, 1), i, i[:1], 16, 2)
    with pytest.raises(sx.Exl3Error, match="SX_ERR_BAD_DTYPE"):
        sx.block_tables(i.float(), i, i.reshape(2, 1), i, i[:1], 16, 2)
