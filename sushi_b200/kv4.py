"""The 4-bit key/value cache of a serving step: block tables, writes and reads, attention.

    t = block_tables(ctx_lens, new_lens, table, free_pages, free_count, cache.page_size, tokens)
    kv4_write(cache, k, v, t.slots)                      # k, v: the step's keys and values
    out = kv4_attention(q, cache, table, t.kv_lens, t.cu_q, max_q)

The reference serves attention from its own host engine and has no counterpart of these calls; names,
checks and errors are those of the rest of the package.  Everything is ordered on the current
stream, allocates nothing but its outputs (and the attention's workspace, once a stream) and can be
recorded in a CUDA graph.
"""

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .exl3 import _DT, Exl3Error, _check, _stream, lib


class Kv4Cache:
    """A pool of pages for one layer's keys and values in 4 bits (sx_kv4): `pages` pages of
    `page_size` tokens (16, 32, 64, 128 or 256) of `kv_heads` heads of `head_dim` (64, 128 or 256)
    channels.  `pool`: an optional uint8 tensor to use, [pages, kv_heads, block_bytes]."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda", pool=None):
        block = lib().sx_kv4_block_bytes(int(head_dim), int(page_size))
        if block == 0 or pages < 1 or kv_heads < 1:
            raise Exl3Error(1)
        self.pages, self.kv_heads, self.head_dim, self.page_size = int(pages), int(kv_heads), int(head_dim), int(page_size)
        if pool is None:
            pool = torch.empty((self.pages, self.kv_heads, block), dtype=torch.uint8, device=device)
        elif pool.dtype != torch.uint8:
            raise Exl3Error(2)
        elif pool.numel() != self.pages * self.kv_heads * block or not pool.is_contiguous() or not pool.is_cuda:
            raise Exl3Error(1)
        self.pool = pool

    def c(self):
        return _lib.SxKv4(self.pool.data_ptr(), self.pages, self.kv_heads, self.head_dim, self.page_size)


class BlockTables(NamedTuple):
    """block_tables' outputs (sx_block_tables)."""

    kv_lens: torch.Tensor    # [requests] int32
    cu_q: torch.Tensor       # [requests + 1] int32
    slots: torch.Tensor      # [tokens] int64
    positions: torch.Tensor  # [tokens] int32
    free_left: torch.Tensor  # [1] int32


def _ints(t, n=None, dtype=torch.int32):
    if t.dtype != dtype:
        raise Exl3Error(2)
    if not t.is_cuda or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise Exl3Error(1)
    return t.data_ptr()


def _table(table, requests):
    if table.dtype != torch.int32:
        raise Exl3Error(2)
    if not table.is_cuda or table.dim() != 2 or table.shape[0] != requests or table.shape[1] < 1 or table.stride(1) != 1:
        raise Exl3Error(1)
    return table.data_ptr(), table.shape[1], max(table.stride(0), table.shape[1]) if requests == 1 else table.stride(0)


def block_tables(ctx_lens, new_lens, table, free_pages, free_count, page_size: int, tokens: int) -> BlockTables:
    """sx_block_tables: the step's table entries (written into `table` [requests, width] int32, in
    place), places and positions of its `tokens` tokens, lengths and row offsets, from the cached and
    new lengths [requests] int32 and the stack free_pages [n] int32 / free_count [1] int32.  The new
    stack height is `free_left` (negative: pages were short)."""
    requests = ctx_lens.numel()
    c, n = _ints(ctx_lens), _ints(new_lens, requests)
    t, width, stride = _table(table, requests)
    f, fc = _ints(free_pages), _ints(free_count, 1)
    i32 = dict(dtype=torch.int32, device=ctx_lens.device)
    tokens = int(tokens)
    if tokens < 0:
        raise Exl3Error(1)
    out = BlockTables(torch.empty(requests, **i32), torch.empty(requests + 1, **i32),
                      torch.empty(tokens, dtype=torch.int64, device=ctx_lens.device), torch.empty(tokens, **i32),
                      torch.empty(1, **i32))
    _check(lib().sx_block_tables(_stream(), c, n, requests, int(page_size), t, width, stride, f, fc, tokens,
                                 *(x.data_ptr() for x in out)))
    return out


def _rows(x, heads, head_dim):
    if x.dtype not in _DT:
        raise Exl3Error(2)
    if not x.is_cuda or x.dim() != 3 or x.shape[1] != heads or x.shape[2] != head_dim or x.stride(2) != 1:
        raise Exl3Error(1)
    return x.data_ptr(), x.stride(0), x.stride(1)


def kv4_write(cache: Kv4Cache, k, v, slots):
    """sx_kv4_write: k and v [tokens, kv_heads, head_dim] (bf16/f16/f32; channels contiguous, any
    strides between tokens and heads) into the places slots [tokens] int64; -1 skips a token."""
    kp, vp = _rows(k, cache.kv_heads, cache.head_dim), _rows(v, cache.kv_heads, cache.head_dim)
    if v.dtype != k.dtype:
        raise Exl3Error(2)
    if v.shape[0] != k.shape[0]:
        raise Exl3Error(1)
    s = _ints(slots, k.shape[0], torch.int64)
    c = cache.c()
    _check(lib().sx_kv4_write(_stream(), ctypes.byref(c), *kp, *vp, _DT[k.dtype], k.shape[0], s))


def kv4_read(cache: Kv4Cache, slots, dtype=torch.bfloat16):
    """sx_kv4_read: the keys and values held in the places slots [tokens] int64, rounded to `dtype`:
    two [tokens, kv_heads, head_dim] tensors (zeros where a slot is -1)."""
    if dtype not in _DT:
        raise Exl3Error(2)
    s = _ints(slots, dtype=torch.int64)
    n = slots.numel()
    k = torch.empty((n, cache.kv_heads, cache.head_dim), dtype=dtype, device=slots.device)
    v = torch.empty_like(k)
    c = cache.c()
    _check(lib().sx_kv4_read(_stream(), ctypes.byref(c), s, n, _DT[dtype], k.data_ptr(), v.data_ptr()))
    return k, v


def kv4_attention_workspace_bytes(cache: Kv4Cache, requests: int, tokens: int, heads: int, max_q: int) -> int:
    c = cache.c()
    return lib().sx_kv4_attention_workspace_bytes(ctypes.byref(c), int(requests), int(tokens), int(heads), int(max_q))


_WS = {}


def _workspace(nbytes, device):
    """The zeroed workspace of the current stream (every call leaves it zeroed, so it is kept).  While
    a graph is being recorded a fresh one is made inside it: memory the recording only plans to zero
    must not serve calls outside."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _WS.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = _WS[key] = torch.zeros(nbytes, dtype=torch.uint8, device=device)
    return ws


def kv4_attention(q, cache: Kv4Cache, table, kv_lens, cu_q, max_q: int, scale=None, window: int = 0, out=None,
                  workspace=None):
    """sx_kv4_attention: q [tokens, heads, head_dim] (bf16/f16; channels contiguous) over the cache.
    Request b's rows are cu_q[b]..cu_q[b+1] (at most max_q), its keys the kv_lens[b] tokens its row
    of `table` [requests, width] names, the step's own last; causal, with a sliding window of
    `window` positions when it is positive.  scale: head_dim**-0.5 when None.  out: an optional
    contiguous tensor of q's shape and dtype.  workspace: an optional zeroed uint8 tensor of
    kv4_attention_workspace_bytes(...) bytes, reused across calls on one stream."""
    if q.dim() != 3:
        raise Exl3Error(1)
    qp, ts, hs = _rows(q, q.shape[1], cache.head_dim)
    requests = kv_lens.numel()
    kl, cu = _ints(kv_lens), _ints(cu_q, requests + 1)
    t, width, stride = _table(table, requests)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise Exl3Error(1)
    c = cache.c()
    need = lib().sx_kv4_attention_workspace_bytes(ctypes.byref(c), requests, q.shape[0], q.shape[1], int(max_q))
    ws = workspace if workspace is not None else _workspace(max(need, 16), q.device)
    _check(lib().sx_kv4_attention(_stream(), ctypes.byref(c), qp, ts, hs, _DT[q.dtype], q.shape[0], q.shape[1], cu, kl, t,
                                  requests, width, stride, int(max_q), cache.head_dim ** -0.5 if scale is None else float(scale),
                                  int(window), out.data_ptr(), ws.data_ptr(), ws.numel()))
    return out
