"""The 4-bit key/value cache of a serving step: block tables, writes and reads, attention.

    t = block_tables(ctx_lens, new_lens, table, free_pages, free_count, cache.page_size, tokens)
    kv4_write(cache, k, v, t.slots)                      # k, v: the step's keys and values
    out = kv4_attention(q, cache, table, t.kv_lens, t.cu_q, max_q)

The reference serves attention from its own host engine and has no counterpart of these calls; names,
checks and errors are those of the rest of the package.  A call's tensors lie on one GPU, the
cache's (SX_ERR_BAD_SHAPE otherwise).  Everything is ordered on that GPU's current stream, allocates
nothing but its outputs (and the attention's workspace, once a stream) and can be recorded in a CUDA
graph.
"""

import contextlib
import ctypes
import threading
from typing import NamedTuple

import torch

from . import _lib
from .exl3 import _DT, Exl3Error, _check, lib

_I32, _I64, _U8 = torch.int32, torch.int64, torch.uint8


def _stream(gpu):
    """The current stream's handle on GPU number `gpu` (as an int: no Stream object a call)."""
    return torch._C._cuda_getCurrentRawStream(gpu)


_HERE = contextlib.nullcontext()


def _current(gpu):
    """GPU number `gpu` as the current one, where launches and allocations go."""
    return _HERE if torch._C._cuda_getDevice() == gpu else torch.cuda.device(gpu)


def _int(v):
    """v as the library's 32-bit integers hold it; refused past them (ctypes would cut it)."""
    v = int(v)
    if not -(1 << 31) <= v < 1 << 31:
        raise Exl3Error(1)
    return v


class Kv4Cache:
    """A pool of pages for one layer's keys and values in 4 bits (sx_kv4): `pages` pages of
    `page_size` tokens (16, 32, 64, 128 or 256) of `kv_heads` heads of `head_dim` (64, 128 or 256)
    channels.  `pool`: an optional uint8 tensor to use, [pages, kv_heads, block_bytes]."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda", pool=None):
        pages, kv_heads, head_dim, page_size = _int(pages), _int(kv_heads), _int(head_dim), _int(page_size)
        block = lib().sx_kv4_block_bytes(head_dim, page_size)
        if block == 0 or pages < 1 or kv_heads < 1:
            raise Exl3Error(1)
        self.pages, self.kv_heads, self.head_dim, self.page_size = pages, kv_heads, head_dim, page_size
        if pool is None:
            pool = torch.empty((self.pages, self.kv_heads, block), dtype=torch.uint8, device=device)
        elif pool.dtype != torch.uint8:
            raise Exl3Error(2)
        if pool.numel() != self.pages * self.kv_heads * block or not pool.is_contiguous() or not pool.is_cuda:
            raise Exl3Error(1)
        self.pool, self.gpu = pool, pool.get_device()
        self._c = _lib.SxKv4(pool.data_ptr(), self.pages, self.kv_heads, self.head_dim, self.page_size)
        self._ref = ctypes.byref(self._c)

    def c(self):
        return self._c


class BlockTables(NamedTuple):
    """block_tables' outputs (sx_block_tables)."""

    kv_lens: torch.Tensor    # [requests] int32
    cu_q: torch.Tensor       # [requests + 1] int32
    slots: torch.Tensor      # [tokens] int64
    positions: torch.Tensor  # [tokens] int32
    free_left: torch.Tensor  # [1] int32


def _ints(t, gpu, n=None, dtype=_I32):
    if t.dtype is not dtype:
        raise Exl3Error(2)
    if t.get_device() != gpu or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise Exl3Error(1)
    return t.data_ptr()


def _table(table, gpu, requests):
    if table.dtype is not _I32:
        raise Exl3Error(2)
    if table.get_device() != gpu or table.dim() != 2:
        raise Exl3Error(1)
    (rows, width), (stride, inner) = table.shape, table.stride()
    if rows != requests or width < 1 or (inner != 1 and width > 1):
        raise Exl3Error(1)
    return table.data_ptr(), width, max(stride, width) if rows == 1 else stride


def block_tables(ctx_lens, new_lens, table, free_pages, free_count, page_size: int, tokens: int) -> BlockTables:
    """sx_block_tables: the step's table entries (written into `table` [requests, width] int32, in
    place), places and positions of its `tokens` tokens, lengths and row offsets, from the cached and
    new lengths [requests] int32 and the stack free_pages [n] int32 / free_count [1] int32.  The new
    stack height is `free_left` (negative: pages were short)."""
    requests = ctx_lens.numel()
    gpu = max(ctx_lens.get_device(), 0)  # a host tensor (-1) is refused like one of another GPU
    c, n = _ints(ctx_lens, gpu), _ints(new_lens, gpu, requests)
    t, width, stride = _table(table, gpu, requests)
    f, fc = _ints(free_pages, gpu), _ints(free_count, gpu, 1)
    tokens, page_size = _int(tokens), _int(page_size)
    if tokens < 0:
        raise Exl3Error(1)
    with _current(gpu):
        # one buffer for the five outputs: slots (64-bit) first
        buf = ctx_lens.new_empty(3 * tokens + 2 * requests + 2)
        slots, positions, kv_lens, cu_q, left = buf.split_with_sizes([2 * tokens, tokens, requests, requests + 1, 1])
        p = buf.data_ptr()
        _check(lib().sx_block_tables(_stream(gpu), c, n, requests, page_size, t, width, stride, f, fc, tokens,
                                     p + 12 * tokens, p + 12 * tokens + 4 * requests, p, p + 8 * tokens,
                                     p + 12 * tokens + 8 * requests + 4))
    return BlockTables(kv_lens, cu_q, slots.view(_I64), positions, left)


def _rows(x, gpu, heads, head_dim):
    if x.dtype not in _DT:
        raise Exl3Error(2)
    if x.get_device() != gpu or x.dim() != 3:
        raise Exl3Error(1)
    (_, h, d), (ts, hs, inner) = x.shape, x.stride()
    if h != heads or d != head_dim or inner != 1:
        raise Exl3Error(1)
    return x.data_ptr(), ts, hs


def kv4_write(cache: Kv4Cache, k, v, slots):
    """sx_kv4_write: k and v [tokens, kv_heads, head_dim] (bf16/f16/f32; channels contiguous, any
    strides between tokens and heads) into the places slots [tokens] int64; -1 skips a token."""
    gpu = cache.gpu
    kp, vp = _rows(k, gpu, cache.kv_heads, cache.head_dim), _rows(v, gpu, cache.kv_heads, cache.head_dim)
    if v.dtype != k.dtype:
        raise Exl3Error(2)
    if v.shape[0] != k.shape[0]:
        raise Exl3Error(1)
    tokens = k.shape[0]
    s = _ints(slots, gpu, tokens, _I64)
    with _current(gpu):
        _check(lib().sx_kv4_write(_stream(gpu), cache._ref, *kp, *vp, _DT[k.dtype], tokens, s))


def kv4_read(cache: Kv4Cache, slots, dtype=torch.bfloat16):
    """sx_kv4_read: the keys and values held in the places slots [tokens] int64, rounded to `dtype`:
    two [tokens, kv_heads, head_dim] tensors (zeros where a slot is -1)."""
    if dtype not in _DT:
        raise Exl3Error(2)
    gpu = cache.gpu
    s = _ints(slots, gpu, dtype=_I64)
    n = slots.numel()
    with _current(gpu):
        kv = slots.new_empty((2, n, cache.kv_heads, cache.head_dim), dtype=dtype)
        k, v = kv.unbind()
        _check(lib().sx_kv4_read(_stream(gpu), cache._ref, s, n, _DT[dtype], k.data_ptr(), v.data_ptr()))
    return k, v


def kv4_attention_workspace_bytes(cache: Kv4Cache, requests: int, tokens: int, heads: int, max_q: int) -> int:
    return lib().sx_kv4_attention_workspace_bytes(cache._ref, _int(requests), _int(tokens), _int(heads), _int(max_q))


class _Kept:
    """A stream's workspace, kept for its next calls.  A call is several launches, the later ones reading what
    the first left in the workspace: `lock` keeps another host thread's launches on the stream from coming
    between them."""

    def __init__(self):
        self.lock, self.buffer = threading.Lock(), None

    def grown(self, nbytes, device):
        if self.buffer is None or self.buffer.numel() < nbytes:
            self.buffer = torch.empty(nbytes, dtype=_U8, device=device)
        return self.buffer


_WS = {}  # (GPU, stream) -> _Kept


def kv4_attention(q, cache: Kv4Cache, table, kv_lens, cu_q, max_q: int, scale=None, window: int = 0, out=None,
                  workspace=None):
    """sx_kv4_attention: q [tokens, heads, head_dim] (bf16/f16; channels contiguous) over the cache.
    Request b's rows are cu_q[b]..cu_q[b+1] (at most max_q; a longer request's may come out NaN), its
    keys the kv_lens[b] tokens its row of `table` [requests, width] names, the step's own last; causal,
    with a sliding window of `window` positions when it is positive.  scale: head_dim**-0.5 when None.  out: an optional
    contiguous tensor of q's shape and dtype.  workspace: an optional uint8 tensor of
    kv4_attention_workspace_bytes(...) bytes, for the calls of one stream by one host thread (without
    it, several threads may call on one stream)."""
    if q.dim() != 3:
        raise Exl3Error(1)
    tokens, heads, _ = q.shape
    max_q, window = _int(max_q), _int(min(window, (1 << 31) - 1))  # a window wider than any cache is none
    gpu = cache.gpu
    qp, ts, hs = _rows(q, gpu, heads, cache.head_dim)
    requests = kv_lens.numel()
    kl, cu = _ints(kv_lens, gpu), _ints(cu_q, gpu, requests + 1)
    t, width, stride = _table(table, gpu, requests)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.get_device() != gpu):
        raise Exl3Error(1)
    if workspace is not None:
        if workspace.dtype is not _U8:
            raise Exl3Error(2)
        if workspace.get_device() != gpu or not workspace.is_contiguous():
            raise Exl3Error(1)
    with _current(gpu):
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        L, st, lock = lib(), _stream(gpu), _HERE
        if workspace is None:
            need = max(L.sx_kv4_attention_workspace_bytes(cache._ref, requests, tokens, heads, max_q), 16)
            if torch.cuda.is_current_stream_capturing():
                workspace = torch.empty(need, dtype=_U8, device=q.device)  # the recorded graph's own
            else:
                kept = _WS.get((gpu, st)) or _WS.setdefault((gpu, st), _Kept())
                lock = kept.lock
        with lock:
            if lock is not _HERE:
                workspace = kept.grown(need, q.device)
            _check(L.sx_kv4_attention(st, cache._ref, qp, ts, hs, _DT[q.dtype], tokens, heads, cu, kl, t, requests, width,
                                      stride, max_q, cache.head_dim ** -0.5 if scale is None else scale, window,
                                      out.data_ptr(), workspace.data_ptr(), workspace.numel()))
    return out
