"""What the Python calls of the 4-bit cache let through to the library (no GPU): tensors that say they are on
a GPU, and a library that records its calls."""

import contextlib
import threading
import time

import pytest
import torch

from sushi_b200 import Exl3Error, kv4


class OnGpu:
    """A host tensor that answers as one of GPU number `gpu` (-1: as the host tensor it is)."""

    def __init__(self, t, gpu=0):
        self.t, self.gpu, self.is_cuda = t, gpu, gpu >= 0

    def get_device(self):
        return self.gpu

    def __getattr__(self, name):
        return getattr(self.t, name)


class Recorder:
    """The library's calls: name, arguments and the current GPU at the time of each."""

    def __init__(self):
        self.calls, self.current = [], [0]

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *a: 64
        return lambda *a: self.calls.append((name, a, self.current[-1])) or 0


@pytest.fixture
def rec(monkeypatch):
    r = Recorder()

    @contextlib.contextmanager
    def device(gpu):
        r.current.append(gpu)
        yield
        r.current.pop()

    monkeypatch.setattr(kv4, "_WS", {})
    monkeypatch.setattr(kv4, "_stream", lambda device: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: r.current[-1], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    r.real = kv4.lib
    return r


def cache(rec, monkeypatch, gpu=0):
    c = kv4.Kv4Cache(3, 2, 64, 16, pool=OnGpu(torch.zeros(3 * 2 * 16 * 72, dtype=torch.uint8), gpu))
    monkeypatch.setattr(kv4, "lib", lambda: rec)
    return c


def tensors(gpu=0):
    i = lambda *s: OnGpu(torch.zeros(s, dtype=torch.int32), gpu)
    x = lambda h: OnGpu(torch.zeros((2, h, 64), dtype=torch.bfloat16), gpu)
    return dict(q=x(4), table=i(2, 3), kv_lens=i(2), cu_q=i(3), out=x(4), workspace=OnGpu(torch.zeros(64, dtype=torch.uint8), gpu),
                k=x(2), v=x(2), slots=OnGpu(torch.zeros(2, dtype=torch.int64), gpu), ctx=i(2), new=i(2), free=i(4), count=i(1))


def attend(c, t, max_q=1, **kw):
    return kv4.kv4_attention(t["q"], c, t["table"], t["kv_lens"], t["cu_q"], max_q, out=t["out"], workspace=t["workspace"], **kw)


CALLS = {
    "attention": (attend, ["q", "table", "kv_lens", "cu_q", "out", "workspace"]),
    "write": (lambda c, t: kv4.kv4_write(c, t["k"], t["v"], t["slots"]), ["k", "v", "slots"]),
    "read": (lambda c, t: kv4.kv4_read(c, t["slots"]), ["slots"]),
    "tables": (lambda c, t: kv4.block_tables(t["ctx"], t["new"], t["table"], t["free"], t["count"], 16, 2),
               ["ctx", "new", "table", "free", "count"]),
}


@pytest.mark.parametrize("elsewhere", [-1, 1])  # on the host, on another GPU
@pytest.mark.parametrize("call,name", [(c, n) for c, (_, names) in CALLS.items() for n in names])
def test_a_tensor_elsewhere_is_refused_before_any_launch(rec, monkeypatch, call, name, elsewhere):
    c, t = cache(rec, monkeypatch), tensors()
    CALLS[call][0](c, t)
    assert len(rec.calls) == 1
    t[name] = OnGpu(t[name].t, elsewhere)
    with pytest.raises(Exl3Error, match="SX_ERR_BAD_SHAPE"):
        CALLS[call][0](c, t)
    assert len(rec.calls) == 1


def test_a_workspace_of_another_type_or_with_gaps_is_refused(rec, monkeypatch):
    c, t = cache(rec, monkeypatch), tensors()
    t["workspace"] = OnGpu(torch.zeros(64))
    with pytest.raises(Exl3Error, match="SX_ERR_BAD_DTYPE"):
        attend(c, t)
    t["workspace"] = OnGpu(torch.zeros(128, dtype=torch.uint8)[::2])
    with pytest.raises(Exl3Error, match="SX_ERR_BAD_SHAPE"):
        attend(c, t)
    assert not rec.calls


@pytest.mark.parametrize("call", list(CALLS))
def test_a_call_runs_on_its_tensors_gpu(rec, monkeypatch, call):
    c = cache(rec, monkeypatch, gpu=1)
    CALLS[call][0](c, tensors(gpu=1))
    assert [at for _, _, at in rec.calls] == [1] and rec.current == [0]


def test_a_cache_on_the_host_is_refused():
    with pytest.raises(Exl3Error, match="SX_ERR_BAD_SHAPE"):
        kv4.Kv4Cache(3, 2, 64, 16, device="cpu")


def test_calls_of_two_threads_on_one_stream_do_not_share_a_workspace_at_a_time(rec, monkeypatch):
    """A call is several launches that pass partial results through the workspace: no other call may be
    under way with it."""
    c, busy, clashes = cache(rec, monkeypatch), set(), []

    def launches(*args):
        ws = args[-2]
        clashes.extend([ws] if ws in busy else [])
        busy.add(ws)
        time.sleep(0.02)
        busy.discard(ws)
        return 0

    rec.sx_kv4_attention = launches
    start = threading.Barrier(4)

    def thread():
        t = tensors()
        t["q"].device = torch.device("cpu")
        start.wait()
        for _ in range(3):
            kv4.kv4_attention(t["q"], c, t["table"], t["kv_lens"], t["cu_q"], 1, out=t["out"])

    threads = [threading.Thread(target=thread) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not clashes


@pytest.mark.parametrize("scale,want", [(2.0 ** 100, "SX_ERR_BAD_SHAPE"), (-3e38, "SX_ERR_BAD_SHAPE"), (2.0 ** 99, "SX_OK"), (0.0, "SX_OK")])
def test_scales(scale, want):
    from test_kv4_host import attention

    assert attention(kv4._lib.load(), tokens=0, scale=scale) == want


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("max_q", [1, 16, 4096])
def test_the_stated_size_of_a_call_is_admitted(head_dim, max_q):
    """requests * kv_heads * table_width * page_size / 2 just below 2^31, in a few shapes; eight times that is refused
    where a request may have many rows."""
    from test_kv4_host import attention, cache

    L = kv4._lib.load()
    for requests, width in ((16, (1 << 32) // (16 * 2 * 64) - 64), (4096, (1 << 32) // (4096 * 2 * 64) - 64)):
        c = cache(head_dim=head_dim)
        assert attention(L, c, tokens=0, requests=requests, width=width, stride=width, max_q=max_q) == "SX_OK"
        if max_q == 4096:
            assert attention(L, c, tokens=0, requests=requests, width=8 * width, stride=8 * width, max_q=max_q) == "SX_ERR_BAD_SHAPE"


def test_integers_past_32_bits_are_refused_or_none(rec, monkeypatch):
    c, t = cache(rec, monkeypatch), tensors()
    attend(c, t, window=(1 << 32) + 16)  # wider than any cache: no window, and not one of 16
    assert rec.calls[-1][1][-4] == (1 << 31) - 1
    past = (1 << 32) + 16
    for call in (lambda: attend(c, t, max_q=past), lambda: attend(c, t, window=-past),
                 lambda: kv4.block_tables(t["ctx"], t["new"], t["table"], t["free"], t["count"], past, 2),
                 lambda: kv4.Kv4Cache(1, 1, 64, past), lambda: kv4.kv4_attention_workspace_bytes(c, 1, 1, 1, past)):
        with pytest.raises(Exl3Error, match="SX_ERR_BAD_SHAPE"):
            call()
    assert len(rec.calls) == 1
