"""Threads that share a device's context: a call runs on its own thread's stream
from beginning to end.  A fake library, no GPU."""
import threading
import time

import pytest

from browsergnn_b200 import _lib, backend

STREAM = threading.local()  # what torch's current stream is of a thread


class FakeLib:
    """Records the stream at the start and at the end of each call."""

    def __init__(self):
        self.stream = None
        self.seen = []
        self.inside = 0
        self.together = 0

    def bgnn_ctx_set_stream(self, h, s):
        self.stream = s
        return 0

    def work(self, h, mine):
        self.inside += 1
        self.together = max(self.together, self.inside)
        first = self.stream
        time.sleep(0.002)  # ctypes drops the interpreter's lock in here
        self.seen.append((mine, first, self.stream))
        self.inside -= 1
        return 0

    bgnn_ctx_synchronize = lambda self, h: self.work(h, STREAM.s)

    def on_handle(self, mine):
        return self.work(None, mine)


@pytest.fixture
def ctx(monkeypatch):
    """A context over the fake library, made by the class's own constructor."""
    import torch

    lib = FakeLib()
    lib.bgnn_ctx_create = lambda device, out: 0
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: Device.current)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: STREAM.s,
                        raising=False)
    return backend.CudaContext(0)


class Device:
    """torch.cuda.device over a fake current device."""

    current = 0

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before, Device.current = Device.current, self.index

    def __exit__(self, *exc):
        Device.current = self.before


def test_a_new_context_leaves_the_current_device(ctx, monkeypatch):
    """A first call with tensors of another device than the current one."""
    made = []

    def create(device, out):
        made.append(device)
        Device.current = device  # as cudaSetDevice in the library does
        return 0

    monkeypatch.setattr(ctx.lib, "bgnn_ctx_create", create)
    monkeypatch.setattr(Device, "current", 0)
    assert backend.CudaContext(1).device == 1
    assert made == [1] and Device.current == 0
    monkeypatch.setattr(ctx.lib, "bgnn_ctx_create", lambda device, out: 3)  # no such device
    monkeypatch.setattr(_lib, "check", lambda rc, h=None: (_ for _ in ()).throw(RuntimeError(rc)))
    with pytest.raises(RuntimeError, match="3"):
        backend.CudaContext(99)
    assert Device.current == 0


@pytest.mark.parametrize("how", ["call", "call_on", "synchronize"])
def test_a_call_keeps_its_threads_stream(ctx, how):
    def run(s):
        STREAM.s = s
        for _ in range(20):
            if how == "call":
                ctx.call("work", s)
            elif how == "call_on":
                ctx.call_on("on_handle", s)
            else:
                ctx.synchronize()

    threads = [threading.Thread(target=run, args=(s,)) for s in (11, 22, 33)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(ctx.lib.seen) == 60
    assert all(mine == first == last for mine, first, last in ctx.lib.seen)
    assert ctx.lib.together == 1


def test_a_failing_call_frees_the_context(ctx):
    STREAM.s = 5
    ctx.lib.fails = lambda h: 1
    ctx.lib.bgnn_last_error = lambda h: b"no"
    with pytest.raises(backend._lib.BGNNError, match="no"):
        ctx.call("fails")
    t = threading.Thread(target=lambda: (setattr(STREAM, "s", 6), ctx.call("work", 6)), daemon=True)
    t.start()
    t.join(10)
    assert ctx.lib.seen == [(6, 6, 6)]


def test_one_context_for_threads_that_ask_at_once(monkeypatch):
    made = []

    class Slow:
        def __init__(self, device):
            time.sleep(0.02)
            made.append(device)

    monkeypatch.setattr(backend, "CudaContext", Slow)
    monkeypatch.setattr(backend, "_contexts", {})
    got = []
    threads = [threading.Thread(target=lambda: got.append(backend.get_context(3))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert made == [3] and len(set(map(id, got))) == 1
