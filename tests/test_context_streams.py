"""How a Context follows torch's streams, on fakes of both (no GPU): which streams wait for which, that a
caller's own stream is not touched after it is gone, and that threads do not change each other's stream
between setting it and launching on it."""
import contextlib
import threading
import time
import types

import pytest
import torch

from wuxianhuabu_b200 import _lib, h3


class World:
    """Streams (some torch's own, some a caller's), events and the library, with what happened to them."""

    def __init__(self, monkeypatch):
        self.log, self.local, self.default = [], threading.local(), FakeStream(self, 0, "default")
        monkeypatch.setattr(h3, "_current_raw_stream", lambda device: self.current().cuda_stream)
        monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.current())
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.current().touch().capturing is not None)
        monkeypatch.setattr(torch.cuda, "stream", self.on)
        monkeypatch.setattr(torch.cuda, "set_stream", lambda s: setattr(self.local, "s", s))
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
        monkeypatch.setattr(torch.cuda, "Event", lambda *a, **k: FakeEvent(self))
        monkeypatch.setattr(_lib, "load", lambda: self.lib)
        self.stream = None  # of the library's context
        self.lib = types.SimpleNamespace(wx_ctx_create=lambda d, h: 0, wx_ctx_set_stream=self._set, work=self._work,
                                         wx_ctx_check_device=self._check, wx_last_error=lambda h: b"")

    def current(self):
        return getattr(self.local, "s", self.default)

    @contextlib.contextmanager
    def on(self, s):
        before = self.current()
        self.local.s = s
        try:
            yield
        finally:
            self.local.s = before

    def _set(self, h, raw):
        time.sleep(0.0005)  # (another thread has time to come between)
        self.stream = getattr(raw, "value", raw) or 0
        return 0

    def _work(self, h, tag):
        time.sleep(0.0005)
        assert self.stream == self.current().cuda_stream, "launched on another thread's stream"
        self.current().touch().queue.append(tag)
        self.log.append((tag, self.current().name))
        return 0

    def _check(self, h):
        assert self.stream == self.current().cuda_stream
        self.current().touch()
        return 0


class FakeStream:
    device_index = 0

    def __init__(self, world, handle, name, external=False):
        self.world, self.cuda_stream, self.name = world, handle, name
        self.stream_id = handle if external else (handle and 8 * handle + 3)  # (torch's own ids are no handles)
        self.dead, self.capturing, self.queue, self.after = False, None, [], set()

    def touch(self):
        assert not self.dead, f"{self.name} is gone"
        return self

    def work(self):
        return set(self.queue) | self.after

    def wait_stream(self, other):
        other.touch()
        assert self.touch().capturing == other.capturing, "an edge between a capture and what is outside it"
        self.after |= other.work()

    def wait_event(self, event):
        assert event.capturing == self.touch().capturing, "an edge between a capture and what is outside it"
        self.after |= event.work


class FakeEvent:
    def __init__(self, world):
        self.world, self.work, self.capturing = world, set(), None

    def record(self, stream=None):
        s = (stream or self.world.current()).touch()
        self.work, self.capturing = s.work(), s.capturing


@pytest.fixture
def world(monkeypatch):
    return World(monkeypatch)


def test_a_call_on_another_stream_waits_for_the_calls_before_it(world):
    ctx = h3.Context(0)
    a, b = FakeStream(world, 16, "a"), FakeStream(world, 32, "b")
    for s, tag in ((a, "1"), (a, "2"), (b, "3"), (world.default, "4"), (a, "5")):
        with world.on(s):
            ctx.call("work", tag)
    assert "2" in b.after and "3" in world.default.after and "4" in a.after
    with world.on(b):
        ctx.check_device()
    assert "5" in b.after


def test_a_callers_stream_may_be_gone_when_the_next_call_comes(world):
    ctx = h3.Context(0)
    own, other = FakeStream(world, 16, "own", external=True), FakeStream(world, 32, "other")
    with world.on(own):
        ctx.call("work", "1")
        ctx.call("work", "2")
    own.dead = True
    with world.on(other):
        ctx.call("work", "3")
    assert {"1", "2"} <= other.after  # still ordered
    with world.on(own2 := FakeStream(world, 16, "own2", external=True)):  # the handle comes again
        ctx.call("work", "4")
    assert "3" in own2.after
    own2.dead = True
    with world.on(FakeStream(world, 16, "own3", external=True)) as _:
        ctx.call("work", "5")
        assert "4" in world.current().after
    world_now = world.current()
    ctx.check_device()
    assert "5" in world_now.after


def test_captured_calls_are_kept_apart_from_direct_ones(world):
    ctx = h3.Context(0)
    a, b, c, d = (FakeStream(world, 16 * (i + 1), "abcd"[i]) for i in range(4))
    with world.on(a):
        ctx.call("work", "1")
    b.capturing = c.capturing = 7
    with world.on(b):
        ctx.call("work", "2")  # no edge from a
    with world.on(c):  # another branch of the same capture: they share scratch
        ctx.call("work", "3")
    assert "2" in c.after and "1" not in b.after | c.after
    with world.on(d):  # a direct call beside the capture: after the direct one before it, with no edge to the capture
        ctx.call("work", "4")
    assert d.after == {"1"}
    with world.on(b):
        ctx.call("work", "5")
    b.capturing = c.capturing = None
    with world.on(a):
        ctx.call("work", "6")
    assert "4" in a.after
    with world.on(b):  # the stream that was captured, now for a direct call
        ctx.call("work", "7")
    assert "6" in b.after
    with world.on(a):
        ctx.call("work", "8")
    assert "7" in a.after


def test_branches_of_a_capture_on_the_stream_used_before(world):
    """Warm-up and capture on one stream: the context sees no change of streams between them."""
    ctx = h3.Context(0)
    a, b = FakeStream(world, 16, "a"), FakeStream(world, 32, "b")
    with world.on(a):
        ctx.call("work", "1")
        a.queue.clear()
        a.capturing = b.capturing = 3
        ctx.call("work", "2")
    with world.on(b):
        ctx.call("work", "3")
    assert "2" in b.after

def test_threads_keep_their_streams(world):
    """More threads than streams' worth of luck: every launch is on its own thread's stream."""
    ctx = h3.Context(0)
    failed = []

    def run(i):
        try:
            with world.on(FakeStream(world, 16 * (i + 1), f"s{i}")):
                for k in range(30):
                    ctx.call("work", f"{i}.{k}")
        except BaseException as e:  # noqa: BLE001 (reported below)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]
    assert len(world.log) == 120


def test_threads_share_one_context(world, monkeypatch):
    made = []

    class Slow(h3.Context):
        def __init__(self, device):
            time.sleep(0.01)
            super().__init__(device)
            made.append(self)

    monkeypatch.setattr(h3, "Context", Slow)
    monkeypatch.setattr(h3, "_contexts", {})
    got = []
    threads = [threading.Thread(target=lambda: got.append(h3.context(0))) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and all(c is made[0] for c in got)
