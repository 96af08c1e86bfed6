"""Text-side calls on several streams: a caller's own stream, branches of a capture, threads. Each call has inputs of
its own, and is compared with the same call alone."""
import threading

import pytest
import torch

from tests.test_gpu_text import _check_device
from tests.test_gpu_text_capture import Step, _clone, _same

pytestmark = pytest.mark.gpu


def _own_stream():
    import ctypes
    handle = ctypes.c_size_t(0)
    rt = torch.cuda.cudart()
    assert int(rt.cudaStreamCreate(ctypes.addressof(handle))) == 0
    return torch.cuda.ExternalStream(handle.value), handle.value


def test_a_stream_of_the_callers_own_and_none_of_it_afterwards():
    """The stream is destroyed between the calls: the context neither touches it nor loses the order."""
    a, b = Step("bf16", 9000, 1, 1), Step("bf16", 8000, 100, 2)
    want = _clone(a.run()), _clone(b.run())
    torch.cuda.synchronize()
    for _ in range(3):
        own, handle = _own_stream()
        assert own.cuda_stream == handle
        with torch.cuda.stream(own):
            assert torch.cuda.current_stream().stream_id == handle  # how the context knows it
            got = [a.run() for _ in range(5)]
        torch.cuda.cudart().cudaStreamDestroy(handle)
        got_b = b.run()
        _check_device()
        torch.cuda.synchronize()
        assert all(_same(x, want[0]) for x in got) and _same(got_b, want[1])


def test_branches_of_one_capture():
    steps = [Step("bf16", 9000, 1, 3), Step("int8", 7000, 2, 4), Step("e4m3", 6000, 90, 5)]
    wants = [_clone(s.run()) for s in steps]
    outs = [None] * 3
    graph = torch.cuda.CUDAGraph()
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        for s in sides:
            s.wait_stream(here)
        outs[0] = steps[0].run()
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                outs[i + 1] = steps[i + 1].run()
        for s in sides:
            here.wait_stream(s)
    for _ in range(10):
        for o in outs:
            for t in o:
                t.zero_()
        graph.replay()
        assert all(_same(o, w) for o, w in zip(outs, wants))
    _check_device()


def test_streams_with_inputs_of_their_own():
    """Calls in turn on three streams, with enough keys that they would overlap: no call finds another's
    partial sums in the workspace."""
    steps = [Step("bf16", 9000, 1, 6), Step("int8", 8000, 3, 7), Step("bf16", 7000, 100, 8)]
    wants = [_clone(s.run()) for s in steps]
    assert not any(torch.equal(wants[0][0], w[0]) for w in wants[1:])
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams[1:]:
        s.wait_stream(streams[0])
    got = []
    for i in range(30):
        with torch.cuda.stream(streams[i % 3]):
            got.append(steps[i % 3].run())
    torch.cuda.synchronize()
    _check_device()
    assert all(_same(o, wants[i % 3]) for i, o in enumerate(got))


def test_threads_with_streams_of_their_own():
    """Threads share the device's context: each one's calls go to its own stream, behind its own inputs."""
    steps = [Step("bf16", 9000, 1, 9), Step("int8", 8000, 3, 10), Step("bf16", 7000, 100, 11), Step("e4m3", 5000, 2, 12)]
    wants = [[] for _ in steps]
    for i, s in enumerate(steps):
        for seed in range(10):
            s.refresh(100 * i + seed)
            wants[i].append(_clone(s.run()))
    torch.cuda.synchronize()
    got, failed = [[] for _ in steps], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for seed in range(10):
                    steps[i].refresh(100 * i + seed)  # (queued on this thread's stream: the call has to follow it)
                    got[i].append(_clone(steps[i].run()))
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 (reported below)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]
    _check_device()
    for g, w in zip(got, wants):
        assert all(_same(x, y) for x, y in zip(g, w))


def test_tensors_on_another_device_than_the_current_one():
    """The calls run where the tensors are: their scratch is allocated there, and the current device stays."""
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    want = []
    for dev in (1, 0):
        with torch.cuda.device(dev):
            steps = Step("bf16", 9000, 1, 20), Step("int8", 6000, 100, 21)
            if dev == 1:
                there = steps
            else:
                want = [_clone(s.run()) for s in steps]
    with torch.cuda.device(0):
        got = [s.run() for s in there]
        assert torch.cuda.current_device() == 0
        for g, w in zip(got, want):
            assert all(x.device.index == 1 for x in g)
            assert _same([x.to("cuda:0") for x in g], w)
    for dev in (0, 1):
        with torch.cuda.device(dev):
            _check_device()
