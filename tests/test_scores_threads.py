"""Threads whose first calls of the operators come at the same time, without a GPU."""
import threading
import time

from loe_speech_recognition_amd import _native


def test_first_calls_at_once_share_one_engine(monkeypatch):
    class Slow:
        def __init__(self):
            time.sleep(0.05)

    monkeypatch.setattr(_native, "Engine", Slow)
    monkeypatch.setattr(_native, "_engine", None)
    monkeypatch.setattr(_native, "_engine_pid", None)
    gate, seen = threading.Barrier(8), []

    def first_call():
        gate.wait()
        seen.append(_native.get_engine())

    threads = [threading.Thread(target=first_call) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(seen) == 8 and all(e is seen[0] for e in seen)


class _TwoDevices:
    """As much of torch.cuda as the order of streams needs: the engine on device 1, device 0 the current one, one of the two
    current streams captured."""

    def __init__(self, captured):
        self.captured, self.now, self.waits = captured, 0, []

    def device(self, device):
        cuda = self

        class Guard:
            def __enter__(self):
                self.before, cuda.now = cuda.now, device

            def __exit__(self, *_):
                cuda.now = self.before

        return Guard()

    def is_current_stream_capturing(self):
        return self.now == self.captured

    def current_device(self):
        return self.now

    def set_device(self, device):
        self.now = device

    def current_stream(self, device):
        return _Stream("current", self)


class _Stream:
    def __init__(self, name, cuda):
        self.name, self.cuda, self.cuda_stream = name, cuda, 7

    def wait_stream(self, other):
        self.cuda.waits.append((self.name, other.name))


def _engine_on_device_1(captured):
    import types

    cuda = _TwoDevices(captured)
    eng = object.__new__(_native.Engine)
    eng.torch = types.SimpleNamespace(cuda=cuda)
    eng.lib = types.SimpleNamespace(lsr_set_stream=lambda *_: 0)
    eng.device, eng.device_index, eng.rows_ctx = 1, 1, None
    eng._raw_stream, eng._stream_handle, eng._stream = lambda index: 7, 5, _Stream("engine", cuda)
    eng._turn = threading.Lock()
    return eng, cuda


def test_captures_on_another_device_are_not_the_engines():
    """Device 0's stream is captured, the engine is on device 1: its streams wait for each other as ever, and the current device
    is what it was."""
    eng, cuda = _engine_on_device_1(captured=0)
    with eng.in_order():
        pass
    eng.on_current_stream(lambda *_: 0)
    assert cuda.waits == [("engine", "current"), ("current", "engine"), ("current", "engine")] and cuda.now == 0


def test_captures_on_the_engines_device_are_seen_from_another():
    import pytest

    eng, cuda = _engine_on_device_1(captured=1)
    with pytest.raises(_native.NativeError, match="own stream"):
        with eng.in_order():
            pass
    eng.on_current_stream(lambda *_: 0)                   # captured without a wait for what came before
    assert cuda.waits == [] and cuda.now == 0
