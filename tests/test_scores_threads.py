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
