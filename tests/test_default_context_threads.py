"""The default context of a device when several threads ask for it first; no GPU is needed for it."""
import threading
import time

from graph_sampling_b200 import ops


def test_threads_that_come_first_get_one_context(monkeypatch):
    class Slow:
        def __init__(self, device):
            time.sleep(0.05)
            self.device = device

    monkeypatch.setattr(ops, "Context", Slow)
    monkeypatch.setattr(ops, "_contexts", {})
    got, start = [], threading.Barrier(8)

    def ask():
        start.wait()
        got.append(ops.default_context("cuda:0"))

    threads = [threading.Thread(target=ask) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert len(got) == 8 and len({id(c) for c in got}) == 1
    assert ops.default_context("cuda:0") is got[0] and ops.default_context("cuda:1") is not got[0]
