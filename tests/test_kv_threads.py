"""Threads that call kv.attention on one stream do not mix their launches on its workspace."""
import threading
import time

import torch

from rocknpu_amd import _lib, kv
from tests.test_kv import small_cache


def test_one_call_at_a_time_on_a_stream(monkeypatch):
    """A library that takes its time notes who is inside: one call a stream, calls on different streams side by side."""
    real = _lib.load()
    mine, inside, most, guard = threading.local(), {0: 0, 1: 0}, {0: 0, 1: 0, "all": 0}, threading.Lock()

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def rocknpu_hip_kv_attention(self, cache, args, ws, nbytes, stream):
            with guard:
                inside[stream] += 1
                most[stream] = max(most[stream], inside[stream])
                most["all"] = max(most["all"], sum(inside.values()))
            time.sleep(0.002)
            with guard:
                inside[stream] -= 1
            return 0

    library = Library()
    monkeypatch.setattr(kv._lib, "load", lambda: library)
    monkeypatch.setattr(kv, "_stream", lambda device: mine.stream)
    monkeypatch.setattr(kv, "workspace_for", lambda device, nbytes: torch.zeros(nbytes, dtype=torch.uint8))
    cache = small_cache(weights=torch.zeros((2, 1, 3)))
    past, cu = torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)

    def calls(stream):
        mine.stream = stream
        for _ in range(20):
            kv.attention(cache, torch.zeros((2, 1, 64)), past, cu, 1, weights_out=cache.weights)

    threads = [threading.Thread(target=calls, args=(i % 2,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert most[0] == most[1] == 1 and most["all"] == 2
