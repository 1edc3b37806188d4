"""Threads that call moe.experts on one stream do not mix their launches on its workspace."""
import threading
import time

import pytest
import torch

from rocknpu_amd import hip, moe


def test_one_call_at_a_time_on_a_stream(monkeypatch):
    """A library that takes its time notes who is inside: one call a stream, calls on different streams side by side."""
    i8, f = (lambda *s: torch.zeros(s, dtype=torch.int8)), torch.zeros
    w = moe.Experts((i8(4, 60, 128), f(4, 60)), (i8(4, 60, 128), f(4, 60)), (i8(4, 100, 64), f(4, 100)), hidden=100, ffn=60)
    r = moe.Routing(torch.zeros((3, 2), dtype=torch.int32), f(3, 2), torch.zeros(moe.plan_words(3, 4, 2), dtype=torch.int32), 4)
    mine, inside, most, guard = threading.local(), {0: 0, 1: 0}, {0: 0, 1: 0, "all": 0}, threading.Lock()

    def library(index, function, *args):
        stream = args[-1]
        with guard:
            inside[stream] += 1
            most[stream] = max(most[stream], inside[stream])
            most["all"] = max(most["all"], sum(inside.values()))
        time.sleep(0.002)
        with guard:
            inside[stream] -= 1
        return 0

    monkeypatch.setattr(hip, "stream_of", lambda device: (0, mine.stream))
    monkeypatch.setattr(hip, "call_on", library)
    monkeypatch.setattr(moe, "workspace_for", lambda device, nbytes: torch.zeros(nbytes, dtype=torch.uint8))

    def calls(stream):
        mine.stream = stream
        for _ in range(20):
            moe.experts(w, i8(3, 128), f(3), r)

    threads = [threading.Thread(target=calls, args=(i % 2,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert most[0] == most[1] == 1 and most["all"] == 2


@pytest.mark.gpu
def test_threads_on_one_stream():
    from tests.test_gpu_moe_experts import layer, tokens_of
    w = layer(26, 8, 256, 192)
    jobs = []
    for i, tokens in enumerate((300, 290, 3, 200)):
        a8, s = tokens_of(60 + i, tokens, 256)
        r = moe.route(torch.randn((tokens, 8), generator=torch.Generator().manual_seed(70 + i)).cuda(), 2)
        jobs.append((a8, s, r, moe.experts(w, a8, s, r)))
    torch.cuda.synchronize()
    outs = [[] for _ in jobs]

    def calls(i):
        a8, s, r, _ = jobs[i]
        for _ in range(50):
            outs[i].append(moe.experts(w, a8, s, r))

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for out, job in zip(outs, jobs):
        assert len(out) == 50 and all(torch.equal(o, job[3]) for o in out)
