"""The checked positions of ``apply_rope_axes`` from several threads: the range search writes into page-locked memory that
belongs to one thread, so a thread never waits for another one's answer.  No GPU: the kernel is a timer that writes later."""
import ctypes
import threading
import time

import pytest
import torch

from pom_b200 import _abi, ops
from pom_b200.operators import apply_rope_axes


class LateLibrary:
    """pom_pos_range of the library, answered some time after the call (or when ``flush`` asks for it)."""

    def __init__(self, delay):
        self.delay, self.jobs, self.lock = delay, [], threading.Lock()

    def pom_pos_range_blocks(self, rows):
        return 1

    def pom_pos_range(self, pos, rows, axes, at, stream):
        self.flush()  # what was enqueued before is done at the latest now
        p = list((ctypes.c_int64 * (rows * axes)).from_address(pos))
        out = (ctypes.c_int64 * (2 * axes)).from_address(at)

        def write():
            for a in range(axes):
                out[2 * a], out[2 * a + 1] = min(p[a::axes]), max(p[a::axes])

        with self.lock:
            self.jobs.append(write)
        if self.delay is not None:
            threading.Timer(self.delay, self.flush).start()
        return 0

    def flush(self):
        with self.lock:
            jobs, self.jobs = self.jobs, []
        for j in jobs:
            j()


@pytest.fixture
def late(monkeypatch):
    lib = LateLibrary(0.01)
    empty, kept = torch.empty, []

    def slow_empty(*args, pin_memory=False, **kw):
        t = empty(*args, **kw)
        if pin_memory:
            time.sleep(0.05)  # page-locking lets other threads run
            kept.append(t)  # a write that comes too late must not end the process
        return t

    class Stream:
        def synchronize(self):
            time.sleep(0.1)
            lib.flush()

    monkeypatch.setattr(_abi, "lib", lambda: lib)
    monkeypatch.setattr(_abi, "stream_of", lambda i: 0)
    monkeypatch.setattr(ops, "_same_device", lambda *a: 0)
    monkeypatch.setattr(ops, "rope_axes", lambda x, pos, tables, transpose=False: x)
    monkeypatch.setattr(torch, "empty", slow_empty)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: lib.flush())
    if isinstance(ops._host_range, threading.local):
        monkeypatch.setattr(ops, "_host_range", threading.local())  # as after the import
    else:
        monkeypatch.setattr(ops, "_host_range", None)
    return lib


def call(position):
    tables = [(torch.ones(10, 2), torch.zeros(10, 2)), (torch.ones(12, 2), torch.zeros(12, 2))]
    pos = torch.tensor([[1, 2], [3, position]])
    return apply_rope_axes(torch.ones(1, 2, 8), pos, tables)


@pytest.mark.parametrize("threads", [2, 5])
def test_first_calls_of_several_threads(late, threads):
    got, ready = {}, threading.Barrier(threads)

    def work(i):
        ready.wait()
        for turn in range(3):
            try:
                call(11 if i % 2 else 12 + i)  # odd threads: inside the table of 12 rows
                got[i, turn] = None
            except Exception as e:  # noqa: BLE001 (what came is compared below)
                got[i, turn] = e

    ts = [threading.Thread(target=work, args=(i,)) for i in range(threads)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    for (i, turn), e in got.items():
        if i % 2:
            assert e is None, (i, turn, repr(e))
        else:
            assert isinstance(e, IndexError) and f"span [2, {12 + i}]" in str(e), (i, turn, repr(e))
    assert len(got) == 3 * threads


def test_a_call_after_an_interrupted_wait_reads_its_own_answer(late, monkeypatch):
    late.delay = None
    with monkeypatch.context() as m:
        def interrupt():
            raise KeyboardInterrupt
        m.setattr(time, "monotonic", interrupt)
        with pytest.raises(KeyboardInterrupt):
            call(40)  # enqueued, and never waited for
    late.delay = 0.01
    call(5)  # must not see the 40 that the first kernel writes late
    with pytest.raises(IndexError, match=r"span \[2, 30\]"):
        call(30)
