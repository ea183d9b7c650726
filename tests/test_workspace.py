"""Scratch of the eager calls: two threads that launch on one stream never share it."""
import threading

import pytest
import torch

from sglite_amd import ops

DEV = torch.device("cpu:0")


@pytest.fixture
def stream(monkeypatch):
    at = {"stream": object()}  # of this test alone
    monkeypatch.setattr(ops, "_stream", lambda device: at["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return at


def test_threads_on_one_stream_have_buffers_of_their_own(stream):
    mine = ops._workspace(1 << 21, DEV)
    assert ops._workspace(1 << 20, DEV) is mine  # a thread's calls on a stream follow each other
    got, both = [], threading.Barrier(2)

    def call():
        t = ops._workspace(1 << 21, DEV)
        both.wait(10)  # both are alive: neither buffer is the other's freed one
        got.append((t, ops._workspace(1 << 20, DEV)))
        both.wait(10)

    threads = [threading.Thread(target=call) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert len(got) == 2 and all(a is b for a, b in got)
    assert len({t.data_ptr() for t in (mine, got[0][0], got[1][0])}) == 3


def test_a_stream_has_its_own_and_it_grows(stream):
    a, first = ops._workspace(100, DEV), stream["stream"]
    stream["stream"] = object()
    assert ops._workspace(100, DEV).data_ptr() != a.data_ptr()
    stream["stream"] = first
    assert ops._workspace(1 << 20, DEV) is a  # the least it takes is 1 MiB
    assert ops._workspace((1 << 20) + 1, DEV).numel() > a.numel()
    assert ops._workspace(0, DEV) is None
