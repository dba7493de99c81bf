"""What calls do with a workspace on the host: one call at a time binds it and
enqueues (no GPU needed: the library's entry is a stand-in)."""
import threading
import time

import pytest
import torch

from b200decode import _lib, ragged
from b200decode.api import DecodeWorkspace


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(ragged, "_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return torch.device("cpu")


class Entry:
    """A library entry that enqueues two launches; says "too small" below `needs` bytes."""

    def __init__(self, ws, needs):
        self.ws, self.needs, self.log = ws, needs, []

    def __call__(self, ref, stream):
        args = ref._obj
        if args.workspace_bytes < self.needs[args.batch]:
            time.sleep(0.002)
            return _lib.B2D_ERR_WORKSPACE
        for launch in range(2):
            self.log.append((args.batch, launch, args.workspace == self.ws.buf.data_ptr()))
            time.sleep(0.002)
        return 0

    def query(self, ref, n):
        n._obj.value = self.needs[ref._obj.batch]
        return 0


def test_one_call_at_a_time_in_a_workspace(host):
    """Threads that share a workspace, some of which make it grow: the launches
    of a call stand together, and each call's go to the buffer of the time."""
    ws = DecodeWorkspace(host)
    entry = Entry(ws, {i: (1 << 20) * (1 + i) for i in range(6)})

    def work(i):
        for _ in range(4):
            a = _lib.GqaArgs()
            a.batch = i
            ragged._call(entry, "entry", a, a, ws, -1, entry.query)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(entry.log) == 48
    for first, second in zip(entry.log[::2], entry.log[1::2]):
        assert first[0] == second[0] and (first[1], second[1]) == (0, 1)
        assert first[2] and second[2]


def test_status_outlives_growth(host):
    """A recorded status that nobody has read yet moves to the larger buffer;
    the arrival counters behind it start at zero."""
    ws = DecodeWorkspace(host)
    ws.buf[:8] = torch.tensor([2, 0, 0, 0, 9, 9, 9, 9], dtype=torch.uint8)
    old = ws.nbytes
    ws.ensure(old + 1)
    assert ws.nbytes > old
    assert ws.buf[:8].tolist() == [2, 0, 0, 0, 0, 0, 0, 0] and not ws.buf[8:].any()


def test_held_buffer_outlives_growth(host):
    """hold() keeps the buffer that a captured decode() was given; a workspace
    that must not grow still refuses to."""
    ws = DecodeWorkspace(host)
    held = ws.buf
    ws.hold()
    ws.hold()
    ws.ensure(ws.nbytes + 1)
    assert [b.data_ptr() for b in ws.held] == [held.data_ptr()] and ws.buf.data_ptr() != held.data_ptr()
    ws.captured = True
    with pytest.raises(ValueError, match="cannot grow"):
        ws.ensure(ws.nbytes + 1)


def test_buffer_made_under_capture_is_left_to_the_graph(host, monkeypatch):
    """A buffer that a capture allocated is zeroed by the graph's replay, not
    before: calls outside of the capture take another one."""
    ws = DecodeWorkspace(host)
    first = ws.buf
    ws.graph_made = True                       # (as _alloc() notes on a GPU)
    ws.buf.fill_(0xAB)                         # what such memory may hold
    ws.for_decode(1000)
    assert ws.buf.data_ptr() != first.data_ptr() and not ws.buf.any() and not ws.graph_made
    assert [b.data_ptr() for b in ws.held] == [first.data_ptr()]
    ws.graph_made = True
    ws.buf.fill_(0xAB)
    a = _lib.GqaArgs()
    entry = Entry(ws, {0: 1})
    ragged._call(entry, "entry", a, a, ws, -1, entry.query)
    assert not ws.buf.any() and len(ws.held) == 2 and all(at_buf for _, _, at_buf in entry.log)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    ws.for_decode(1000)
    assert ws.held[-1] is ws.buf
