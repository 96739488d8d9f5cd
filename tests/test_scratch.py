"""Scratch shared by the calls of a stream: who gets which buffer, with the
capture state of the stream faked (no GPU needed)."""
import pytest
import torch

from vates_b200 import scratch
from vates_b200.scratch import Scratch

CPU = torch.device("cpu")


@pytest.fixture
def capture(monkeypatch):
    state = {"id": 0}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["id"] > 0)

    class Lib:
        @staticmethod
        def vb_stream_capture_id(st):
            return state["id"]

    monkeypatch.setattr(scratch, "lib", Lib)
    return state


def test_calls_of_a_stream_share_a_buffer(capture):
    s = Scratch(16)
    a = s.get(100, CPU, 1)
    assert a.numel() >= 100 and not a.any()
    assert s.get(50, CPU, 1) is a and s.get(50, CPU, 2) is not a
    b = s.get(200, CPU, 1)
    assert b.numel() >= 200 and s.get(100, CPU, 1) is b
    assert s.get(1, CPU, 3).numel() >= 16


def test_a_capture_never_takes_or_leaves_an_eager_buffer(capture):
    s = Scratch(16)
    eager = s.get(100, CPU, 1)
    capture["id"] = 7
    a = s.get(50, CPU, 1)
    assert a is not eager and not a[:16].any()
    assert s.get(40, CPU, 1) is a          # the calls of one capture
    assert s.get(40, CPU, 2) is not a      # a stream that was forked in it
    capture["id"] = 0
    assert s.get(100, CPU, 1) is eager
    capture["id"] = 8
    b = s.get(50, CPU, 1)
    assert b is not a and b is not eager and not b[:16].any()


def test_a_first_call_in_a_capture_leaves_nothing_behind(capture):
    """Its zero fill has not run when the capture ends."""
    s = Scratch(16)
    capture["id"] = 3
    a = s.get(50, CPU, 1)
    a.fill_(9)
    capture["id"] = 0
    b = s.get(50, CPU, 1)
    assert b is not a and not b.any()


def test_a_larger_call_in_a_capture(capture):
    s = Scratch(16)
    capture["id"] = 3
    a = s.get(50, CPU, 1)
    b = s.get(500, CPU, 1)
    assert b is not a and b.numel() >= 500 and not b[:16].any() and s.get(50, CPU, 1) is b


def test_a_capture_without_a_number_shares_nothing(capture, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    s = Scratch(16)
    assert s.get(50, CPU, 1) is not s.get(50, CPU, 1)


def test_buffers_of_captures_are_let_go(capture):
    """A graph's pool keeps its memory: what is held here is the last capture's, and
    that only until the next eager call. (A capture that is under way then takes
    another buffer, which it fills again.)"""
    s = Scratch(16)
    for capture["id"] in (3, 4):
        for st in (1, 2):
            s.get(50, CPU, st)
    assert len(s._captured) == 2 and s._capture == 4
    a = s.get(50, CPU, 1)
    capture["id"] = 0
    s.get(50, CPU, 9)
    assert not s._captured
    capture["id"] = 4
    b = s.get(50, CPU, 1)
    assert b is not a and not b[:16].any()


def test_the_default_stream_is_not_asked(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: 1 / 0)
    s = Scratch(16)
    assert s.get(50, CPU, 0) is s.get(50, CPU, 0)


def test_moe_workspace_keeps_what_graphs_may_hold(capture, monkeypatch):
    from vates_b200 import moe_block
    monkeypatch.setattr(moe_block, "stream_handle", lambda: 1)
    w = moe_block.Workspace(CPU)
    capture["id"] = 2
    first = w.get(64)  # nothing was there: the graph's own
    assert not first.any() and w.buf is None
    capture["id"] = 0
    small = w.get(64)
    assert small is not first and not small.any()
    capture["id"] = 5
    assert w.get(64) is small
    assert w.get(128) is not small and w.buf is small
    capture["id"] = 0
    large = w.get(128)
    assert large is w.buf and not large.any() and w.get(64) is large
    assert any(t is small for t in w._outgrown)
