"""Graphs of a preconditioner that is gone, while another is captured.

On the CPU, with a stand-in for the capture: a graph destroyed in one would
end the process on a GPU.
"""
import contextlib
import gc
import threading

import pytest
import torch

from kfac_pytorch_amd.preconditioner import base


class Graph:
    capturing = False
    replays = 0

    def replay(self):
        Graph.replays += 1


@contextlib.contextmanager
def capture(graph):
    Graph.capturing = True
    try:
        yield
    finally:
        Graph.capturing = False


class Stream:
    def wait_stream(self, other):
        pass


@pytest.fixture
def cuda(monkeypatch):
    gc.collect()
    Graph.replays = 0
    for name, value in [
            ("is_available", lambda: True), ("Stream", Stream),
            ("CUDAGraph", Graph), ("graph", capture),
            ("current_stream", Stream),
            ("stream", lambda s: contextlib.nullcontext()),
            ("is_current_stream_capturing", lambda: Graph.capturing)]:
        monkeypatch.setattr(torch.cuda, name, value)
    yield
    gc.collect()
    base._CapturedGraph._dropped.clear()


class Owner:
    """What _run_graphed needs of a preconditioner, in a reference cycle."""

    def __init__(self):
        self.me = self

    run = base.KFACBase._run_graphed


def test_collector_waits_for_the_end_of_a_capture(cuda):
    seen = []
    owner = Owner()
    assert gc.isenabled()
    owner.run("pred", lambda: seen.append((Graph.capturing, gc.isenabled())),
              1)
    assert seen == [(False, True), (True, False)]
    assert gc.isenabled() and Graph.replays == 1
    owner.run("pred", seen.clear, 1)  # replayed, not run
    assert len(seen) == 2 and Graph.replays == 2


def test_collector_stays_off_where_it_was(cuda):
    gc.disable()
    try:
        Owner().run("pred", lambda: None, 1)
        assert not gc.isenabled()
    finally:
        gc.enable()


def test_collector_is_back_after_a_failed_capture(cuda):
    def fails_in_capture():
        if Graph.capturing:
            raise RuntimeError("not capturable")

    owner = Owner()
    owner.run("pred", fails_in_capture, 1)
    assert gc.isenabled() and owner._graph_disabled


def test_a_graph_dropped_within_a_capture_is_kept_until_after_it(cuda):
    dropped = base._CapturedGraph._dropped
    owner = Owner()
    owner.run("pred", lambda: None, 1)
    graph = id(owner._graphs["pred"][0].graph)
    with capture(None):  # somebody's own
        del owner
        gc.collect()
        assert [id(g) for g in dropped] == [graph]
        base._CapturedGraph.sweep()
        assert len(dropped) == 1
    owner = Owner()
    owner.run("pred", lambda: None, 1)
    assert not dropped
    del owner
    gc.collect()  # outside a capture nothing is kept
    assert not dropped


def test_what_was_put_off_goes_with_the_next_collection(cuda):
    """Without another preconditioner that captures."""
    dropped = base._CapturedGraph._dropped
    owner = Owner()
    owner.run("pred", lambda: None, 1)
    with capture(None):
        del owner
        gc.collect()
        gc.collect()
        assert len(dropped) == 1
    gc.collect()
    assert not dropped


def test_a_graph_dropped_while_another_thread_captures(cuda, monkeypatch):
    """The thread that drops it does not capture itself."""
    here = threading.current_thread()
    monkeypatch.setattr(
        torch.cuda, "is_current_stream_capturing",
        lambda: Graph.capturing and threading.current_thread() is not here)
    dropped = base._CapturedGraph._dropped
    owner = Owner()
    owner.run("pred", lambda: None, 1)
    captures, goes_on = threading.Event(), threading.Event()

    def work():
        if Graph.capturing:
            captures.set()
            assert goes_on.wait(30)

    other = Owner()
    thread = threading.Thread(target=other.run, args=("pred", work, 1))
    thread.start()
    try:
        assert captures.wait(30)
        owner.me = None  # no cycle: it goes at once
        del owner
        assert len(dropped) == 1
        base._CapturedGraph.sweep()
        assert len(dropped) == 1
    finally:
        goes_on.set()
        thread.join()
    assert base._CapturedGraph._captures == 0
    gc.collect()
    assert not dropped
    assert not getattr(other, "_graph_disabled", False)


def test_captures_are_counted_when_they_fail(cuda):
    def fails_in_capture():
        if Graph.capturing:
            raise RuntimeError("not capturable")

    Owner().run("pred", fails_in_capture, 1)
    assert base._CapturedGraph._captures == 0
