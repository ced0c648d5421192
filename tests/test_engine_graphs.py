"""What the engine does with its HIP graphs around a capture, and which launch mode "auto" takes (no GPU needed: the pieces are
called on an engine without a device)."""
import gc
import types

import pytest
import torch

from scarches_amd import engine as E


@pytest.fixture
def device(monkeypatch):
    """A device that is never busy: what was asked of it, in order."""
    log = types.SimpleNamespace(calls=[], capturing=False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: log.calls.append("synchronize"))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: log.capturing)
    return log


class Graph:
    """Says when it is destroyed."""
    def __init__(self, log):
        self.log = log

    def __del__(self):
        self.log.calls.append("destroyed")


def bare(log):
    eng = E.CVAEEngine.__new__(E.CVAEEngine)
    eng.device, eng._graph_size = "cuda:0", None
    eng._plans = {1: dict(fwd=Graph(log))} if log is not None else {}
    return eng


def test_graphs_go_behind_a_wait(device):
    eng = bare(device)
    eng._invalidate()
    assert device.calls == ["synchronize", "destroyed"] and eng._plans == {}
    eng = bare(device)
    eng.close()
    assert device.calls == ["synchronize", "destroyed"] * 2
    del eng
    assert device.calls == ["synchronize", "destroyed"] * 2         # nothing left to wait for
    eng = bare(device)
    del eng
    assert device.calls == ["synchronize", "destroyed"] * 3


def test_an_engine_that_goes_in_a_capture(device):
    eng = bare(device)
    eng.me = eng                                                    # (only the garbage collector finds it)
    graph = eng._plans[1]["fwd"] = object()
    buffer = eng.flat_p = object()
    device.calls.clear()
    device.capturing = True
    del eng
    gc.collect()
    assert device.calls == [] and len(E._DROPPED) == 1
    assert E._DROPPED[0]["_plans"][1]["fwd"] is graph and E._DROPPED[0]["flat_p"] is buffer
    E._DROPPED.clear()


def test_no_garbage_is_collected_in_a_capture(device, monkeypatch):
    seen = []

    class Capture:
        def __init__(self, graph):
            pass

        def __enter__(self):
            seen.append((gc.isenabled(), len(E._DROPPED)))

        def __exit__(self, *exc):
            return False
    stream = types.SimpleNamespace(wait_stream=lambda s: None)
    monkeypatch.setattr(torch.cuda, "Stream", lambda **kw: stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: Capture(None))
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: "graph")
    monkeypatch.setattr(torch.cuda, "graph", Capture)
    eng = bare(None)
    monkeypatch.setattr(eng, "_warm", lambda *a: (0, 0, 0), raising=False)
    restored = []
    monkeypatch.setattr(eng, "_restore", restored.append, raising=False)
    E._DROPPED.append(dict(_plans={1: dict(fwd=Graph(device))}))

    def step(*a):
        seen.append(gc.isenabled())
        if a[2] < 0:
            raise RuntimeError("in the step")
    monkeypatch.setattr(eng, "_step_and_adam", step, raising=False)
    assert eng._capture(4, 0.0, None, False)["fwd"] == "graph"
    assert seen[-2:] == [(False, 0), False] and gc.isenabled() and device.calls == ["synchronize", "destroyed"]
    with pytest.raises(RuntimeError, match="in the step"):
        eng._capture(-1, 0.0, None, False)
    assert gc.isenabled() and eng._graph_size == 4
    with pytest.raises(RuntimeError, match="in the step"):
        eng._record(-1, 0.0, None, False)
    assert restored == [0, 0, 0] and eng._rec is None               # the warm-up's step is taken back, whatever came of it


def test_auto_captures_one_batch_size(device, monkeypatch):
    """A ragged last minibatch, and everything behind an encoder pass, takes the recorded plan."""
    eng = bare(None)
    assert eng._auto_launch(4096, 1) is True and eng._auto_launch(E.GRAPH_MAX_B + 1, 1) == "plan" == eng._auto_launch(4096, 2)
    eng._graph_size = 4096
    assert eng._auto_launch(4096, 1) is True and eng._auto_launch(1000, 1) == "plan"

    def stop(B):
        raise KeyError("far enough")
    for size, then in ((4096, 0), (None, None)):            # a pass in front of the first step changes nothing
        eng._graph_size = size
        monkeypatch.setattr(eng, "_ensure", stop, raising=False)
        monkeypatch.setattr(eng, "lib", None, raising=False)
        monkeypatch.setattr(eng, "p", None, raising=False)
        with pytest.raises(KeyError):
            eng.encode(None, None, 512)
        assert eng._graph_size == then
    eng._graph_size = 0
    assert eng._auto_launch(4096, 1) == eng._auto_launch(128, 1) == "plan"
