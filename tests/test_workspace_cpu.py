"""Which workspace a call gets, eagerly and while its stream is captured, without a GPU: torch's
streams and the state of a capture are stood in for, the memory is the host's."""
import contextlib
import sys
import types
import weakref

import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd  # noqa: E402, F401

D = sys.modules["triton_ext_amd.dot"]  # (the name `dot` of the package is the function)

CPU = torch.device("cpu")


@pytest.fixture
def world(monkeypatch):
    """A stream 7 that is current; world.capture: the number of the capture it is part of."""
    w = types.SimpleNamespace(capture=0)
    monkeypatch.setattr(D, "_workspaces", {})
    monkeypatch.setattr(D, "_capture_of", lambda device, stream: w.capture, raising=False)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s, device=None: s)
    for name in ("stream", "device"):
        monkeypatch.setattr(torch.cuda, name, lambda x: contextlib.nullcontext())
    w.get = lambda n: D.workspace_for(types.SimpleNamespace(workspace_bytes=n), CPU, 7)
    return w


def test_eager_calls_share_and_grow(world):
    a = world.get(70000)
    assert a.numel() >= 70000 and not a.any()
    assert world.get(65536) is a
    b = world.get(200000)
    assert b.numel() >= 200000 and not b.any() and world.get(70000) is b
    assert world.get(0) is None


def test_a_captured_call_outlives_larger_ones(world):
    """The memory that a graph was given belongs to nobody else, whatever is called later."""
    eager = world.get(70000)
    world.capture = 1
    graph = world.get(70000)
    assert graph is not eager and world.get(65536) is graph
    assert not graph[:65536].any()
    where = weakref.ref(eager)
    world.capture = 0
    assert world.get(70000) is eager
    del eager
    world.get(1 << 20)  # the eager buffer goes, no graph reads it
    assert where() is None


def test_every_capture_clears_its_own_counters(world):
    """A graph starts on counters that it clears itself, so the order of replays does not matter."""
    world.capture = 1
    first = world.get(70000)
    first[:65536] = 1  # (as if the graph's fill had not run yet)
    world.capture = 2
    second = world.get(70000)
    assert second is not first and not second[:65536].any()
    assert second.data_ptr() != first.data_ptr()
    world.capture = 0
    third = world.get(70000)  # and calls outside of captures have theirs
    assert third is not first and third is not second and not third.any()


def test_a_capture_grows(world):
    world.capture = 3
    a = world.get(70000)
    b = world.get(300000)
    assert b is not a and b.numel() >= 300000 and not b[:65536].any()
    assert world.get(70000) is b
