"""Where a call that names a stream allocates and copies, without a GPU: streams, launches and the
workspace are stood in for, torch's operations on host tensors are watched."""
import contextlib
import sys
import types

import pytest

torch = pytest.importorskip("torch")

from torch.utils._python_dispatch import TorchDispatchMode  # noqa: E402

import triton_ext_amd as tx  # noqa: E402
from triton_ext_amd import cache as C  # noqa: E402
from triton_ext_amd import capi  # noqa: E402

D = sys.modules["triton_ext_amd.dot"]
BF, I32 = torch.bfloat16, torch.int32
MAKES = ("empty", "zeros", "clone", "copy", "fill", "zero_")


class Watch(TorchDispatchMode):
    """Notes the current stream under every operation that makes or writes memory."""

    def __init__(self, world):
        super().__init__()
        self.world = world

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        name = func.overloadpacket.__name__
        if any(m in name for m in MAKES):
            self.world.seen.append((name, self.world.now))
        return func(*args, **(kwargs or {}))


@pytest.fixture
def world(monkeypatch):
    w = types.SimpleNamespace(now=0, seen=[], launched=[])

    @contextlib.contextmanager
    def stream(s):
        before, w.now = w.now, s
        yield
        w.now = before

    def launch(f, *args):
        w.launched.append(args[-1])
        return 0
    native = capi.calls()
    monkeypatch.setattr(C, "_native", types.SimpleNamespace(form=native.form, call=launch,
                                                            addresses=native.addresses))
    monkeypatch.setattr(C, "_forms", {})
    lib = capi.load()

    class Library:
        tx_dot_launch = tx_attn_fwd_launch = staticmethod(lambda *args: launch(*args))

        def __getattr__(self, name):
            return getattr(lib, name)
    monkeypatch.setattr(capi, "load", lambda *name: Library())
    for module in (C, D):
        monkeypatch.setattr(module, "_current_stream", lambda device: w.now)
    monkeypatch.setattr(D, "_workspaces", {})
    monkeypatch.setattr(D, "_capturing", lambda: False)
    monkeypatch.setattr(D, "_capture_of", lambda device, s: 0)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s, device=None: s)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", stream)
    return w


def apart(*shape, dtype=BF):
    """A tensor whose elements lie apart, so that the call copies it."""
    return torch.zeros(*shape, 2, dtype=dtype)[..., 0]


def ints(*shape):
    return apart(*shape, dtype=I32)


def pools():
    return [torch.zeros(8, 16, 2, 64, dtype=BF) for _ in range(2)]


CALLS = {  # entry point, arguments, keywords
    "rotary": lambda: ("rotary", (apart(5, 2, 64), ints(5), apart(32, dtype=torch.float32)), {}),
    "append": lambda: ("paged_append", (apart(2, 2, 64), apart(2, 2, 64), *pools(),
                                        torch.zeros(2, 4, dtype=I32), ints(2)),
                       {"q": apart(2, 4, 64), "inv_freq": apart(32, dtype=torch.float32)}),
    "attention": lambda: ("paged_attention", (apart(2, 4, 64), *pools(),
                                              torch.zeros(2, 4, dtype=I32), ints(2), ints(3)),
                          {"sm_scale": 0.1, "return_lse": True}),
    "odd base": lambda: ("paged_attention", (torch.zeros(513, dtype=BF)[1:].view(2, 4, 64), *pools(),
                                             torch.zeros(2, 4, dtype=I32), torch.zeros(2, dtype=I32)),
                         {"sm_scale": 0.1}),
    "copy": lambda: ("page_copy", (pools(), ints(3), ints(3)), {}),
    "reserve": lambda: ("page_reserve", (ints(2, 4), ints(2), ints(8), ints(2), 16), {}),
    "fork": lambda: ("page_fork", (pools(), ints(2, 4), ints(2), ints(8), ints(1), ints(1)), {}),
    "free": lambda: ("page_free", (ints(2, 4), ints(2), ints(8), apart(2, dtype=torch.bool), 16), {}),
    "dot": lambda: ("dot", (torch.zeros(40, 50, dtype=BF), torch.zeros(50, 60, dtype=BF)),
                    {"acc": torch.zeros(40, 60)}),  # (rows not 16 bytes apart)
    "dot, decode": lambda: ("dot", (torch.zeros(16, 4104, dtype=BF), torch.zeros(4104, 4096, dtype=BF)), {}),
    "dot_scaled": lambda: ("dot_scaled", (torch.zeros(32, 64, dtype=torch.uint8), None, "e4m3",
                                          torch.zeros(64, 40, dtype=torch.uint8), None, "e4m3"), {}),
    "dense attention": lambda: ("attention", (torch.zeros(1, 1, 128, 32, dtype=BF).expand(1, 2, 128, 32),
                                              *[torch.zeros(1, 2, 128, 32, dtype=BF)] * 2, True, 0.5), {}),
    "compact": lambda: ("page_compact", (pools(), ints(2, 4), ints(8)), {}),
}


@pytest.mark.parametrize("current", [0, 5])
@pytest.mark.parametrize("stream", [None, 0, 5, 9])
@pytest.mark.parametrize("name", sorted(CALLS))
def test_memory_of_a_call_is_its_streams(world, name, stream, current):
    """Copies, results and scratch memory are made on the stream that the kernel runs on."""
    world.now = current
    want = current if stream is None else stream
    for _ in range(2):  # the first call of a form, and a later one
        entry, args, kw = CALLS[name]()
        del world.seen[:], world.launched[:]
        with Watch(world):
            getattr(tx, entry)(*args, stream=stream, **kw)
        assert world.launched == [want]
        assert world.seen and all(s == want for _, s in world.seen), world.seen
        assert world.now == current
