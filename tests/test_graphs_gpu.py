"""Captured calls that need a workspace: replayed after larger calls on the same stream, in another
order than captured, with memory allocated and written between the replays."""
import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd as tx  # noqa: E402
from cachecase import Cache, gen, randn, starts  # noqa: E402
from dotcase import say  # noqa: E402

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class Attend:
    """A call over one long sequence, whose keys many workgroups share: parts and counters."""

    def __init__(self, gpu, seed, n, length, Hq=4, D=128):
        self.c = Cache(seed, [length], 16, 1, D, BF, BF).fill()
        self.dev = self.c.to(gpu)
        self.q = randn(gen(seed + 1), n, Hq, D, dtype=BF).to(gpu)
        self.cu, self.scale = starts([n]).to(gpu), D ** -0.5

    def __call__(self):
        return tx.paged_attention(self.q, cu_q=self.cu, sm_scale=self.scale, **self.dev)


def bystanders(gpu):
    """Fills what the allocator has to give in sizes like a workspace's."""
    got = [torch.full((n,), 1.0, device=gpu) for n in (1 << 14, 1 << 20, 1 << 22, 1 << 23, 1 << 24) * 3]
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("warm", [False, True])
def test_replays_after_a_larger_call(gpu, warm):
    say("graph, then a larger call", warm)
    small, large = Attend(gpu, 1, 1, 9000), Attend(gpu, 2, 700, 3000, D=256)
    want = small()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    if warm:
        with torch.cuda.stream(side):
            small()
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = small()
    first = large()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            again = large()
        torch.cuda.synchronize()
        others = bystanders(gpu)
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(again, first)
        assert all(bool((x == 1.0).all()) for x in others)
        del others


def test_graphs_replayed_in_another_order(gpu):
    """Two captures without a call before them, the second replayed first."""
    say("two graphs")
    calls = [Attend(gpu, 3, 1, 12000), Attend(gpu, 4, 3, 15000)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for f in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append([f(), f()])  # (two calls of a capture share its workspace)
        graphs.append(g)
    for i in (1, 1, 0, 1, 0, 0):
        others = bystanders(gpu)
        for o in outs[i]:
            o.zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i]) for o in outs[i]), i
        assert all(bool((x == 1.0).all()) for x in others)
    with torch.cuda.stream(side):
        eager = [f() for f in calls]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, want))


def test_split_dot_in_a_graph(gpu):
    """The decode dot's partials and counters, in a graph that outlives a larger call's workspace."""
    say("dot in a graph")
    g = gen(5)
    a, b = randn(g, 16, 8192, dtype=BF).to(gpu), randn(g, 8192, 8192, dtype=BF).to(gpu)
    big = randn(g, 80, 8192, dtype=BF).to(gpu)
    want = tx.dot(a, b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c = tx.dot(a, b)
    for _ in range(3):
        with torch.cuda.stream(side):
            tx.dot(big, b)
        torch.cuda.synchronize()
        others = bystanders(gpu)
        c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, want)
        assert all(bool((x == 1.0).all()) for x in others)
        del others


def test_pages_in_a_graph_after_larger_books(gpu):
    """page_fork's lists of pages lie in the workspace too."""
    say("fork in a graph")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    kc = randn(gen(6), 64, 4, 1, 8, dtype=BF).to(gpu)
    table = torch.full((6, 4), -1, dtype=torch.int32, device=gpu)
    table[0, :2] = i32([3, 9])
    length, refs = i32([6, 0, 0, 0, 0, 0]), torch.zeros(64, dtype=torch.int32, device=gpu)
    refs[[3, 9]] = 1
    parent, child = i32([0, 0, 0]), i32([2, 4, 5])
    cache = kc.clone()
    want = tx.page_fork([cache], table, length, refs, parent, child)
    torch.cuda.synchronize()
    side, graph, replayed = torch.cuda.Stream(), torch.cuda.CUDAGraph(), kc.clone()
    with torch.cuda.graph(graph, stream=side):
        got = tx.page_fork([replayed], table, length, refs, parent, child)
    many = torch.zeros(1 << 20, dtype=torch.int32, device=gpu)
    for _ in range(3):
        with torch.cuda.stream(side):
            tx.page_reserve(table, length, many, length + 1, 4)
        torch.cuda.synchronize()
        others = bystanders(gpu)
        replayed.copy_(kc)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(replayed, cache)
        assert all(bool((x == 1.0).all()) for x in others)
        del others


def test_a_stream_knows_its_capture(gpu):
    import ctypes
    L, n = tx.load(), ctypes.c_uint64(5)
    side, seen = torch.cuda.Stream(), []
    assert L.tx_stream_capture(side.cuda_stream, ctypes.byref(n)) == tx.OK and n.value == 0
    for _ in range(2):
        graph, x = torch.cuda.CUDAGraph(), torch.zeros(8, device=gpu)
        with torch.cuda.graph(graph, stream=side):
            x.add_(1)
            assert L.tx_stream_capture(side.cuda_stream, ctypes.byref(n)) == tx.OK
            seen.append(n.value)
    assert L.tx_stream_capture(side.cuda_stream, ctypes.byref(n)) == tx.OK and n.value == 0
    assert seen[0] and seen[1] and seen[0] != seen[1]
    assert L.tx_stream_capture(side.cuda_stream, None) == tx.ERR_INVALID
