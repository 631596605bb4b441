"""Rotary positions, the paged cache and the attention over it against 64-bit oracles on the
CPU, at the sizes and contents where they can go wrong."""
import math

import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd as tx  # noqa: E402
from cachecase import (E4M3, F, Cache, attend64, check, gen, randn, rotate64, rotate_bound,  # noqa: E402
                       starts, u)
from dotcase import say  # noqa: E402

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


# ---- rotary positions -------------------------------------------------------

@pytest.mark.parametrize("shape,rot,dtype", [
    ((1, 1, 2), 2, torch.float32), ((1, 3, 64), 64, BF), ((7, 5, 128), 128, HF),
    ((33, 40, 128), 64, BF), ((130, 2, 80), 20, torch.float32), ((5, 3, 70), 6, HF),
    ((2, 3, 50, 64), 32, BF), ((3, 2, 1, 256), 256, torch.float32), ((0, 3, 64), 64, BF),
    ((2, 0, 5, 64), 64, BF)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(gpu, shape, rot, dtype, interleaved, inverse):
    say("rotary", shape, rot, dtype, interleaved, inverse)
    g = gen(sum(shape) + rot)
    x = randn(g, *shape, dtype=dtype)
    inv_freq, _ = tx.rotary_frequencies(rot)
    N = shape[0] if len(shape) == 3 else shape[2]
    pshape = (N,) if len(shape) == 3 or not inverse else (shape[0], N)
    pos = torch.randint(0, 200000, pshape, generator=g)
    got = tx.rotary(x.to(gpu), pos.to(gpu, torch.int32 if inverse else torch.int64),
                    inv_freq.to(gpu), interleaved=interleaved, scale=1.25, inverse=inverse)
    if len(shape) == 3:
        ref, mag = rotate64(x, pos, inv_freq, interleaved, 1.25, inverse)
    else:
        ref, mag = rotate64(x.transpose(1, 2), pos.expand(shape[0], N), inv_freq, interleaved,
                            1.25, inverse)
        ref, mag = ref.transpose(1, 2), mag.transpose(1, 2)
    check(got, ref, rotate_bound(ref, mag, dtype), "rotary")
    assert torch.equal(got[..., rot:].cpu(), x[..., rot:])  # copied as they are


@pytest.mark.parametrize("far", [0, 2 ** 31 - 1, 2 ** 40])
def test_rotary_far_positions(gpu, far):
    g = gen(5)
    x = randn(g, 3, 2, 64)
    inv_freq, _ = tx.rotary_frequencies(64, scaling="yarn", factor=16.0)
    pos = torch.tensor([far, max(far - 1, 0), far // 2])
    got = tx.rotary(x.to(gpu), pos.to(gpu), inv_freq.to(gpu))
    # the angle's own rounding in 64 bits grows with it
    ref, mag = rotate64(x, pos, inv_freq, False, 1.0)
    check(got, ref, rotate_bound(ref, mag, torch.float32) + mag * far * 2.0 ** -51, "far")


@pytest.mark.parametrize("view", ["broadcast", "qkv", "odd base", "strided last", "in place"])
def test_rotary_views(gpu, view):
    g = gen(6)
    inv_freq, _ = tx.rotary_frequencies(64)
    pos = torch.arange(17)
    out = None
    if view == "broadcast":
        x = randn(g, 17, 1, 64, dtype=BF).to(gpu).expand(17, 4, 64)
    elif view == "qkv":
        x = randn(g, 17, 12, 64, dtype=BF).to(gpu)[:, 2:9]
    elif view == "odd base":
        x = randn(g, 17 * 3 * 64 + 1, dtype=BF).to(gpu)[1:].view(17, 3, 64)
    elif view == "strided last":
        x = randn(g, 17, 3, 128, dtype=BF).to(gpu)[..., ::2]
    else:
        x = randn(g, 17, 3, 64, dtype=BF).to(gpu)
        out = x
    before = x.cpu()
    got = tx.rotary(x, pos.to(gpu), inv_freq.to(gpu), out=out)
    assert out is None or got is out
    ref, mag = rotate64(before, pos, inv_freq, False, 1.0)
    check(got, ref, rotate_bound(ref, mag, BF), view)


def test_rotary_gradient(gpu):
    """The inverse against the formula's gradient and against differences, fp32."""
    g = gen(7)
    x, dy = randn(g, 4, 2, 16), randn(g, 4, 2, 16)
    inv_freq, _ = tx.rotary_frequencies(8)
    pos, scale, f = torch.tensor([0, 3, 77, 4096]), 0.75, inv_freq.to(gpu)
    dx = tx.rotary(dy.to(gpu), pos.to(gpu), f, scale=scale, inverse=True).double().cpu()
    xr = x.double().requires_grad_()
    y, _ = rotate64(xr, pos, inv_freq, False, scale)
    want, = torch.autograd.grad(y, xr, dy.double())
    _, mag = rotate64(dy, pos, inv_freq, False, scale, True)
    check(dx, want, rotate_bound(want, mag, torch.float32), "formula")
    # the map is linear: a difference over a step of 1 has roundings only, 2 of each value
    for i in range(0, x.numel(), 7):
        e = torch.zeros(x.numel())
        e[i] = 1.0
        e = e.view(x.shape)
        up, down = (tx.rotary((x + s * e).to(gpu), pos.to(gpu), f, scale=scale).double().cpu()
                    for s in (0.5, -0.5))
        num = float(((up - down) * dy.double()).sum())
        slack = float(((x.abs() + 1).sum(-1, keepdim=True) * dy.abs()).amax()) * 32 * 12 * F
        assert abs(num - float(dx.flatten()[i])) <= slack


# ---- new tokens into the cache ----------------------------------------------

APPENDS = [
    # n, lens, Hq, Hkv, D, rot, page, dtype, cache, layout
    ([1, 1, 1], [1, 17, 64], 4, 2, 64, 64, 16, BF, BF, "nhd"),
    ([3, 0, 40, 1], [3, 5, 100, 33], 6, 3, 80, 40, 8, HF, HF, "hnd"),
    ([5, 130], [70, 130], 8, 1, 128, 128, 64, BF, E4M3, "nhd"),
    ([2, 2], [9, 2], 0, 2, 64, 0, 4, HF, E4M3, "hnd"),
    ([4, 1], [2, 1], 2, 2, 96, 96, 1, BF, BF, "nhd"),  # kv_len shorter than what is new
    ([1], [300], 5, 5, 256, 128, 128, HF, HF, "nhd"),
    ([3], [3], 2, 1, 14, 6, 16, BF, BF, "nhd"),  # odd pieces: single elements
]


@pytest.mark.parametrize("n,lens,Hq,Hkv,D,rot,page,dtype,cache,layout", APPENDS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(gpu, n, lens, Hq, Hkv, D, rot, page, dtype, cache, layout, interleaved):
    say("append", n, lens, Hq, Hkv, D, rot, page, dtype, cache, layout, interleaved)
    holes = [(0, 0, -1), (len(n) - 1, 0, 10 ** 6)] if len(n) > 1 and page < 16 else []
    c = Cache(1, lens, page, Hkv, D, dtype, cache, layout, holes=holes)
    T = sum(n) + 2  # two rows that belong to no sequence
    qkv = randn(c.g, T, Hq + 2 * Hkv, D, dtype=dtype) * 3
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    inv_freq, scale = tx.rotary_frequencies(rot, scaling="yarn", factor=4.0) if rot else (None, 1.0)
    dev, d = c.to(gpu), qkv.to(gpu)
    got = tx.paged_append(d[:, Hq:Hq + Hkv], d[:, Hq + Hkv:], dev["k_cache"], dev["v_cache"],
                          dev["page_table"], dev["kv_len"], starts(n).to(gpu),
                          q=d[:, :Hq] if Hq else None,
                          inv_freq=None if inv_freq is None else inv_freq.to(gpu),
                          interleaved=interleaved, scale=scale, k_scale=dev["k_scale"],
                          v_scale=dev["v_scale"])
    bits = {1: torch.uint8, 2: torch.int16}[c.k.element_size()]
    want = {t: getattr(c, t).clone() for t in "kv"}
    touched = torch.zeros(c.P, page, dtype=torch.bool)
    t = 0
    for b, m in enumerate(n):
        for i in range(m):
            p = torch.tensor(lens[b] - m + i)
            at = c.place(b, int(p))
            for name, row in (("q", q[t]), ("k", k[t]), ("v", v[t])):
                if rot and name != "v":
                    ref, mag = rotate64(row, p, inv_freq, interleaved, scale)
                    bound = rotate_bound(ref, mag, dtype)
                else:
                    ref, mag = row.double(), torch.zeros(row.shape, dtype=torch.float64)
                    bound = torch.zeros(())
                if name == "q":
                    if Hq:
                        check(got[t], ref, bound, "q")
                    continue
                if at is None:
                    continue
                touched[at] = True
                dev_row = dev[name + "_cache"][at].cpu()
                if cache == E4M3:
                    sc = getattr(c, name + "_scale").double()[:, None]
                    ref, mag = (ref / sc).clamp(-448.0, 448.0), mag / sc
                    bound = u(E4M3) * ref.abs() + 2.0 ** -10 + 12 * F * (mag + ref.abs())
                check(dev_row.to(torch.float64), ref, bound, name)
            t += 1
    if Hq:
        assert torch.equal(got[t:].cpu(), q[t:])
    for name in "kv":  # nothing else has changed
        after = dev[name + "_cache"].cpu()
        assert torch.equal(after[~touched].view(bits), want[name][~touched].view(bits))


# ---- attention over the cache -----------------------------------------------

def attend(gpu, n, lens, Hq, Hkv, D, page, dtype, cache, causal=True, window=0, layout="nhd",
           holes=(), width=0, extra=0, decode=False, seed=3, amp=1.0, view=False):
    say("attend", n, lens, Hq, Hkv, D, page, dtype, cache, causal, window, layout, holes, width)
    c = Cache(seed, lens, page, Hkv, D, dtype, cache, layout, holes=holes, width=width).fill(amp)
    T = sum(n) + extra
    q = randn(c.g, T, Hq, D, dtype=dtype) * amp
    dev = c.to(gpu)
    scale = D ** -0.5
    dq = torch.cat((q, q + 1, q), dim=1).to(gpu)[:, :Hq] if view else q.to(gpu)
    o, lse = tx.paged_attention(dq, cu_q=None if decode else starts(n).to(gpu), sm_scale=scale,
                                causal=causal, window=window, return_lse=True, **dev)
    torch.cuda.synchronize()
    ro, rl, bo, bl = attend64(q, c, n, causal, window, scale)
    check(o, ro, bo, "o")
    check(lse, rl, bl, "lse")
    return c, dev, q, o, lse


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, HF), (BF, E4M3), (HF, E4M3)])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 64), (8, 1, 128), (14, 2, 128), (6, 2, 96),
                                      (16, 2, 256), (3, 1, 16), (40, 1, 80)])
def test_attend_decode(gpu, dtype, cache, Hq, Hkv, D):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 64, 0, 100, 511, 1000]
    attend(gpu, [1] * len(lens), lens, Hq, Hkv, D, 16, dtype, cache, decode=True)


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, HF), (HF, E4M3)])
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (8, 1, 128), (6, 2, 72 + 8), (2, 1, 256),
                                      (5, 5, 32)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 50), (False, 0),
                                           (False, 200)])
def test_attend_ragged(gpu, dtype, cache, Hq, Hkv, D, causal, window):
    n = [0, 1, 5, 33, 64, 200, 3, 0]
    lens = [4, 1, 100, 33, 300, 777, 2, 0]  # (2 of 3: positions before the sequence)
    attend(gpu, n, lens, Hq, Hkv, D, 16, dtype, cache, causal, window, extra=3)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 64, 128, 512])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_attend_page_sizes(gpu, page, layout):
    attend(gpu, [1, 7, 70], [130, 66, 333], 8, 2, 64, page, BF, BF, layout=layout, view=True)
    attend(gpu, [1, 7, 70], [130, 66, 333], 4, 4, 128, page, HF, E4M3, layout=layout, window=90)


def test_attend_holes(gpu):
    """Entries without a page: their tokens are not attended to, whatever the entry says."""
    holes = [(0, 1, -1), (0, 5, 2 ** 31 - 1), (1, 0, -2 ** 31), (1, 1, 10 ** 6), (2, 0, -1)]
    for causal in (True, False):
        attend(gpu, [1, 40, 16], [200, 90, 16], 4, 2, 128, 16, BF, BF, causal, holes=holes)
    attend(gpu, [1, 1], [200, 90], 4, 2, 64, 16, HF, E4M3, holes=holes[:4], decode=True)


def test_attend_table_shorter_than_the_sequence(gpu):
    attend(gpu, [1, 20], [500, 90], 4, 2, 128, 16, BF, BF, width=4)


def test_attend_heads_of_eight_dims(gpu):
    attend(gpu, [1, 20], [50, 90], 4, 2, 8, 16, BF, BF)


@pytest.mark.parametrize("dtype,cache,D", [(BF, BF, 128), (HF, E4M3, 128), (HF, HF, 64),
                                           (BF, BF, 256)])
def test_attend_long(gpu, dtype, cache, D):
    """One sequence whose keys are shared out among many workgroups, next to short ones."""
    attend(gpu, [1, 1, 1], [40001, 3, 700], 8, 2, D, 64, dtype, cache, decode=True)
    attend(gpu, [5, 1, 17], [20011, 3, 700], 8, 2, D, 16, dtype, cache)
    attend(gpu, [100], [9000], 4, 1, D, 32, dtype, cache)


@pytest.mark.parametrize("amp", [0.0, 30.0])
def test_attend_flat_and_peaked(gpu, amp):
    """All scores alike, and scores of thousands: one key takes all."""
    attend(gpu, [1, 70], [900, 500], 4, 1, 128, 16, BF, BF, amp=amp)


def test_attend_many_sequences(gpu):
    g = gen(9)
    lens = torch.randint(0, 60, (700,), generator=g).tolist()
    attend(gpu, [1] * 700, lens, 2, 1, 64, 16, BF, BF, decode=True)
    n = [min(x, i % 4) for i, x in enumerate(lens)]
    attend(gpu, n, lens, 2, 1, 64, 16, BF, BF)


def test_attend_offsets_past_32_bits(gpu):
    """Pages that start more than 2^32 bytes (and 2^31 elements) into the cache."""
    P, page, Hkv, D = 70000, 32, 8, 128
    cache = torch.empty((P, page, Hkv, D), dtype=BF, device=gpu)  # 4.3 GiB
    c = Cache(4, [100, 33], page, Hkv, D, BF, BF).fill()
    ids = [P - 1 - 17 * i for i in range(c.P)]
    table = c.table.clone()
    for i, x in enumerate(ids):
        cache[x] = c.k[i].to(gpu)
        table[c.table == i] = x
    vids = [x for x in ids]
    vcache = torch.empty_like(cache)
    for i, x in enumerate(vids):
        vcache[x] = c.v[i].to(gpu)
    n = [1, 33]
    q = randn(c.g, 34, 16, D, dtype=BF)
    o, lse = tx.paged_attention(q.to(gpu), cache, vcache, table.to(gpu), c.kv_len.to(gpu),
                                starts(n).to(gpu), sm_scale=D ** -0.5, return_lse=True)
    ro, rl, bo, bl = attend64(q, c, n, True, 0, D ** -0.5)
    check(o, ro, bo, "o")
    check(lse, rl, bl, "lse")
    # and written there
    k = randn(c.g, 34, Hkv, D, dtype=BF)
    tx.paged_append(k.to(gpu), k.to(gpu), cache, vcache, table.to(gpu), c.kv_len.to(gpu),
                    starts(n).to(gpu))
    for b, at in ((0, [99]), (1, list(range(33)))):
        for i, j in enumerate(at):
            p = int(table[b, j // page])
            assert torch.equal(cache[p, j % page].cpu(), k[b + i])


def test_attend_twice_alike_and_on_streams(gpu):
    """The same call twice gives the same bits; calls on two streams do not disturb each other."""
    c, dev, q, o, lse = attend(gpu, [1, 9], [30000, 800], 8, 2, 128, 16, BF, BF)
    cu, dq = starts([1, 9]).to(gpu), q.to(gpu)
    call = lambda: tx.paged_attention(dq, cu_q=cu, sm_scale=128 ** -0.5, return_lse=True, **dev)  # noqa: E731
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(call())
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, o) and torch.equal(b, lse)


def test_step_in_a_graph(gpu):
    """Reserve, append and attend captured once and replayed as the sequences grow."""
    page, Hq, Hkv, D, B = 4, 4, 2, 64, 3
    g = gen(11)
    P, W = 64, 16
    inv_freq = tx.rotary_frequencies(D)[0].to(gpu)
    kc, vc = (torch.zeros(P, page, Hkv, D, dtype=BF, device=gpu) for _ in range(2))
    table = torch.full((B, W), -1, dtype=torch.int32, device=gpu)
    length = torch.tensor([0, 5, 3], dtype=torch.int32, device=gpu)
    refs = torch.zeros(P, dtype=torch.int32, device=gpu)
    table, length, refs, _ = tx.page_reserve(table, torch.zeros_like(length), refs, length, page)
    qkv = torch.zeros(B, Hq + 2 * Hkv, D, dtype=BF, device=gpu)

    def step(table, length, refs, kc, vc):
        t, n, r, missing = tx.page_reserve(table, length, refs, length + 1, page,
                                           out=(table, length, refs))
        q = tx.paged_append(qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], kc, vc, t, n, q=qkv[:, :Hq],
                            inv_freq=inv_freq)
        return tx.paged_attention(q, kc, vc, t, n, sm_scale=D ** -0.5), missing

    eager = [x.clone() for x in (table, length, refs, kc, vc)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*[x.clone() for x in eager])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o, missing = step(table, length, refs, kc, vc)
    for _ in range(9):
        qkv.copy_(randn(g, *qkv.shape, dtype=BF))
        want, short = step(*eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and int(missing) == int(short) == 0
        for a, b in zip((table, length, refs, kc, vc), eager):
            assert torch.equal(a, b)
    assert length.tolist() == [9, 14, 12]


# ---- pages ------------------------------------------------------------------

class Books:
    """The books by the rules, one entry after the other."""

    def __init__(self, seed, S, W, P, page, fill=0.5):
        g = gen(seed)
        self.page = page
        self.refs = [0] * P
        self.table = [[-1] * W for _ in range(S)]
        self.len = [0] * S
        order = torch.randperm(P, generator=g).tolist()
        for s in range(S):
            n = int(torch.randint(0, W * page + 1, (1,), generator=g))
            k = -(-n // page)
            if len(order) - k < P * (1 - fill):
                continue
            self.len[s] = n
            for w in range(k):
                p = order.pop()
                self.table[s][w] = p
                self.refs[p] = 1

    def to(self, dev):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        return i32(self.table).view(len(self.len), -1), i32(self.len), i32(self.refs)

    def take(self):
        for p, r in enumerate(self.refs):
            if r == 0:
                self.refs[p] = 1
                return p
        return None

    def reserve(self, new):
        W, missing = len(self.table[0]), 0
        free = [p for p, r in enumerate(self.refs) if r == 0]
        for s, n in enumerate(new):
            n = max(self.len[s], min(n, W * self.page))
            for w in range(-(-self.len[s] // self.page), -(-n // self.page)):
                if free:
                    self.table[s][w] = free.pop(0)
                    self.refs[self.table[s][w]] = 1
                else:
                    self.table[s][w] = -1
                    missing += 1
            self.len[s] = n
        return missing

    def fork(self, pairs):
        copies, missing, S = [], 0, len(self.len)
        free = [p for p, r in enumerate(self.refs) if r == 0]
        for a, c in pairs:
            if not (0 <= a < S and 0 <= c < S):
                continue
            used = -(-self.len[a] // self.page)
            row = self.table[a][:used] + [-1] * (len(self.table[a]) - used)
            if self.len[a] % self.page:
                old = row[used - 1]
                row[used - 1] = free.pop(0) if free else -1
                if row[used - 1] < 0:
                    missing += 1
                else:
                    copies.append((old, row[used - 1]))
            for p in row[:used]:
                if p >= 0:
                    self.refs[p] += 1
            self.table[c], self.len[c] = row, self.len[a]
        return copies, missing

    def free(self, drop):
        for s, d in enumerate(drop):
            if d:
                for w in range(-(-self.len[s] // self.page)):
                    if self.table[s][w] >= 0:
                        self.refs[self.table[s][w]] -= 1
                self.table[s] = [-1] * len(self.table[s])
                self.len[s] = 0

    def compact(self):
        U = sum(r > 0 for r in self.refs)
        holes = [p for p in range(U) if self.refs[p] == 0]
        movers = [p for p in range(U, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return list(to.items())


def same(books, table, length, refs):
    t, n, r = books.to("cpu")
    assert torch.equal(table.cpu(), t)
    assert length is None or torch.equal(length.cpu(), n)
    assert torch.equal(refs.cpu(), r)


@pytest.mark.parametrize("S,W,P,page", [(1, 1, 1, 1), (3, 5, 40, 4), (70, 30, 5000, 16),
                                        (1500, 3, 6000, 2), (20, 64, 600, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_pages_reserve_and_free(gpu, S, W, P, page, in_place):
    say("reserve", S, W, P, page, in_place)
    b = Books(S + W, S, W, P, page)
    g = gen(1)
    for _ in range(3):
        t, n, r = b.to(gpu)
        new = torch.randint(-3, W * page + 9, (S,), generator=g).tolist()
        out = (t, n, r) if in_place else None
        got = tx.page_reserve(t, n, r, torch.tensor(new, dtype=torch.int32, device=gpu), page,
                              out=out)
        missing = b.reserve(new)
        same(b, *got[:3])
        assert int(got[3]) == missing
        drop = (torch.rand(S, generator=g) < 0.4)
        t, n, r = b.to(gpu)
        got = tx.page_free(t, n, r, drop.to(gpu), page, out=(t, n, r) if in_place else None)
        b.free(drop.tolist())
        same(b, *got)


@pytest.mark.parametrize("S,W,P,page,caches,heads", [
    (2, 1, 8, 4, 1, 1), (12, 9, 300, 8, 3, 2), (40, 6, 130, 16, 2, 1), (1100, 2, 1700, 2, 1, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_pages_fork_free_compact(gpu, S, W, P, page, caches, heads, in_place):
    """Forked sequences share pages; freed, the pages are kept for who is left; compacted,
    what a sequence reads stays the same."""
    say("fork", S, W, P, page, caches, heads, in_place)
    b = Books(S, S, W, P, page, fill=0.8)
    half = S // 2
    drop = [s >= half for s in range(S)]
    b.free(drop)
    g = gen(2)
    data = [randn(g, P, page, heads, 16, dtype=BF) for _ in range(caches)]
    dev = [x.to(gpu) for x in data]
    pairs = [(int(torch.randint(0, half, (1,), generator=g)), s) for s in range(half, S)]
    pairs[0:0] = [(-1, half), (S, half)]  # no such sequence: skipped
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    t, n, r = b.to(gpu)
    got = tx.page_fork(dev, t, n, r, i32([a for a, _ in pairs]), i32([c for _, c in pairs]),
                       out=(t, n, r) if in_place else None)
    copies, missing = b.fork(pairs)
    same(b, *got[:3])
    assert int(got[3]) == missing
    for x in data:
        for a, c in copies:
            x[c] = x[a]
    for x, y in zip(data, dev):
        assert torch.equal(x, y.cpu())
    drop = torch.rand(S, generator=g) < 0.6
    t, n, r = tx.page_free(*got[:3], drop.to(gpu), page)
    b.free(drop.tolist())
    same(b, t, n, r)
    t, r, moved = tx.page_compact(dev, t, r, out=(t, r) if in_place else None)
    moves = b.compact()
    same(b, t, n, r)
    assert int(moved) == len(moves)
    for x in data:
        for a, c in moves:
            x[c] = x[a]
    for x, y in zip(data, dev):
        assert torch.equal(x, y.cpu())
    used = sum(k > 0 for k in b.refs)
    assert all(k > 0 for k in b.refs[:used])


def test_page_copy(gpu):
    g = gen(3)
    a, b = randn(g, 50, 16, 2, 24, dtype=BF), randn(g, 50, 3, 4096, dtype=torch.float32)
    b8 = torch.zeros(50, 5, 16, dtype=torch.uint8)
    dev = [a.to(gpu), b.to(gpu), b8.to(gpu)]
    src, dst = [0, 1, 7, -1, 50, 9, 8], [49, 40, 41, 3, 4, -5, 8]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    tx.page_copy(dev, i32(src), i32(dst))
    for x, y in zip((a, b, b8), dev):
        for s, d in ((0, 49), (1, 40), (7, 41)):
            x[d] = x[s]
        assert torch.equal(x, y.cpu())
    tx.page_copy(dev, i32([]), i32([]))
    tx.page_copy([], i32([1]), i32([2]))


def test_generation_matches_attention_without_a_cache(gpu):
    """A prompt in chunks, then tokens one by one, against softmax over all of it at once."""
    g = gen(12)
    page, Hq, Hkv, D, N = 16, 8, 2, 64, 150
    inv_freq, _ = tx.rotary_frequencies(D)
    q, k, v = (randn(g, N, h, D, dtype=BF) for h in (Hq, Hkv, Hkv))
    kc, vc = (torch.full((20, page, Hkv, D), math.nan, dtype=BF, device=gpu) for _ in range(2))
    table = torch.full((1, 12), -1, dtype=torch.int32, device=gpu)
    length = torch.zeros(1, dtype=torch.int32, device=gpu)
    refs = torch.zeros(20, dtype=torch.int32, device=gpu)
    got, at, pos = [], 0, torch.arange(N)
    for m in [70, 41, 30] + [1] * 9:
        table, length, refs, missing = tx.page_reserve(table, length, refs, length + m, page)
        rows = slice(at, at + m)
        cu = starts([m]).to(gpu)
        qr = tx.paged_append(k[rows].to(gpu), v[rows].to(gpu), kc, vc, table, length, cu,
                             q=q[rows].to(gpu), inv_freq=inv_freq.to(gpu))
        got.append(tx.paged_attention(qr, kc, vc, table, length, cu, sm_scale=D ** -0.5))
        at += m
    # the same from the rotated, rounded q and k
    c = Cache(0, [N], page, Hkv, D, BF, BF)
    c.k, c.v, c.table, c.P = kc.cpu(), vc.cpu(), table.cpu(), 20
    c.W = 12
    rq, mag = rotate64(q, pos, inv_freq, False, 1.0)
    qr = tx.rotary(q.to(gpu), pos.to(gpu), inv_freq.to(gpu)).cpu()
    check(qr, rq, rotate_bound(rq, mag, BF), "q")
    o, _, bo, _ = attend64(qr, c, [N], True, 0, D ** -0.5)
    check(torch.cat(got), o, bo, "o")
    assert int(missing) == 0
