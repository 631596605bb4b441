"""Calls that name a stream, while torch's current stream is busy: inputs that the call copies first
(strided, off 16 bytes) are copied in the named stream's order."""
import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd as tx  # noqa: E402
from cachecase import Cache, gen, randn, starts  # noqa: E402
from dotcase import say  # noqa: E402

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def busy(gpu):
    x = torch.randn(8192, 8192, device=gpu, dtype=BF)

    def work():
        for _ in range(20):  # some 20 ms
            x @ x
    work()
    torch.cuda.synchronize()
    return work


def both(call, busy):
    """The call on the current stream, and on another while the current one is busy."""
    want = call(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        busy()
        got = call(side.cuda_stream)
        side.synchronize()
        with torch.cuda.stream(side):
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        torch.cuda.synchronize()


def apart(x):
    return torch.stack((x, x), dim=-1)[..., 0]


def odd(x):
    flat = torch.cat((x.new_zeros(1), x.flatten()))
    return flat[1:].view(x.shape)


@pytest.mark.parametrize("lie", [apart, odd])
def test_attention_and_append(gpu, busy, lie):
    say("stream=", lie.__name__)
    c = Cache(1, [4000, 50, 7000], 16, 2, 128, BF, BF).fill()
    n = [30, 1, 2]
    dev = c.to(gpu)
    q, k = lie(randn(gen(2), 33, 8, 128, dtype=BF).to(gpu)), lie(randn(gen(3), 33, 2, 128, dtype=BF).to(gpu))
    f = lie(tx.rotary_frequencies(128)[0].to(gpu))
    books = {t: lie(dev[t]) for t in ("kv_len",)}
    cu = lie(starts(n).to(gpu))
    both(lambda s: tx.paged_attention(q, cu_q=cu, sm_scale=0.1, return_lse=True, stream=s,
                                      **{**dev, **books}), busy)
    pools = [dev["k_cache"].clone(), dev["v_cache"].clone()]
    both(lambda s: (tx.paged_append(k, k, *pools, dev["page_table"], books["kv_len"], cu, q=q,
                                    inv_freq=f, stream=s), *[p.view(torch.int16) for p in pools]), busy)
    pos = lie(torch.arange(33, device=gpu))
    both(lambda s: (tx.rotary(q, pos, f, stream=s),), busy)


def test_books(gpu, busy):
    say("stream=, books")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    table = torch.full((6, 4), -1, dtype=torch.int32, device=gpu)
    table[0, :2] = i32(3, 9)
    length, refs = i32(6, 0, 0, 0, 0, 0), torch.zeros(64, dtype=torch.int32, device=gpu)
    refs[[3, 9]] = 1
    t, n, r = apart(table), apart(length), apart(refs)
    pool = randn(gen(6), 64, 4, 1, 8, dtype=BF).to(gpu)
    src, dst = apart(i32(3, 9)), apart(i32(11, 12))
    drop, more, parent, child = apart(length > 0), apart(length + 5), apart(i32(0)), apart(i32(4))
    both(lambda s: tx.page_reserve(t, n, r, more, 4, stream=s), busy)
    both(lambda s: tx.page_free(t, n, r, drop, 4, stream=s), busy)
    both(lambda s: tx.page_fork([pool], t, n, r, parent, child, stream=s), busy)
    both(lambda s: tx.page_compact([pool], t, r, stream=s), busy)

    def copy(s):
        tx.page_copy([pool], src, dst, stream=s)
        return (pool,)
    both(copy, busy)


@pytest.mark.parametrize("stream", [None, 0])
def test_host_tensors_are_refused(gpu, stream):
    """Before anything is launched, also where the stream is named."""
    kc = torch.zeros(8, 16, 2, 64, dtype=BF)
    t, n, r = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    q, k = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
    for call in (lambda s: tx.rotary(q, n, torch.zeros(32), stream=s),
                 lambda s: tx.paged_append(k, k, kc, kc, t, n, stream=s),
                 lambda s: tx.paged_attention(q, kc, kc, t, n, sm_scale=0.1, stream=s),
                 lambda s: tx.page_copy([kc], n, n, stream=s),
                 lambda s: tx.page_reserve(t, n, r, n, 16, stream=s),
                 lambda s: tx.page_fork([kc], t, n, r, n[:1], n[:1], stream=s),
                 lambda s: tx.page_free(t, n, r, n > 0, 16, stream=s),
                 lambda s: tx.page_compact([kc], t, r, stream=s)):
        with pytest.raises(ValueError):
            call(stream)


def test_dots_and_dense_attention(gpu, busy):
    say("stream=, dots")
    g = gen(7)
    a, b = randn(g, 70, 301, dtype=BF).to(gpu), randn(g, 301, 90, dtype=BF).to(gpu)
    acc = randn(g, 70, 90).to(gpu)
    both(lambda s: (tx.dot(a, b, acc=acc, stream=s),), busy)
    few, wide = randn(g, 16, 4100, dtype=BF).to(gpu), randn(g, 4100, 4096, dtype=BF).to(gpu)
    both(lambda s: (tx.dot(few, wide, stream=s),), busy)
    x, y = (torch.randint(0, 100, n, generator=g).to(torch.uint8).to(gpu) for n in ((40, 64), (64, 72)))
    both(lambda s: (tx.dot_scaled(x, None, "e4m3", y, None, "e4m3", stream=s),), busy)
    q, k = randn(g, 2, 1, 256, 64, dtype=BF).to(gpu).expand(2, 4, 256, 64), randn(g, 2, 4, 256, 64, dtype=BF).to(gpu)
    both(lambda s: tx.attention(q, k, k, True, 0.2, return_lse=True, stream=s), busy)
