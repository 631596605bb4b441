"""The paged cache held in 4 bits against 64-bit oracles on the CPU: what append writes, what read
gives back, the attention over it, at the sizes and contents where they can go wrong."""
import math
import os
import sys

import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd as tx  # noqa: E402
from cache4case import BLOCK, MANY_THREADS, Cache4, nearest, quantise, scale_bytes, scale_values, values  # noqa: E402
from cachecase import E4M3, F, Cache, attend64, check, gen, randn, rotate64, rotate_bound, starts  # noqa: E402
from dotcase import say  # noqa: E402

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def books(dev):
    return {k: dev[k] for k in ("k_cache", "v_cache", "page_table", "kv_len", "k_scale", "v_scale",
                                "k_block_scale", "v_block_scale")}


def raw(t):
    return t.view(torch.uint8).cpu()


def sequences(n):
    """(sequence, place) of every row."""
    return [(b, i) for b, k in enumerate(n) for i in range(k)]


# ---- new tokens into the cache ----------------------------------------------

def awkward(g, T, H, D, dtype):
    """Values whose quotients lie on and next to the codes' borders, zeros of both signs, tiny and
    huge ones."""
    x = randn(g, T, H, D)
    step = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0])
    pick = torch.randint(0, 16, x.shape, generator=g)
    e = torch.randint(-6, 6, (T, H, 1), generator=g).float()
    near = step[pick] * torch.sign(x) * 2.0 ** e * (1 + torch.randint(-1, 2, x.shape, generator=g) * 2.0 ** -7)
    x = torch.where(torch.arange(T)[:, None, None] % 3 == 0, near, x)
    x[:, :, 1::7] = -0.0
    if T > 4:
        top = torch.finfo(dtype).max
        x[1, :, :D // 2] = top * torch.sign(x[1, :, :D // 2])
        x[2] *= torch.finfo(dtype).tiny / 4
        x[3] = 0.0
        x[4, :, 1::2] *= 1e-3
    return x.to(dtype)


APPENDS = [
    # n, lens, Hkv, D, page, dtype, layout
    ([1, 1, 1], [1, 17, 64], 2, 64, 16, BF, "hnd"),
    ([3, 0, 40, 1], [3, 5, 100, 33], 3, 96, 8, HF, "nhd"),
    ([5, 130], [70, 130], 1, 128, 64, BF, "nhd"),
    ([2, 2], [9, 2], 2, 32, 4, HF, "hnd"),
    ([4, 1], [2, 1], 2, 160, 1, BF, "nhd"),  # kv_len shorter than what is new
    ([7], [300], 5, 256, 128, HF, "hnd"),
    ([6, 3], [6, 40], 1, 288, 2, BF, "hnd"),
]


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("n,lens,Hkv,D,page,dtype,layout", APPENDS)
def test_append_is_the_nearest_code(gpu, n, lens, Hkv, D, page, dtype, layout, scaled, kind):
    """Without a rotation every code and every scale is the oracle's, and nothing else is written."""
    say("append4", n, lens, Hkv, D, page, dtype, layout, scaled, kind)
    holes = [(0, 0, -1), (len(n) - 1, 0, 10 ** 6)] if len(n) > 1 and page < 16 else []
    c = Cache4(1, lens, page, Hkv, D, dtype, kind, layout, holes=holes, scaled=scaled)
    T = sum(n) + 2  # two rows that belong to no sequence
    kv = awkward(c.g, T, 2 * Hkv, D, dtype)
    if T > 8:
        kv[5, 0, 3], kv[6, -1, D - 1] = math.nan, -math.inf
    dev = c.to(gpu)
    d = kv.to(gpu)
    assert tx.paged_append(d[:, :Hkv], d[:, Hkv:], cu_q=starts(n).to(gpu), **books(dev)) is None
    for which, x in (("k", kv[:, :Hkv]), ("v", kv[:, Hkv:])):
        y = x.float()
        scale = c.k_scale if which == "k" else c.v_scale
        if scale is not None:
            y = y / scale[:, None]
        codes, sb = quantise(y.double(), kind, dtype)
        for t, (b, i) in enumerate(sequences(n)):
            c.put(which, b, lens[b] - n[b] + i, codes[t], sb[t])
    for name, want in (("k_cache", c.k), ("v_cache", c.v), ("k_block_scale", c.kb), ("v_block_scale", c.vb)):
        got = raw(dev[name])
        assert torch.equal(got, want), (name, int((got != want).sum()))


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,lens,Hq,Hkv,D,rot,page,dtype,layout", [
    ([1, 1, 1], [1, 17, 6400], 4, 2, 64, 64, 16, BF, "hnd"),
    ([3, 0, 40, 1], [3, 5, 100, 33], 6, 3, 96, 40, 8, HF, "nhd"),  # halves of 20: no whole pieces
    ([50, 9], [7000, 9], 8, 8, 128, 128, 64, BF, "hnd"),
    ([2, 2], [9, 2], 0, 2, 64, 32, 4, HF, "nhd"),
    ([4, 30], [2, 300], 1, 1, 256, 12, 32, BF, "hnd"),
])
def test_append_rotated(gpu, n, lens, Hq, Hkv, D, rot, page, dtype, layout, interleaved, kind):
    """Rotated keys are off by the rotation's roundings before they are quantised, so a scale is that
    of a largest magnitude this far off, and a code one of those next to the value under its scale."""
    say("append4 rotated", n, lens, Hq, Hkv, D, rot, page, dtype, layout, interleaved, kind)
    c = Cache4(2, lens, page, Hkv, D, dtype, kind, layout)
    T = sum(n) + 1
    qkv = randn(c.g, T, Hq + 2 * Hkv, D, dtype=dtype) * 3
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv]
    inv_freq, scale = tx.rotary_frequencies(rot, scaling="yarn", factor=4.0)
    dev, d = c.to(gpu), qkv.to(gpu)
    got = tx.paged_append(d[:, Hq:Hq + Hkv], d[:, Hq + Hkv:], cu_q=starts(n).to(gpu),
                          q=d[:, :Hq] if Hq else None, inv_freq=inv_freq.to(gpu),
                          interleaved=interleaved, scale=scale, **books(dev))
    seq = sequences(n)
    pos = torch.tensor([lens[b] - n[b] + i for b, i in seq])
    live = len(seq)
    if Hq:
        ref, mag = rotate64(q[:live], pos, inv_freq, interleaved, scale)
        check(got[:live], ref, rotate_bound(ref, mag, dtype), "q")
        assert torch.equal(got[live:].cpu(), q[live:])
    y, mag = rotate64(k[:live], pos, inv_freq, interleaved, scale)
    off = rotate_bound(torch.zeros_like(y), mag, torch.float32) + F * y.abs()  # rounded to fp32
    off = torch.where(torch.arange(D) < rot, off, 0.0)
    codes, sb = raw(dev["k_cache"]), raw(dev["k_block_scale"])
    for t, (b, i) in enumerate(seq):
        at = c.place(b, lens[b] - n[b] + i)
        if at is None:
            continue
        a = y[t].abs().unflatten(-1, (-1, BLOCK[kind]))
        o = off[t].unflatten(-1, (-1, BLOCK[kind]))
        least = scale_bytes((a - o).amax(-1).clamp(min=0.0), kind, dtype).int()
        most = scale_bytes((a + o).amax(-1), kind, dtype).int()
        s = sb[at].int()
        assert bool(((s >= least) & (s <= most)).all()), (t, b, i)
        # the code's magnitude between those of the value, less and more
        unit = scale_values(sb[at], kind)[..., None]
        z = y[t].unflatten(-1, (-1, BLOCK[kind]))
        lo, hi = ((nearest(((z + w * o).abs() / unit)) * torch.where(torch.signbit(z + w * o), -1, 1))
                  for w in (-1.0, 1.0))
        nib = torch.stack((codes[at] & 15, codes[at] >> 4), -1).flatten(-2).int()
        x = ((nib & 7) * torch.where(nib >= 8, -1, 1)).unflatten(-1, (-1, BLOCK[kind]))
        assert bool(((x >= lo) & (x <= hi)).all()), (t, b, i)
    # v is not rotated
    want, _ = quantise(qkv[:, Hq + Hkv:].double(), kind, dtype)
    vc = raw(dev["v_cache"])
    for t, (b, i) in enumerate(seq):
        at = c.place(b, lens[b] - n[b] + i)
        assert at is None or torch.equal(vc[at], want[t])


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("Hq,Hkv,D,rot,interleaved", [(8, 2, 128, 128, False), (8, 2, 64, 32, True),
                                                      (12, 3, 96, 40, False), (6, 2, 128, 76, False)])
def test_append_rotates_step_by_step(gpu, Hq, Hkv, D, rot, interleaved, kind):
    """Sines rounded once to fp32, products and their sum each rounded to fp32: keys at a border of two
    codes go where these steps lead.  (An angle off by 2^-51 changes a sine's rounding once in 2^26, and that
    a value's once in 2^12: of 2 million values none.)"""
    n, lens = [1500, 1, 500], [30000, 7, 3000]
    c = Cache4(31, lens, 16, Hkv, D, HF, kind, "hnd")
    qkv = randn(c.g, sum(n), Hq + 2 * Hkv, D, dtype=HF)
    inv_freq, scale = tx.rotary_frequencies(rot)
    assert scale == 1.0
    dev, d = c.to(gpu), qkv.to(gpu)
    got = tx.paged_append(d[:, Hq:Hq + Hkv], d[:, Hq + Hkv:], cu_q=starts(n).to(gpu), q=d[:, :Hq],
                          inv_freq=inv_freq.to(gpu), interleaved=interleaved, **books(dev))
    pos = torch.cat([torch.arange(lens[b] - k, lens[b]) for b, k in enumerate(n)])
    angle = pos.double()[:, None] * inv_freq.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = qkv[:, :Hq + Hkv].float()
    i, j = ((slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot)))
    a, z = y[..., i].clone(), y[..., j].clone()
    y[..., i], y[..., j] = a * cos - z * sin, z * cos + a * sin
    assert torch.equal(got.cpu(), y[:, :Hq].to(HF))
    codes, sb = quantise(y[:, Hq:].double(), kind, HF)
    k, _ = tx.paged_read(cu_q=starts(n).to(gpu), tokens=sum(n), dtype=torch.float32, **books(dev))
    assert torch.equal(k.cpu().double(), values(codes, sb, kind))


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("Hq,D,rot,interleaved,odd", [
    (4, 64, 32, False, False), (4, 64, 64, False, False), (5, 96, 96, False, False), (16, 96, 40, False, False),
    (4, 64, 0, False, False), (4, 64, 32, False, True), (33, 96, 96, False, True), (4, 64, 32, True, False),
    (300, 128, 16, False, False), (2, 4128, 4128, False, False)])
def test_append_in_place(gpu, Hq, D, rot, interleaved, odd, kind):
    """q_out may be q: what comes back is what a tensor of its own gets."""
    n = [3, 1, 7, 30]
    c = Cache4(5, [9, 1, 20, 31], 4, 1, D, BF, kind)
    T = sum(n) + 1
    store = randn(c.g, T * (Hq + 2) * D + 1, dtype=BF)[int(odd):]
    y = store[:T * (Hq + 2) * D].view(T, Hq + 2, D)
    freq = tx.rotary_frequencies(rot)[0].to(gpu) if rot else None

    def run(own):
        dev = c.to(gpu)
        d = torch.empty(T * (Hq + 2) * D + 8, dtype=BF, device=gpu)[int(odd):][:y.numel()].view(y.shape).copy_(y)
        q = d[:, :Hq]
        out = torch.empty(T, Hq, D, dtype=BF, device=gpu) if own else q
        got = tx.paged_append(d[:, Hq:Hq + 1], d[:, Hq + 1:], cu_q=starts(n).to(gpu), q=q, inv_freq=freq,
                              interleaved=interleaved, q_out=out, **books(dev))
        assert got is out
        return [out.clone()] + [raw(dev[x]) for x in ("k_cache", "v_cache", "k_block_scale", "v_block_scale")]

    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("lie", ["odd base", "odd strides", "strided last", "broadcast"])
def test_append_views(gpu, lie, kind):
    """Tokens that are not read 16 bytes at a time, and scales in an order of their own."""
    c = Cache4(3, [5, 9], 8, 2, 64, BF, kind)
    T, dev = 6, c.to(gpu)
    n = [2, 4]
    if lie == "odd base":
        store = randn(c.g, T * 4 * 64 + 1, dtype=BF)
        make = lambda s: s[1:].view(T, 4, 64)  # noqa: E731
    elif lie == "odd strides":
        store = randn(c.g, T, 4, 65, dtype=BF)
        make = lambda s: s[..., :64]  # noqa: E731
    elif lie == "strided last":
        store = randn(c.g, T, 4, 128, dtype=BF)
        make = lambda s: s[..., ::2]  # noqa: E731
    else:
        store = randn(c.g, T, 1, 64, dtype=BF)
        make = lambda s: s.expand(T, 4, 64)  # noqa: E731
    kv, d = make(store), make(store.to(gpu))
    for name in ("k_block_scale", "v_block_scale"):  # tokens last, every second byte
        t = dev[name]
        wide = torch.empty(t.shape[0], t.shape[3], t.shape[2], 2 * t.shape[1], dtype=t.dtype, device=gpu)
        wide.view(torch.uint8).fill_(9)
        dev[name] = wide.permute(0, 3, 2, 1)[:, ::2]
        dev[name].view(torch.uint8).copy_(t.view(torch.uint8))
    tx.paged_append(d[:, :2], d[:, 2:], cu_q=starts(n).to(gpu), **books(dev))
    for which, x in (("k", kv[:, :2]), ("v", kv[:, 2:])):
        codes, sb = quantise(x.double(), kind, BF)
        for t, (b, i) in enumerate(sequences(n)):
            c.put(which, b, c.lens[b] - n[b] + i, codes[t], sb[t])
    for name, want in (("k_cache", c.k), ("v_cache", c.v), ("k_block_scale", c.kb), ("v_block_scale", c.vb)):
        assert torch.equal(raw(dev[name]), want), name
    k, v = tx.paged_read(cu_q=starts(n).to(gpu), tokens=T, dtype=torch.float32, **books(dev))
    for got, x in ((k, kv[:, :2]), (v, kv[:, 2:])):
        codes, sb = quantise(x.double(), kind, BF)
        assert torch.equal(got.cpu().double(), values(codes, sb, kind))


# ---- tokens out of a cache --------------------------------------------------

READS = [
    # n, lens, Hkv, D, page, layout
    ([1, 1, 1], [1, 17, 64], 2, 64, 16, "hnd"),
    ([3, 0, 40, 1], [3, 5, 100, 33], 3, 96, 8, "nhd"),
    ([5, 130], [70, 130], 1, 128, 64, "hnd"),
    ([4, 1, 2], [2, 1, -3], 2, 160, 1, "nhd"),  # more rows than tokens
    ([300], [300], 2, 256, 4, "hnd"),
]


@pytest.mark.parametrize("out", [BF, HF, torch.float32])
@pytest.mark.parametrize("kind", ["mx", "nv", BF, HF, E4M3])
@pytest.mark.parametrize("n,lens,Hkv,D,page,layout", READS)
def test_read(gpu, n, lens, Hkv, D, page, layout, kind, out):
    say("read", n, lens, Hkv, D, page, layout, kind, out)
    holes = [(0, 0, -1), (len(n) - 1, 0, 10 ** 6)] if len(n) > 1 and page < 16 else []
    held = [max(x, 0) for x in lens]
    if isinstance(kind, str):
        c = Cache4(5, held, page, Hkv, D, BF, kind, layout, holes=holes, scaled=True).fill(2.0)
    else:
        c = Cache(5, held, page, Hkv, D, kind, kind, layout, holes=holes).fill(2.0)
    c.lens, c.kv_len = list(lens), torch.tensor(lens, dtype=torch.int32)
    T, dev = sum(n) + 3, c.to(gpu)
    cu = starts(n).to(gpu)
    k, v = tx.paged_read(cu_q=cu, tokens=T, dtype=out, **dev)
    # rows of a larger tensor, in an order of their own, as outputs
    big = torch.full((T, Hkv, 2, D), 7.0, dtype=out, device=gpu)
    k2, v2 = tx.paged_read(cu_q=cu, k_out=big[:, :, 0], v_out=big[:, :, 1], **dev)
    assert k2.data_ptr() == big.data_ptr() and torch.equal(k2, k) and torch.equal(v2, v)
    odd = torch.empty(T * Hkv * D + 1, dtype=out, device=gpu)[1:].view(T, Hkv, D)
    k3, v3 = tx.paged_read(cu_q=cu, tokens=T, k_out=odd, dtype=out, **dev)
    assert torch.equal(k3, k) and torch.equal(v3, v)
    for which, got in (("k", k), ("v", v)):
        got = got.cpu()
        assert got.dtype == out
        for t in range(T):
            b, i = sequences(n)[t] if t < sum(n) else (0, 0)
            j = c.lens[b] - n[b] + i
            x = torch.zeros(Hkv, D, dtype=torch.float64)
            if t < sum(n) and c.place(b, j) is not None:
                x = c.rows(which, b)[0][j]
            # products of 24 bits with a head's factor: rounded to fp32, then to the type
            assert torch.equal(got[t], x.float().to(out)), (which, t)
    if max(n) == 1 and not holes:
        one = tx.paged_read(dtype=out, **dev)
        assert torch.equal(one[0], k[:len(n)]) and torch.equal(one[1], v[:len(n)])


@pytest.mark.parametrize("cache,D,page", [(BF, 14, 16), (E4M3, 33, 4), (HF, 1, 1), (E4M3, 8, 8)])
def test_read_odd_heads(gpu, cache, D, page):
    c = Cache(6, [20, 7], page, 3, D, cache if cache != E4M3 else BF, cache).fill()
    dev = c.to(gpu)
    k, v = tx.paged_read(cu_q=starts([20, 7]).to(gpu), tokens=27, dtype=torch.float32, **dev)
    for which, got in (("k", k), ("v", v)):
        want = torch.cat([c.rows(which, b)[0] for b in (0, 1)]).float()
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("kind", ["mx", "nv"])
def test_read_every_code_and_scale(gpu, kind):
    """All 256 scales, in fp32 and rounded to the types."""
    B = 32 // BLOCK[kind]
    codes = torch.arange(16, dtype=torch.uint8).repeat(2)
    codes = (codes[0::2] | codes[1::2] << 4).expand(256, 1, 1, 16).contiguous()
    sb = torch.arange(256, dtype=torch.uint8).view(256, 1, 1, 1).expand(256, 1, 1, B).contiguous()
    table = torch.arange(256, dtype=torch.int32).view(256, 1)
    length = torch.ones(256, dtype=torch.int32)
    want = values(codes, sb, kind).view(256, 1, 32)
    dev = [t.to(gpu) for t in (codes, sb, table, length)]
    s = dev[1] if kind == "mx" else dev[1].view(E4M3)
    for out in (torch.float32, BF, HF):
        k, v = tx.paged_read(dev[0], dev[0], dev[2], dev[3], dtype=out, k_block_scale=s, v_block_scale=s)
        assert torch.equal(k, v) or bool(k.isnan().any())
        # (2^-127 and 6 * 2^127 are fp32's as well)
        ref = want.float().to(out)
        same = (k.cpu() == ref) | (k.cpu().isnan() & ref.isnan())
        assert bool(same.all()), (out, torch.nonzero(~same)[:4])


@pytest.mark.parametrize("kind", ["mx", "nv"])
def test_read_every_code_and_scale_of_both(gpu, kind):
    """As before, with codes and scales of their own in K and V, and every one of both compared."""
    B = 32 // BLOCK[kind]
    codes = torch.arange(16, dtype=torch.uint8).repeat(2)
    kc = (codes[0::2] | codes[1::2] << 4).expand(256, 1, 1, 16).contiguous()
    vc = kc.flip(-1).contiguous()
    ks = torch.arange(256, dtype=torch.uint8).view(256, 1, 1, 1).expand(256, 1, 1, B).contiguous()
    vs = ks.flip(0).contiguous()
    table, length = torch.arange(256, dtype=torch.int32).view(256, 1), torch.ones(256, dtype=torch.int32)
    byte = torch.uint8 if kind == "mx" else E4M3
    for out in (torch.float32, BF, HF):
        got = tx.paged_read(kc.to(gpu), vc.to(gpu), table.to(gpu), length.to(gpu), dtype=out,
                            k_block_scale=ks.to(gpu).view(byte), v_block_scale=vs.to(gpu).view(byte))
        for x, c, s in zip(got, (kc, vc), (ks, vs)):
            ref = values(c, s, kind).view(256, 1, 32).float().to(out)
            same = (x.cpu() == ref) | (x.cpu().isnan() & ref.isnan())
            assert bool(same.all()), (out, torch.nonzero(~same)[:4])


# ---- attention over the cache -----------------------------------------------

def small_weights(c, n, bo):
    """What weights below fp16's normal range add to bounds of bf16 rows under e4m3 scales, whose
    products are taken in fp16: half its least step, 2^-25, for each key, relative to a sum of
    weights of at least 1 (the reference is a score of the row)."""
    if c.kind != "nv":
        return bo
    bo, at, G = bo.clone(), 0, bo.shape[1] // c.Hkv
    for b, k in enumerate(n):
        V, _ = c.rows("v", b)
        bo[at:at + k] += 2.0 ** -25 * V.abs().sum(0).repeat_interleave(G, 0)
        at += k
    return bo


def attend(gpu, n, lens, Hq, Hkv, D, page, dtype, kind, causal=True, window=0, layout="hnd", holes=(),
           width=0, extra=0, decode=False, scale=None, amp=1.0, scaled=False, q_amp=1.0, views=False):
    say("attend4", n if len(n) < 9 else len(n), lens if len(lens) < 9 else len(lens), Hq, Hkv, D, page, dtype,
        kind, causal, window, layout, scaled)
    c = Cache4(3, lens, page, Hkv, D, dtype, kind, layout, holes=holes, width=width, scaled=scaled).fill(amp)
    T = sum(n) + extra
    q = (randn(c.g, T, Hq, D) * q_amp).to(dtype)
    scale = D ** -0.5 if scale is None else scale
    dev = c.to(gpu)
    cu = None if decode else starts(n).to(gpu)
    o, lse = tx.paged_attention(q.to(gpu), cu_q=cu, sm_scale=scale, causal=causal, window=window,
                                return_lse=True, **books(dev))
    ro, rl, bo, bl = attend64(q, c, n, causal, window, scale)
    check(o, ro, small_weights(c, n, bo), "o")
    check(lse, rl, bl, "lse")
    return c, dev, q, o, lse


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 1, 64), (8, 8, 64), (16, 2, 128), (5, 5, 32), (6, 2, 96), (8, 1, 256),
                                      (3, 1, 160), (32, 1, 128)])
def test_attend_decode(gpu, dtype, kind, Hq, Hkv, D):
    attend(gpu, [1] * 5, [1, 31, 32, 33, 700], Hq, Hkv, D, 16, dtype, kind, decode=True)


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 40), (False, 7)])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 1, 128), (2, 2, 256), (3, 3, 96)])
def test_attend_ragged(gpu, dtype, kind, Hq, Hkv, D, causal, window):
    attend(gpu, [5, 0, 64, 1, 33], [5, 40, 200, 0, 90], Hq, Hkv, D, 16, dtype, kind, causal, window,
           "nhd", extra=3)


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("rows", [15, 16, 17, 32, 33, 128, 129, 300])
def test_rows_of_a_sequence(gpu, rows, D, kind):
    """New tokens times heads of a kv head: at and past the rows of a unit in each form."""
    G = 1 if rows % 3 else 3
    n = rows // G
    attend(gpu, [n, 1, n], [n + 75, 1, 700], 2 * G, 2, D, 16, BF, kind)
    attend(gpu, [n], [n + 40], 2 * G, 2, D, 16, BF, kind, window=33, scaled=True)


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("D", [32, 160, 192, 224])
@pytest.mark.parametrize("n", [1, 20, 150])
def test_head_dims_between(gpu, n, D, kind):
    """Heads whose dims a form fills up with none."""
    attend(gpu, [n, 1], [n + 300, 70], 4, 2, D, 16, HF if n == 20 else BF, kind, layout="hnd")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 6, 40])
def test_parts_of_every_number(gpu, n, D):
    """One unit (n * 3 rows) of 1, 2, .. blocks of keys: as many parts, in sets of any rest."""
    for blocks in list(range(1, 28)) + [33, 41, 64, 65, 66]:
        attend(gpu, [n], [max(n, blocks * (64 if n == 40 else 128) - 5)], 3, 1, D, 64, BF, "mx")


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 32, 64, 512])
def test_attend_page_sizes(gpu, page, layout):
    kind = "mx" if layout == "hnd" else "nv"
    attend(gpu, [1, 3, 2], [150, 3, 600], 4, 2, 128, page, BF, kind, layout=layout)
    attend(gpu, [90, 40], [600, 41], 2, 2, 64, page, HF, kind, layout=layout)


def test_attend_holes(gpu):
    """Pages that are not there, in the middle, at the end and all of a sequence's."""
    holes = [(0, 2, -1), (0, 3, 10 ** 6), (1, 0, -7), (2, 0, -1), (2, 1, -1)]
    for kind in ("mx", "nv"):
        for n in ([1, 1, 1], [20, 5, 9], [150, 5, 20]):
            attend(gpu, n, [200, 5, 30], 4, 2, 64, 16, BF, kind, holes=holes)


def test_attend_table_shorter_than_the_sequence(gpu):
    attend(gpu, [2, 40], [100, 400], 4, 2, 128, 16, BF, "mx", width=3)


@pytest.mark.parametrize("kind,D,dtype", [("mx", 128, BF), ("nv", 128, HF), ("mx", 64, HF), ("nv", 256, BF)])
def test_attend_long(gpu, kind, D, dtype):
    """Many workgroups to a sequence."""
    attend(gpu, [1, 2], [20000, 9000], 8, 2, D, 64, dtype, kind)
    attend(gpu, [70], [20000], 4, 1, D, 64, dtype, kind)


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("amp,q_amp", [(0.0, 1.0), (30.0, 1.0), (1.0, 100.0), (1e-3, 1e-3)])
def test_attend_flat_and_peaked(gpu, amp, q_amp, kind):
    for dtype in (BF, HF):
        attend(gpu, [3, 50], [300, 64], 4, 2, 64, 16, dtype, kind, amp=amp, q_amp=q_amp)


@pytest.mark.parametrize("q_amp", [2.0 ** -120, 2.0 ** 60])
def test_attend_queries_far_from_one(gpu, q_amp):
    """Rows that fp16 has no place for, under e4m3 scales: scores are theirs all the same."""
    attend(gpu, [3, 50], [300, 64], 4, 2, 64, 16, BF, "nv", q_amp=q_amp, scale=min(1.0, 1 / q_amp))


@pytest.mark.parametrize("n", [1, 40, 200])
def test_more_sequences_than_lanes(gpu, n):
    """Units are dealt out 64 sequences at a time; some have none, some many rows."""
    g = gen(n)
    lens = torch.randint(0, 400, (150,), generator=g).tolist()
    new = [min(x, (i * 7) % (n + 1)) for i, x in enumerate(lens)]
    attend(gpu, new, lens, 4, 2, 64, 16, BF, "mx", extra=5)


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("n", [1, 20, 90])
def test_scales_of_any_sign(gpu, n, kind):
    """Negative and zero k_scale: scores change their sign, or are all alike."""
    c = Cache4(5, [n + 100], 16, 3, 128, BF, kind).fill()
    c.k_scale = torch.tensor([-1.0, 0.0, 0.5])
    c.v_scale = torch.tensor([0.5, -2.0, 0.0])
    q = randn(c.g, n, 6, 128, dtype=BF)
    dev = c.to(gpu)
    o, lse = tx.paged_attention(q.to(gpu), cu_q=starts([n]).to(gpu), sm_scale=0.1, return_lse=True, **books(dev))
    ro, rl, bo, bl = attend64(q, c, [n], True, 0, 0.1)
    check(o, ro, small_weights(c, [n], bo), "o")
    check(lse, rl, bl, "lse")


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("which", ["k_block_scale", "v_block_scale"])
@pytest.mark.parametrize("n", [6, 12, 150])
def test_nan_reaches_those_who_attend_to_it(gpu, n, which, kind):
    """One block without numbers: the rows of earlier tokens are as without it, bit by bit, the
    others NaN in every dim."""
    length, at = n + 70, n + 64
    c = Cache4(7, [length, 40], 16, 2, 128, BF, kind).fill()
    q = randn(c.g, n + 1, 4, 128, dtype=BF).to(gpu)
    cu = starts([n, 1]).to(gpu)
    bads = [255, 254] if kind == "mx" else [0x7f, 0xff]
    clean = c.to(gpu)
    o, lse = tx.paged_attention(q, cu_q=cu, sm_scale=0.1, return_lse=True, **books(clean))
    assert bool(torch.isfinite(o).all())
    for bad in bads:
        dev = c.to(gpu)
        page, slot = c.place(0, at)
        raw_scales = dev[which].view(torch.uint8)
        raw_scales[page, slot, 1, -1] = bad
        o2, lse2 = tx.paged_attention(q, cu_q=cu, sm_scale=0.1, return_lse=True, **books(dev))
        hit = torch.zeros(n + 1, 4, dtype=torch.bool)
        hit[at - 70:n, 2:] = True  # tokens from position `at` on, the second kv head's rows
        assert torch.equal(o2[~hit], o[~hit]) and torch.equal(lse2[~hit], lse[~hit])
        assert bool(o2[hit].isnan().all()) and bool(lse2[hit].isnan().all())


def test_attend_offsets_past_32_bits(gpu):
    """Pages and heads further apart than 2^31 bytes, of codes and of scales."""
    for n in ([1, 1], [40, 9]):
        c = Cache4(9, [40, 33], 16, 2, 64, BF, "mx", spare=0).fill()
        dev = c.to(gpu)
        far = dict(dev)
        for name in ("k_cache", "v_cache", "k_block_scale", "v_block_scale"):
            t = dev[name]
            step = 2 ** 30 + 2 ** 29 + 64  # bytes from page to page
            store = torch.zeros(step * (c.P - 1) + 2 ** 16, dtype=torch.uint8, device=gpu)
            wide = store.as_strided(t.shape, (step,) + t.contiguous().stride()[1:])
            wide.copy_(t)
            far[name] = wide
        assert c.P * step > 2 ** 32
        q = randn(c.g, sum(n), 4, 64, dtype=BF).to(gpu)
        cu = starts(n).to(gpu)
        want = tx.paged_attention(q, cu_q=cu, sm_scale=0.1, **books(dev))
        assert torch.equal(tx.paged_attention(q, cu_q=cu, sm_scale=0.1, **books(far)), want)
        k, v = tx.paged_read(cu_q=cu, tokens=sum(n), dtype=BF, **books(far))
        k2, v2 = tx.paged_read(cu_q=cu, tokens=sum(n), dtype=BF, **books(dev))
        assert torch.equal(k, k2) and torch.equal(v, v2)
        x = randn(c.g, sum(n), 2, 64, dtype=BF).to(gpu)
        for d in (dev, far):
            tx.paged_append(x, -x, cu_q=cu, **books(d))
        for name in ("k_cache", "v_cache", "k_block_scale", "v_block_scale"):
            assert torch.equal(dev[name], far[name])


def test_alike_twice_and_on_streams(gpu):
    """The same bits from run to run, also from two streams at once."""
    c, dev, q, o, lse = attend(gpu, [1, 1, 7], [9000, 30, 700], 8, 2, 128, 16, BF, "mx")
    cu, d = starts([1, 1, 7]).to(gpu), q.to(gpu)
    torch.cuda.synchronize()
    for _ in range(3):
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for s in streams:
            with torch.cuda.stream(s):
                outs += [tx.paged_attention(d, cu_q=cu, sm_scale=128 ** -0.5, **books(dev)) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, o) for x in outs)
    named = torch.cuda.Stream()
    got = tx.paged_attention(d, cu_q=cu, sm_scale=128 ** -0.5, stream=named.cuda_stream, **books(dev))
    k, v = tx.paged_read(cu_q=cu, tokens=9, dtype=BF, stream=named.cuda_stream, **books(dev))
    torch.cuda.synchronize()
    assert torch.equal(got, o)
    assert all(torch.equal(a, b) for a, b in zip((k, v), tx.paged_read(cu_q=cu, tokens=9, dtype=BF, **books(dev))))


# ---- together ---------------------------------------------------------------

@pytest.mark.parametrize("kind", ["mx", "nv"])
def test_step_in_a_graph(gpu, kind):
    """Reserve, append, attend and read captured once and replayed as the sequences grow; the same
    step by step without a graph; forks and moves of pages with their scales."""
    S, W, P, page, Hq, Hkv, D = 6, 12, 64, 16, 4, 2, 64
    g = gen(11)
    make = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=torch.uint8, device=gpu).view(dtype)  # noqa: E731
    B = D // BLOCK[kind]

    def new():
        t = E4M3 if kind == "nv" else torch.uint8
        return dict(k_cache=make(P, Hkv, page, D // 2).permute(0, 2, 1, 3),
                    v_cache=make(P, Hkv, page, D // 2).permute(0, 2, 1, 3),
                    k_block_scale=make(P, Hkv, B, page, dtype=t).permute(0, 3, 1, 2),
                    v_block_scale=make(P, Hkv, B, page, dtype=t).permute(0, 3, 1, 2)), dict(
                        table=torch.full((S, W), -1, dtype=torch.int32, device=gpu),
                        length=torch.zeros(S, dtype=torch.int32, device=gpu),
                        refs=torch.zeros(P, dtype=torch.int32, device=gpu))
    inv_freq = tx.rotary_frequencies(D)[0].to(gpu)
    x = torch.zeros(S, Hq + 2 * Hkv, D, dtype=BF, device=gpu)

    def step(cache, b):
        tx.page_reserve(b["table"], b["length"], b["refs"], b["length"] + 1, page,
                        out=(b["table"], b["length"], b["refs"]))
        q = tx.paged_append(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], page_table=b["table"], kv_len=b["length"],
                            q=x[:, :Hq], inv_freq=inv_freq, **cache)
        o = tx.paged_attention(q, page_table=b["table"], kv_len=b["length"], sm_scale=D ** -0.5, **cache)
        k, v = tx.paged_read(page_table=b["table"], kv_len=b["length"], dtype=BF, **cache)
        return o, k, v
    (c1, b1), (c2, b2) = new(), new()
    inputs = [randn(g, S, Hq + 2 * Hkv, D, dtype=BF).to(gpu) for _ in range(40)]
    x.copy_(inputs[0])
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(c1, b1)
    for t in inputs:
        x.copy_(t)
        graph.replay()
        want = step(c2, b2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip((*c1.values(), *b1.values()), (*c2.values(), *b2.values())):
        assert torch.equal(a.view(torch.uint8) if a.dtype == E4M3 else a,
                           b.view(torch.uint8) if b.dtype == E4M3 else b)
    # two rows end and become copies of others; their rows then read what their parents' do
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    drop = torch.tensor([False, False, False, False, True, True], device=gpu)
    t, n, r = tx.page_free(b2["table"], b2["length"], b2["refs"], drop, page)
    t, n, r, missing = tx.page_fork(list(c2.values()), t, n, r, i32([1, 2]), i32([4, 5]))
    assert int(missing) == 0
    t, r, moved = tx.page_compact(list(c2.values()), t, r)
    cu = starts([40] * 6).to(gpu)
    k, v = tx.paged_read(page_table=t, kv_len=n, cu_q=cu, tokens=240, dtype=BF, **c2)
    k, v = k.view(6, 40, Hkv, D), v.view(6, 40, Hkv, D)
    k0, v0 = tx.paged_read(page_table=b1["table"], kv_len=b1["length"], cu_q=cu, tokens=240, dtype=BF, **c1)
    k0, v0 = k0.view(6, 40, Hkv, D), v0.view(6, 40, Hkv, D)
    for i, j in ((0, 0), (1, 1), (2, 2), (3, 3), (4, 1), (5, 2)):
        assert torch.equal(k[i], k0[j]) and torch.equal(v[i], v0[j])
    # and attention over the cache is attention over what is read
    q = randn(g, 6, Hq, D, dtype=BF)
    o = tx.paged_attention(q.to(gpu), page_table=t, kv_len=n, sm_scale=D ** -0.5, **c2)
    kd, vd = k.cpu().double(), v.cpu().double()
    s = torch.einsum("bhgd,blhd->bhgl", q.double().view(6, Hkv, 2, D), kd) * D ** -0.5
    want = torch.einsum("bhgl,blhd->bhgd", s.softmax(-1), vd).reshape(6, Hq, D)
    mag = torch.einsum("bhgl,blhd->bhgd", s.softmax(-1), vd.abs()).reshape(6, Hq, D)
    check(o, want, (2.0 ** -8 + 2.0 ** -12) * mag + 2.0 ** -8 * want.abs(), "o")


@pytest.mark.parametrize("kind", ["mx", "nv"])
def test_generation_example(gpu, kind):
    """The example with a cache in 4 bits: it runs, its beams share pages, and what the cache holds of
    every sequence is the same after pages were freed and moved."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(tx.__file__)), "..", "examples"))
    import paged_generation as ex
    d, fed, got = ex.generate(sequences=3, tokens=6, beams=2, cache_dtype=kind)
    assert int(d.missing) == 0 and d.length.tolist() == [f.shape[0] for f in fed]
    assert all(bool(torch.isfinite(x).all()) for x in got)
    assert int((d.refs > 1).sum()) == sum((int(n) - 6) // d.page for n in d.length[:3].tolist())

    def held(rows):
        n = d.length[rows].tolist()
        return [tx.paged_read(d.k[i], d.v[i], d.table[rows], d.length[rows], starts(n).to(gpu), tokens=sum(n),
                              dtype=BF, k_block_scale=d.ks[i], v_block_scale=d.vs[i]) for i in range(2)]
    d.free(torch.arange(6, device=gpu) % 2 == 1)
    rows = torch.tensor([0, 2, 4], device=gpu)
    before = held(rows)
    d.compact()
    used = int((d.refs > 0).sum())
    assert bool((d.refs[:used] > 0).all()) and not d.refs[used:].any()
    for (k, v), (k0, v0) in zip(held(rows), before):
        assert torch.equal(k, k0) and torch.equal(v, v0)


def test_graph_replayed_after_a_larger_call(gpu):
    """The captured call's workspace is its graph's."""
    c, dev, q, o, _ = attend(gpu, [1], [9000], 4, 1, 128, 16, BF, "mx")
    big = Cache4(13, [3000], 16, 1, 256, BF, "nv").fill()
    bd, bq = big.to(gpu), randn(big.g, 700, 4, 256, dtype=BF).to(gpu)
    d, cu, bcu = q.to(gpu), starts([1]).to(gpu), starts([700]).to(gpu)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = tx.paged_attention(d, cu_q=cu, sm_scale=128 ** -0.5, **books(dev))
    for _ in range(3):
        with torch.cuda.stream(side):
            tx.paged_attention(bq, cu_q=bcu, sm_scale=0.1, **books(bd))
        torch.cuda.synchronize()
        others = [torch.full((m,), 1.0, device=gpu) for m in (1 << 14, 1 << 20, 1 << 22) * 3]
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, o) and all(bool((y == 1.0).all()) for y in others)


def test_nothing_to_do(gpu):
    """No tokens, no sequences, no pages."""
    c = Cache4(15, [0, 0], 16, 2, 64, BF, "mx")
    dev = c.to(gpu)
    q = torch.zeros(0, 4, 64, dtype=BF, device=gpu)
    cu = torch.zeros(3, dtype=torch.int32, device=gpu)
    o, lse = tx.paged_attention(q, cu_q=cu, sm_scale=0.1, return_lse=True, **books(dev))
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    k, v = tx.paged_read(cu_q=cu, tokens=0, dtype=BF, **books(dev))
    assert k.shape == (0, 2, 64)
    assert tx.paged_append(q[:, :2], q[:, :2], cu_q=cu, **books(dev)) is None
    none = {n: dev[n][:0] for n in ("k_cache", "v_cache", "k_block_scale", "v_block_scale")}
    kv = torch.tensor([5, 9], dtype=torch.int32, device=gpu)
    table = torch.zeros(2, 4, dtype=torch.int32, device=gpu)
    q = torch.ones(2, 4, 64, dtype=BF, device=gpu)
    for n in (1, 100):
        x = q.repeat_interleave(n, 0)
        o, lse = tx.paged_attention(x, page_table=table, kv_len=kv, cu_q=starts([n, n]).to(gpu), sm_scale=0.1,
                                    return_lse=True, **none)
        assert not o.any() and bool((lse == -math.inf).all())
    k, v = tx.paged_read(page_table=table, kv_len=kv, dtype=BF, **none)
    assert k.shape == (2, 2, 64) and not k.any() and not v.any()
    got = tx.paged_append(q[:, :2], q[:, :2], page_table=table, kv_len=kv, q=q, **none)
    assert torch.equal(got, q)


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("n,lens,Hq,Hkv,D,rot,page,dtype,layout,interleaved", MANY_THREADS)
def test_append_tokens_of_more_than_a_workgroup(gpu, n, lens, Hq, Hkv, D, rot, page, dtype, layout, interleaved,
                                                kind):
    """Heads that are rotated in a token's last workgroup, of fewer threads than there are pairs."""
    test_append_rotated(gpu, n, lens, Hq, Hkv, D, rot, page, dtype, layout, interleaved, kind)


@pytest.mark.parametrize("kind,dtype", [("mx", BF), ("mx", HF), ("nv", BF), ("nv", HF)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 20, 150])
def test_small_weights_add_up(gpu, n, D, kind, dtype):
    """One key outweighs all the others, and what it holds is 0: the result is what the small weights
    add up to.  In fp16 a weight (2^7 or more at a row's reference) is off by half its least step, 2^-25."""
    L, less = 600, 26.3  # keys, and how far below the one the others are: a factor of 2^less
    c = Cache4(21, [L], 16, 1, D, dtype, kind, "hnd")
    one, two56 = (127, 135) if kind == "mx" else (0x38, 0x78)  # scales of 1 and 256
    blocks = D // BLOCK[kind]
    for j in range(L):
        k = torch.zeros(1, D // 2, dtype=torch.uint8)
        k[0, 0] = 6 if j == 0 else 0  # dim 0: 4 or 0
        c.put("k", 0, j, k, torch.full((1, blocks), one, dtype=torch.uint8))
        v = torch.full((1, D // 2), 0 if j == 0 else 0x66, dtype=torch.uint8)
        c.put("v", 0, j, v, torch.full((1, blocks), two56, dtype=torch.uint8))
    assert torch.equal(c.rows("k", 0)[0][:2, 0, 0], torch.tensor([4.0, 0.0], dtype=torch.float64))
    assert torch.equal(c.rows("v", 0)[0][:2, 0, -1], torch.tensor([0.0, 1024.0], dtype=torch.float64))
    q = torch.zeros(n, 1, D, dtype=dtype)
    q[:, :, 0] = 1.0
    o, lse = tx.paged_attention(q.to(gpu), cu_q=starts([n]).to(gpu), sm_scale=less * math.log(2.0) / 4, causal=False,
                                return_lse=True, **books(c.to(gpu)))
    small = (L - 1) * 2.0 ** -less
    want = torch.full((n, 1, D), small * 1024.0 / (1 + small), dtype=torch.float64)
    # roundings: of a weight (bf16: relative; fp16: absolute, here larger), of the result, and of the
    # score, (D + 2) F and less * 4 F of the exponent's
    bound = (L - 1) * 1024.0 * 2.0 ** -32 if (kind, dtype) != ("mx", BF) else 2.0 ** -8 * want
    bound = bound + torch.finfo(dtype).eps / 2 * want + (D + 2 + 4) * less * F * want
    check(o, want, bound, "o")
    top = torch.full((n, 1), less, dtype=torch.float64)
    check(lse, top + math.log2(1 + small), (D + 10) * F * top, "lse")


@pytest.mark.parametrize("kind", ["mx", "nv"])
@pytest.mark.parametrize("n", [2, 20, 150])
def test_infinite_query(gpu, n, kind):
    """A row of q with an infinity and finite dims past fp16's range: every score is the infinity's, here
    -infinity, so that the row attends to nothing; other rows stay as they are."""
    D = 128
    c = Cache4(23, [200], 16, 1, D, BF, kind, "hnd").fill()
    for j in range(200):  # dims 0 and 1: -1 and 1
        page, slot = c.place(0, j)
        c.k[page, slot, 0, 0] = 0x2a
        c.kb[page, slot, 0, 0] = 127 if kind == "mx" else 0x38
    q = randn(c.g, n, 1, D, dtype=BF)
    dev, cu = c.to(gpu), starts([n]).to(gpu)
    o, lse = tx.paged_attention(q.to(gpu), cu_q=cu, sm_scale=0.1, causal=False, return_lse=True, **books(dev))
    assert bool(torch.isfinite(o).all())
    q[1, 0, 0], q[1, 0, 1] = math.inf, 1e30
    o2, lse2 = tx.paged_attention(q.to(gpu), cu_q=cu, sm_scale=0.1, causal=False, return_lse=True, **books(dev))
    rest = torch.arange(n) != 1
    assert torch.equal(o2[rest], o[rest]) and torch.equal(lse2[rest], lse[rest])
    assert not o2[1].any() and bool((lse2[1] == -math.inf).all())
    q[1, 0, 0] = -math.inf  # every score is infinity: no numbers
    o2, lse2 = tx.paged_attention(q.to(gpu), cu_q=cu, sm_scale=0.1, causal=False, return_lse=True, **books(dev))
    assert torch.equal(o2[rest], o[rest]) and bool(o2[1].isnan().all())
