"""The paged attention's forms at the sizes where one takes over from another, its scales and
non-finite values, calls of one form after another, and large books of pages."""
import math
import os
import sys

import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd as tx  # noqa: E402
from cachecase import E4M3, Cache, attend64, check, gen, randn, rotate64, rotate_bound, starts  # noqa: E402
from dotcase import say  # noqa: E402
from test_cache_gpu import Books, attend, same  # noqa: E402

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("cache", [BF, E4M3])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("rows", [15, 16, 17, 32, 33, 128, 129, 300])
def test_rows_of_a_sequence(gpu, rows, D, cache):
    """New tokens times heads of a kv head: at and past the rows of a unit in each form."""
    G = 1 if rows % 3 else 3
    n = rows // G
    attend(gpu, [n, 1, n], [n + 75, 1, 700], 2 * G, 2, D, 16, BF, cache)
    attend(gpu, [n], [n + 40], 2 * G, 2, D, 16, BF, cache, window=33)


@pytest.mark.parametrize("page", [1, 2, 8, 16])
@pytest.mark.parametrize("D,cache", [(64, E4M3), (128, E4M3), (256, HF), (64, HF)])
def test_many_heads_of_small_pages(gpu, page, D, cache):
    """One token of 16 heads a kv head, pages of fewer rows than a load takes."""
    attend(gpu, [1, 1, 1], [301, 31, 64], 16, 1, D, page, HF, cache, decode=True, layout="hnd")
    attend(gpu, [150], [301], 2, 2, D, page, HF, cache)


@pytest.mark.parametrize("n", [1, 40, 200])
def test_more_sequences_than_lanes(gpu, n):
    """Units are dealt out 64 sequences at a time; some have none, some many rows."""
    g = gen(n)
    lens = torch.randint(0, 400, (150,), generator=g).tolist()
    new = [min(x, (i * 7) % (n + 1)) for i, x in enumerate(lens)]
    attend(gpu, new, lens, 4, 2, 64, 16, BF, BF, extra=5)


def test_uneven_parts_of_one_batch(gpu):
    """One sequence with most of the keys, next to empty and short ones, in every form."""
    for n in (1, 6, 50):
        attend(gpu, [n, 0, 1, n, 1], [30000, 0, 1, n, 200], 8, 2, 128, 64, BF, BF)


@pytest.mark.parametrize("n", [1, 20, 90])
def test_scales_of_any_sign(gpu, n):
    """Negative and zero k_scale: scores change their sign, or are all alike."""
    c = Cache(5, [n + 100], 16, 3, 128, HF, E4M3).fill()
    c.k_scale = torch.tensor([-1 / 64, 0.0, 1 / 64])
    c.v_scale = torch.tensor([1 / 64, -1 / 64, 0.0])
    q = randn(c.g, n, 6, 128, dtype=HF)
    o, lse = tx.paged_attention(q.to(gpu), cu_q=starts([n]).to(gpu), sm_scale=0.1,
                                return_lse=True, **c.to(gpu))
    ro, rl, bo, bl = attend64(q, c, [n], True, 0, 0.1)
    check(o, ro, bo, "o")
    check(lse, rl, bl, "lse")
    assert not o[:, 4:].any()


@pytest.mark.parametrize("n", [1, 20, 90])
def test_scale_zero_takes_the_mean(gpu, n):
    c = Cache(6, [n + 50], 16, 1, 64, BF, BF).fill()
    q = randn(c.g, n, 2, 64, dtype=BF)
    o, lse = tx.paged_attention(q.to(gpu), cu_q=starts([n]).to(gpu), sm_scale=0.0,
                                return_lse=True, **c.to(gpu))
    ro, rl, bo, bl = attend64(q, c, [n], True, 0, 0.0)
    check(o, ro, bo, "o")
    check(lse, rl, bl, "lse")


@pytest.mark.parametrize("n", [1, 20, 90])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_nonfinite_values(gpu, n, value):
    """A NaN among the keys that are attended to comes out as NaN, in its kv head only; one where
    nothing is attended to (past the sequence, in a page the table does not name) stays there."""
    c = Cache(7, [n + 70], 16, 2, 128, BF, BF).fill()  # (poisoned with NaN past the sequence)
    at = c.place(0, 11)
    c.k[at][0, 3] = value
    q = randn(c.g, n, 4, 128, dtype=BF).abs() + 0.5
    o, lse = tx.paged_attention(q.to(gpu), cu_q=starts([n]).to(gpu), sm_scale=0.1,
                                return_lse=True, **c.to(gpu))
    assert bool(torch.isnan(o[:, :2]).all())
    assert bool(torch.isfinite(o[:, 2:]).all()) and bool(torch.isfinite(lse[:, 2:]).all())
    c.k[at][0, 3] = 0.0  # and of q: all scores of a row are NaN
    q[-1, 1, 5] = math.nan
    o = tx.paged_attention(q.to(gpu), cu_q=starts([n]).to(gpu), sm_scale=0.1, **c.to(gpu)).cpu()
    bad = torch.zeros(n, 4, dtype=torch.bool)
    bad[-1, 1] = True
    assert bool(torch.isnan(o[bad]).all()) and bool(torch.isfinite(o[~bad]).all())


@pytest.mark.parametrize("sm_scale", [1.0, 0.4])
def test_growing_maximum(gpu, sm_scale):
    """Scores that rise by more and by less than the step at which sums are rescaled, block after
    block, past what fp16 could hold without it."""
    for n, G in ((1, 2), (40, 2), (150, 1)):
        c = Cache(8, [600], 16, 1, 64, HF, HF).fill()
        steps = torch.arange(600, dtype=torch.float64) // 32 * 3.0
        for j in range(600):
            c.k[c.place(0, j)][0] = 0.0
            c.k[c.place(0, j)][0, 0] = float(steps[j])
        q = torch.zeros(n, G, 64, dtype=HF)
        q[:, :, 0] = 3.0
        o, lse = tx.paged_attention(q.to(gpu), cu_q=starts([n]).to(gpu),
                                    sm_scale=sm_scale, return_lse=True, **c.to(gpu))
        ro, rl, bo, bl = attend64(q, c, [n], True, 0, sm_scale)
        check(o, ro, bo, "o")
        check(lse, rl, bl, "lse")


def test_calls_of_one_form(gpu):
    """What a call has found for a form holds for the next of that form, not for others: other
    addresses, alignment and layouts between them."""
    inv_freq = tx.rotary_frequencies(64)[0].to(gpu)
    pos = torch.arange(9)
    for i in range(3):
        g = gen(i)
        store = randn(g, 9 * 4 * 64 + 8, dtype=BF).to(gpu)
        for x in (store[:-8].view(9, 4, 64), store[1:-7].view(9, 4, 64),  # odd base
                  store[:-8].view(4, 9, 64).transpose(0, 1), store[:-8].view(9, 64, 4).transpose(1, 2)):
            got = tx.rotary(x, pos.to(gpu), inv_freq)
            ref, mag = rotate64(x.cpu(), pos, inv_freq.cpu(), False, 1.0)
            check(got, ref, rotate_bound(ref, mag, BF), "rotary")
    c = Cache(9, [50, 70], 16, 2, 64, BF, BF).fill()
    dev = c.to(gpu)
    for i in range(3):
        store = randn(c.g, 2 * 4 * 64 + 8, dtype=BF).to(gpu)
        for q in (store[:-8].view(2, 4, 64), store[1:-7].view(2, 4, 64),
                  store[:-8].view(4, 2, 64).transpose(0, 1), store[:-8].view(2, 64, 4).transpose(1, 2)):
            o = tx.paged_attention(q, sm_scale=0.125, **dev)
            ro, _, bo, _ = attend64(q.cpu().contiguous(), c, [1, 1], True, 0, 0.125)
            check(o, ro, bo, "o")
    wide = torch.zeros(2, 2, dtype=torch.int32, device=gpu)  # lengths that lie apart
    wide[:, 0] = dev["kv_len"]
    apart = dict(dev, kv_len=wide[:, 0])
    assert torch.equal(tx.paged_attention(q, sm_scale=0.125, **apart), o)
    with pytest.raises(ValueError):  # the same shapes on another device
        tx.paged_attention(q, sm_scale=0.125, **dict(dev, kv_len=c.kv_len))


# ---- pages ------------------------------------------------------------------

@pytest.mark.parametrize("in_place", [False, True])
def test_free_pages_far_apart(gpu, in_place):
    """The pages that are wanted lie thousands apart, in a pool that is nearly full."""
    b = Books(0, 40, 30, 20000, 4, fill=0.0)
    held = set(range(0, 20000, 1500))
    b.table = [[-1] * 30 for _ in range(40)]
    b.len = [0] * 40
    b.refs = [0 if p in held else 1 for p in range(20000)]
    t, n, r = b.to(gpu)
    new = [5 if s % 4 == 0 else 0 for s in range(40)]  # 2 pages for every fourth: more than there are
    got = tx.page_reserve(t, n, r, torch.tensor(new, dtype=torch.int32, device=gpu), 4,
                          out=(t, n, r) if in_place else None)
    missing = b.reserve(new)
    same(b, *got[:3])
    assert int(got[3]) == missing > 0


@pytest.mark.parametrize("in_place", [False, True])
def test_fork_into_many(gpu, in_place):
    """More children than a workgroup has threads."""
    S, W, P = 1300, 3, 4000
    b = Books(3, S, W, P, 4, fill=0.9)
    b.free([s >= 100 for s in range(S)])
    g = gen(4)
    pairs = [(int(torch.randint(0, 100, (1,), generator=g)), s) for s in range(100, S)]
    data = randn(g, P, 4, 1, 8, dtype=BF)
    dev = data.to(gpu)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    t, n, r = b.to(gpu)
    got = tx.page_fork([dev], t, n, r, i32([a for a, _ in pairs]), i32([c for _, c in pairs]),
                       out=(t, n, r) if in_place else None)
    copies, missing = b.fork(pairs)
    same(b, *got[:3])
    assert int(got[3]) == missing
    for a, c in copies:
        data[c] = data[a]
    assert torch.equal(data, dev.cpu())


@pytest.mark.parametrize("P", [100, 262144, 262145, 300001])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact_pools_of_any_size(gpu, P, in_place):
    say("compact", P, in_place)
    g = gen(P)
    refs = (torch.rand(P, generator=g) < 0.3).to(torch.int32)
    used = int(refs.sum())
    pages = refs.nonzero()[:, 0]
    table = torch.full((7, 50), -1, dtype=torch.int32)
    pick = pages[torch.randperm(used, generator=g)[:min(used, 300)]]
    table.view(-1)[:pick.numel()] = pick.to(torch.int32)
    data = torch.arange(P, dtype=torch.int32)[:, None].repeat(1, 4)
    dev, t, r = data.to(gpu), table.to(gpu), refs.to(gpu)
    t2, r2, moved = tx.page_compact([dev], t, r, out=(t, r) if in_place else None)
    holes = (refs[:used] == 0).nonzero()[:, 0]
    movers = (refs[used:] > 0).nonzero()[:, 0] + used
    assert int(moved) == movers.numel() == holes.numel()
    to = torch.arange(P)
    to[movers] = holes
    want = torch.where(table >= 0, to[table.clamp_min(0).long()].to(torch.int32), table)
    assert torch.equal(t2.cpu(), want)
    assert torch.equal(r2.cpu(), (torch.arange(P) < used).to(torch.int32))
    data[holes] = data[movers]
    assert torch.equal(dev.cpu(), data)


@pytest.mark.parametrize("S,W,P", [(1, 1, 1), (3, 100, 513), (4096, 1, 700), (4097, 1, 700),
                                   (64, 64, 5000), (17, 241, 5000), (7, 40, 131072), (7, 40, 131073)])
def test_forms_of_free(gpu, S, W, P):
    """Entries and pages at and past where every workgroup goes through the table; pages that
    several rows hold, holes, lengths past the table and below nothing."""
    say("free", S, W, P)
    g = gen(S + W)
    page = 4
    table = torch.randint(-1, min(P + 2, 200000), (S, W), generator=g).to(torch.int32)
    table[:, : W // 3] = table[0, : W // 3]
    table[0, 0] = P - 1
    length = torch.randint(-3, W * page + 9, (S,), generator=g).to(torch.int32)
    length[0] = W * page
    refs = torch.randint(0, 1 << 20, (P,), generator=g).to(torch.int32)
    drop = torch.rand(S, generator=g) < 0.5
    drop[0] = True
    held = (torch.arange(W)[None] < ((length + page - 1) // page)[:, None]) & drop[:, None]
    given = table[held & (table >= 0) & (table < P)].long()
    want = (torch.where(drop[:, None], -1, table), torch.where(drop, 0, length),
            refs - torch.bincount(given, minlength=P).to(torch.int32))
    for kind in (False, True):
        t, n, r, d = (x.to(gpu) for x in (table, length, refs, drop))
        got = tx.page_free(t, n, r, d, page, out=(t, n, r) if kind else None)
        for x, y in zip(got, want):
            assert torch.equal(x.cpu(), y)
    assert int(given.numel()) > 0


@pytest.mark.parametrize("S", [1, 5000])
def test_free_of_rows_without_entries(gpu, S):
    table = torch.empty((S, 0), dtype=torch.int32, device=gpu)
    length = torch.full((S,), 3, dtype=torch.int32, device=gpu)
    refs = torch.arange(9, dtype=torch.int32, device=gpu)
    drop = torch.arange(S, device=gpu) % 2 == 0
    t, n, r = tx.page_free(table, length, refs, drop, 4)
    assert t.shape == (S, 0) and torch.equal(r, refs)
    assert torch.equal(n, torch.where(drop, 0, length))


# ---- together -----------------------------------------------------------------

@pytest.mark.parametrize("kind", [BF, E4M3])
def test_generation_example(gpu, kind):
    """The example's outputs against the same layers over whole sequences at once: chunks, beams
    and replayed steps change the order of sums only, so two runs' roundings stay within what the
    layers make of them."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(tx.__file__)), "..", "examples"))
    import paged_generation as ex
    d, fed, got = ex.generate(sequences=3, tokens=6, beams=2, cache_dtype=None if kind == BF else kind)
    assert int(d.missing) == 0
    assert d.length.tolist() == [f.shape[0] for f in fed]
    # each row alone, in one chunk
    for row in range(len(fed)):
        one = ex.Decoder(rows=1, cache_dtype=None if kind == BF else kind)
        n = torch.tensor([fed[row].shape[0]], dtype=torch.int32, device=gpu)
        one.reserve(n)
        want = one.forward(fed[row], slice(0, 1), starts([fed[row].shape[0]]).to(gpu)).double()
        # where the order of sums tips a rounding to bf16, that value is off by 2^-7: in norm, over a
        # layer's six roundings and two layers, less than sqrt(12) 2^-8.  A cached e4m3 value that is
        # tipped (one in 16 at most: the ratio of the types' steps) is off by 2^-3: 2^-5 in norm
        off = (got[row].double() - want).norm() / want.norm()
        assert float(off) < 4 * 2.0 ** -8 + (2.0 ** -5 if kind == E4M3 else 0.0), (row, float(off))
    shared = int((d.refs > 1).sum())
    assert shared == sum((int(n) - 6) // d.page for n in d.length[:3].tolist())
    d.free(torch.arange(6, device=gpu) % 2 == 1)
    before = [x.clone() for x in (d.k[0][d.table[0, 0]], d.v[1][d.table[0, 0]])]
    d.compact()
    assert torch.equal(d.k[0][d.table[0, 0]], before[0]) and torch.equal(d.v[1][d.table[0, 0]], before[1])
    used = int((d.refs > 0).sum())
    assert bool((d.refs[:used] > 0).all()) and not d.refs[used:].any()
