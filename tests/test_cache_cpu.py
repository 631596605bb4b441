"""The paged cache's entry points without a GPU: what they refuse, and their plans."""
import ctypes
import math

import pytest

import triton_ext_amd as tx
from triton_ext_amd import capi

torch = pytest.importorskip("torch")
BF = torch.bfloat16


def books(S=2, W=4, P=8):
    return (torch.full((S, W), -1, dtype=torch.int32), torch.zeros(S, dtype=torch.int32),
            torch.zeros(P, dtype=torch.int32))


def caches(P=8, page=16, Hkv=2, D=64, dtype=BF):
    return torch.zeros(P, page, Hkv, D, dtype=dtype), torch.zeros(P, page, Hkv, D, dtype=dtype)


def test_rotary_refusals():
    x, pos, f = torch.zeros(5, 2, 64), torch.arange(5), torch.zeros(32)
    bad = [((x[0], pos, f), {}), ((x, pos[:4], f), {}), ((x, pos.float(), f), {}),
           ((x, pos, f.double()), {}), ((x, pos, f[None]), {}),
           ((x.view(1, 2, 5, 64), torch.arange(4), f), {}), ((x, pos, f), {"out": x[:, :1]}),
           ((x, pos, f), {"out": x.half()})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            tx.rotary(*args, **kw)
    with pytest.raises(NotImplementedError):
        tx.rotary(x.double(), pos, f)
    for f in (torch.zeros(33), torch.zeros(0)):  # more dims than there are, and none
        with pytest.raises(tx.TxError) as e:
            tx.rotary(x, pos, f)
        assert e.value.code == tx.ERR_INVALID
    with pytest.raises(tx.TxError) as e:
        tx.rotary(x, pos, torch.zeros(32), scale=math.inf)
    assert e.value.code == tx.ERR_INVALID
    with pytest.raises(tx.TxError) as e:  # a view whose rows overlap is not written to
        tx.rotary(x, pos, torch.zeros(32), out=torch.zeros(5, 1, 64).expand(5, 2, 64))
    assert e.value.code == tx.ERR_INVALID


def test_rotary_frequencies():
    f, s = tx.rotary_frequencies(64)
    assert f.dtype == torch.float32 and f.shape == (32,) and s == 1.0
    want = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    assert torch.equal(f, want.float())
    lin, _ = tx.rotary_frequencies(64, scaling="linear", factor=8.0)
    assert torch.equal(lin, (want / 8).float())
    ntk, _ = tx.rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert float(ntk[0]) == 1.0  # the fastest stays, the slowest goes factor times slower
    assert abs(float(ntk[-1]) * 8 / float(want[-1]) - 1) < 1e-6
    y, s = tx.rotary_frequencies(64, scaling="yarn", factor=8.0, context=4096)
    assert abs(s - (0.1 * math.log(8.0) + 1)) < 1e-12
    assert float(y[0]) == 1.0 and abs(float(y[-1]) * 8 / float(want[-1]) - 1) < 1e-6
    assert bool((y <= f).all()) and bool((y >= lin).all())
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=64, scaling="other"),
                dict(rot_dim=64, scaling="linear", factor=0.5), dict(rot_dim=2, scaling="ntk")):
        with pytest.raises(ValueError):
            tx.rotary_frequencies(**bad)


def append(**kw):
    kc, vc = caches()
    t, n, _ = books()
    a = dict(k=torch.zeros(2, 2, 64, dtype=BF), v=torch.zeros(2, 2, 64, dtype=BF), k_cache=kc,
             v_cache=vc, page_table=t, kv_len=n)
    a.update(kw)
    return tx.paged_append(**a)


def attend(**kw):
    kc, vc = caches()
    t, n, _ = books()
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF), k_cache=kc, v_cache=vc, page_table=t, kv_len=n,
             sm_scale=0.125)
    a.update(kw)
    return tx.paged_attention(**a)


@pytest.mark.parametrize("call", [append, attend])
def test_paged_refusals(call):
    kc, vc = caches()
    t, n, _ = books()
    f8 = [x.to(torch.float8_e4m3fn) for x in (kc, vc)]
    for kw in (dict(k_cache=kc[0]), dict(v_cache=vc[:7]), dict(k_cache=kc[..., :32]),
               dict(page_table=t.long()), dict(page_table=t[0]), dict(page_table=t[:1]),
               dict(page_table=t.t().contiguous().t()), dict(kv_len=n.long()), dict(kv_len=n[:1]),
               dict(cu_q=torch.zeros(2, dtype=torch.int32)),
               dict(cu_q=torch.zeros(3, dtype=torch.int64)),
               dict(k_scale=torch.ones(2)),
               dict(k_cache=f8[0], v_cache=f8[1], k_scale=torch.ones(3)),
               dict(k_cache=f8[0], v_cache=f8[1], v_scale=torch.ones(2).double()),
               dict(k_cache=kc.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(NotImplementedError):
        call(k_cache=kc.half(), v_cache=vc.half())
    kc, vc = caches(page=12)
    with pytest.raises(tx.TxError) as e:
        call(k_cache=kc, v_cache=vc)
    assert e.value.code == tx.ERR_UNSUPPORTED and "power of two" in str(e.value)


def test_append_refusals():
    k = torch.zeros(2, 2, 64, dtype=BF)
    for kw in (dict(k=k[0]), dict(v=k[:1]), dict(v=k.half()), dict(k=torch.cat((k, k))),
               dict(q=torch.zeros(2, 4, 32, dtype=BF)), dict(q=torch.zeros(3, 4, 64, dtype=BF)),
               dict(q=k, q_out=k[:, :1]), dict(q_out=k), dict(inv_freq=torch.zeros(4).double())):
        with pytest.raises(ValueError):
            append(**kw)
    with pytest.raises(NotImplementedError):
        append(k=k.float())
    with pytest.raises(tx.TxError):
        append(inv_freq=torch.zeros(33))


def test_attend_refusals():
    q = torch.zeros(2, 4, 64, dtype=BF)
    for kw in (dict(q=q[0]), dict(q=torch.cat((q, q))), dict(out=q.half()), dict(out=q[:, :2])):
        with pytest.raises(ValueError):
            attend(**kw)
    with pytest.raises(NotImplementedError):
        attend(q=q.float())
    for kw in (dict(q=q[:, :3]), dict(sm_scale=-1.0), dict(sm_scale=math.nan), dict(window=-1),
               dict(out=torch.zeros(2, 1, 64, dtype=BF).expand(2, 4, 64))):
        with pytest.raises(tx.TxError) as e:
            attend(**kw)
        assert e.value.code == tx.ERR_INVALID
    for D in (264, 20):
        kc, vc = caches(D=D)
        with pytest.raises(tx.TxError) as e:
            attend(q=torch.zeros(2, 4, D, dtype=BF), k_cache=kc, v_cache=vc)
        assert e.value.code == tx.ERR_UNSUPPORTED


def _attn_plan(**kw):
    f = dict(T=4, B=4, pages=64, table_width=8, Hq=8, Hkv=2, head_dim=128, page_size=16,
             dtype=tx.BF16, cache_type=tx.BF16, causal=1, window=0, ragged=0, sm_scale=0.1,
             q_st=1024, q_sh=128, o_st=1024, o_sh=128, k_sp=4096, k_st=256, k_sh=128, v_sp=4096,
             v_st=256, v_sh=128, table_s=8)
    f.update(kw)
    d = capi.PagedAttnDesc()
    for k, v in f.items():
        setattr(d, k, v)
    p = capi.PagedAttnPlan()
    return tx.load().tx_paged_attn_plan_create(ctypes.byref(d), ctypes.byref(p)), p


def test_attend_plans():
    L = tx.load()
    assert L.tx_paged_attn_plan_create(None, None) == tx.ERR_INVALID
    rc, p = _attn_plan()
    assert rc == tx.OK and p.grid_x > 0
    for bad in (dict(T=-1), dict(T=5), dict(B=0), dict(Hq=7), dict(Hkv=0), dict(page_size=0),
                dict(page_size=24), dict(head_dim=0), dict(head_dim=4), dict(head_dim=512),
                dict(dtype=tx.F32), dict(cache_type=tx.F16), dict(causal=2), dict(ragged=7),
                dict(window=-2), dict(sm_scale=math.inf), dict(q_st=1025), dict(o_sh=4),
                dict(k_sp=-8), dict(k_st=64), dict(v_sh=4), dict(table_s=3),
                dict(cache_type=tx.F8E4M3, k_st=264, head_dim=128), dict(T=2 ** 32, B=2 ** 32)):
        rc, _ = _attn_plan(**bad)
        assert rc in (tx.ERR_INVALID, tx.ERR_UNSUPPORTED), bad
        assert L.tx_get_last_error()
    # a plan that was edited is not launched
    a = ctypes.c_void_p(4096)
    for field in ("variant", "rows", "slots", "units", "grid_x", "block_threads",
                  "workspace_bytes"):
        rc, p = _attn_plan()
        setattr(p, field, getattr(p, field) + 1)
        assert L.tx_paged_attn_launch(ctypes.byref(p), a, a, a, a, a, None, None, None, a, None,
                                      a, 1 << 40, None) == tx.ERR_INVALID
    rc, p = _attn_plan()
    args = [a, a, a, a, a, None, None, None, a, None]
    for i in (0, 1, 2, 3, 4, 8):  # NULL where an array is needed
        bad = list(args)
        bad[i] = None
        assert L.tx_paged_attn_launch(ctypes.byref(p), *bad, a, 1 << 40, None) == tx.ERR_INVALID
    for i in (0, 1, 2, 8):  # less than 16-byte aligned
        bad = list(args)
        bad[i] = ctypes.c_void_p(4104)
        assert L.tx_paged_attn_launch(ctypes.byref(p), *bad, a, 1 << 40, None) == tx.ERR_INVALID
    bad = list(args)
    bad[5] = a  # cu_q for a plan without
    assert L.tx_paged_attn_launch(ctypes.byref(p), *bad, a, 1 << 40, None) == tx.ERR_INVALID
    if p.workspace_bytes:
        assert L.tx_paged_attn_launch(ctypes.byref(p), *args, None, 0, None) == tx.ERR_WORKSPACE
    if not torch.cuda.is_available():
        assert L.tx_paged_attn_launch(ctypes.byref(p), *args, a, 1 << 40, None) == tx.ERR_NO_DEVICE
    # no tokens: nothing to do, and nothing to give
    rc, p = _attn_plan(T=0, B=0)
    assert rc == tx.OK
    assert L.tx_paged_attn_launch(ctypes.byref(p), *[None] * 11, 0, None) == tx.OK


def test_page_refusals():
    t, n, r = books()
    kc, vc = caches()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        tx.page_reserve(t, n[:1], r, n, 16)
    with pytest.raises(ValueError):
        tx.page_reserve(t, n, r, n[:1], 16)
    with pytest.raises(ValueError):
        tx.page_reserve(t.long(), n, r, n, 16)
    with pytest.raises(ValueError):
        tx.page_reserve(t, n, r, n, 16, out=(t, n))
    with pytest.raises(ValueError):
        tx.page_reserve(t, n, r, n, 16, out=(t, n, r[:3]))
    with pytest.raises(ValueError):
        tx.page_free(t, n, r, n, 16)
    with pytest.raises(tx.TxError) as e:
        tx.page_free(t, n, r, n.bool(), 12)
    assert e.value.code == tx.ERR_UNSUPPORTED
    with pytest.raises(ValueError):
        tx.page_fork([], t, n, r, i32(0), i32(1))
    with pytest.raises(ValueError):
        tx.page_fork([kc], t, n, r, i32(0, 1), i32(1))
    with pytest.raises(ValueError):  # a pool of other pages
        tx.page_fork([kc[:5]], t, n, r, i32(0), i32(1))
    with pytest.raises(ValueError):
        tx.page_copy([kc, vc], i32(0), i32(1, 2))
    with pytest.raises(ValueError):  # a page is not one block of memory
        tx.page_copy([kc[:, :, :1]], i32(0), i32(1))
    with pytest.raises(ValueError):
        tx.page_copy([kc] * 129, i32(0), i32(1))
    with pytest.raises(tx.TxError) as e:  # pages of 24 bytes
        tx.page_copy([torch.zeros(4, 3, 4, dtype=BF)], i32(0), i32(1))
    assert e.value.code == tx.ERR_INVALID


def test_pages_in_any_order_in_memory_are_one_block():
    from triton_ext_amd.cache import _page_bytes
    k = torch.zeros(8, 2, 16, 64, dtype=BF)
    assert _page_bytes(k, "k", 8) == (4096, 4096)
    assert _page_bytes(k.permute(0, 2, 1, 3), "k", 8) == (4096, 4096)
    kv = torch.zeros(8, 2, 16, 2, 64, dtype=BF)  # k and v of a page together
    assert _page_bytes(kv[:, 0], "k", 8) == (8192, 4096)
