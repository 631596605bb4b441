"""The 4-bit paged cache's entry points without a GPU: what they refuse, their plans, and the oracle
that the GPU tests compare with."""
import ctypes
import math

import pytest

import triton_ext_amd as tx
from cache4case import BLOCK, LEVELS, quantise, scale_values, values
from triton_ext_amd import cache4 as cache4_module, capi

torch = pytest.importorskip("torch")
BF, HF, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def cache4(P=8, page=16, Hkv=2, D=64, kind="mx"):
    s = (P, page, Hkv, D // BLOCK[kind])
    scales = [torch.zeros(s, dtype=torch.uint8).view(torch.uint8 if kind == "mx" else E4M3) for _ in range(2)]
    return dict(k_cache=torch.zeros(P, page, Hkv, D // 2, dtype=torch.uint8),
                v_cache=torch.zeros(P, page, Hkv, D // 2, dtype=torch.uint8), k_block_scale=scales[0],
                v_block_scale=scales[1], page_table=torch.zeros(2, 4, dtype=torch.int32),
                kv_len=torch.zeros(2, dtype=torch.int32))


def append(**kw):
    a = dict(k=torch.zeros(2, 2, 64, dtype=BF), v=torch.zeros(2, 2, 64, dtype=BF), **cache4())
    a.update(kw)
    return tx.paged_append(**a)


def attend(**kw):
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF), sm_scale=0.125, **cache4())
    a.update(kw)
    return tx.paged_attention(**a)


def read(**kw):
    a = dict(dtype=BF, **cache4())
    a.update(kw)
    return tx.paged_read(**a)


@pytest.mark.parametrize("call", [append, attend, read])
def test_refusals(call):
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    bad = [dict(k_block_scale=None), dict(v_block_scale=None), dict(k_cache=u8(8, 16, 2, 31)),
           dict(v_cache=u8(9, 16, 2, 32)), dict(k_cache=torch.zeros(8, 16, 2, 32), v_cache=torch.zeros(8, 16, 2, 32)),
           dict(k_cache=u8(8, 16, 64), v_cache=u8(8, 16, 64)), dict(k_block_scale=u8(8, 16, 2, 4)),
           dict(v_block_scale=u8(8, 16, 3, 2)), dict(v_block_scale=u8(8, 16, 2, 4).view(E4M3)),
           dict(k_cache=u8(8, 16, 2, 64)[..., ::2]), dict(page_table=torch.zeros(2, 4)),
           dict(page_table=torch.zeros(3, 4, dtype=torch.int32)), dict(kv_len=torch.zeros(2)),
           dict(cu_q=torch.zeros(2, dtype=torch.int32)), dict(k_scale=torch.zeros(3)),
           dict(v_scale=torch.zeros(2, dtype=HF))]
    for kw in bad:
        if call is read and "cu_q" in kw:
            kw = dict(kw, tokens=2)
        with pytest.raises(ValueError):
            call(**kw)
    for kind in (torch.float32, torch.float8_e5m2, BF):
        s = torch.zeros(8, 16, 2, 2).to(kind)
        with pytest.raises(NotImplementedError):
            call(k_block_scale=s, v_block_scale=s)
    odd = [dict(page_size=12)]  # (sizes of pages are powers of two)
    for kw in odd:
        with pytest.raises(tx.TxError) as e:
            call(**cache4(page=kw["page_size"]))
        assert e.value.code == tx.ERR_UNSUPPORTED
    # rows that are not whole 16 bytes apart
    c = u8(8, 16, 2, 40)[..., :32]
    with pytest.raises(tx.TxError) as e:
        call(k_cache=c, v_cache=c)
    assert e.value.code == tx.ERR_INVALID


def test_append_refusals():
    x = torch.zeros(2, 2, 64, dtype=BF)
    for kw in (dict(k=x[0]), dict(v=x[:1]), dict(v=x.half()), dict(k=x[:, :1], v=x[:, :1]), dict(q=x[0]),
               dict(q=x.half()), dict(q_out=x), dict(q=x, q_out=x[:1]), dict(inv_freq=torch.zeros(4, 4)),
               dict(k=x[..., :32], v=x[..., :32])):
        with pytest.raises(ValueError):
            append(**kw)
    with pytest.raises(NotImplementedError):
        append(k=x.float(), v=x.float())
    for kw in (dict(inv_freq=torch.zeros(33)), dict(scale=math.inf),
               dict(k_block_scale=torch.zeros(8, 16, 2, 1, dtype=torch.uint8).expand(8, 16, 2, 2)),
               dict(v_block_scale=torch.zeros(8, 1, 2, 2, dtype=torch.uint8).expand(8, 16, 2, 2))):
        with pytest.raises(tx.TxError) as e:
            append(**kw)
        assert e.value.code == tx.ERR_INVALID


def test_attend_refusals():
    q = torch.zeros(2, 4, 64, dtype=BF)
    for kw in (dict(q=q[0]), dict(q=q[..., :32]), dict(out=q[:1]), dict(out=q.half())):
        with pytest.raises(ValueError):
            attend(**kw)
    with pytest.raises(NotImplementedError):
        attend(q=q.float())
    for kw in (dict(sm_scale=-1.0), dict(window=-1), dict(q=torch.zeros(2, 3, 64, dtype=BF))):
        with pytest.raises(tx.TxError) as e:
            attend(**kw)
        assert e.value.code == tx.ERR_INVALID
    wide = cache4(D=288)
    with pytest.raises(tx.TxError) as e:
        attend(q=torch.zeros(2, 4, 288, dtype=BF), **wide)
    assert e.value.code == tx.ERR_UNSUPPORTED


def test_read_refusals():
    plain = dict(k_cache=torch.zeros(8, 16, 2, 64, dtype=BF), v_cache=torch.zeros(8, 16, 2, 64, dtype=BF),
                 k_block_scale=None, v_block_scale=None)
    cu = torch.zeros(3, dtype=torch.int32)
    rows = torch.zeros(2, 2, 64, dtype=BF)
    for kw in (dict(dtype=None), dict(cu_q=cu), dict(tokens=3), dict(cu_q=cu, tokens=-1),
               dict(k_out=rows[:1]), dict(k_out=rows.half()), dict(v_out=rows.expand(2, 2, 2, 64)),
               dict(k_out=torch.zeros(2, 2, 128, dtype=BF)[..., ::2]), dict(plain, k_scale=torch.zeros(2)),
               dict(plain, v_cache=torch.zeros(8, 16, 2, 64, dtype=HF))):
        with pytest.raises(ValueError):
            read(**kw)
    for kw in (dict(dtype=torch.int32), dict(plain, k_cache=torch.zeros(8, 16, 2, 64),
                                             v_cache=torch.zeros(8, 16, 2, 64))):
        with pytest.raises(NotImplementedError):
            read(**kw)
    with pytest.raises(tx.TxError) as e:  # rows that overlap are not written
        read(k_out=rows[:1].expand(2, 2, 64))
    assert e.value.code == tx.ERR_INVALID


def test_no_number_of_rows_stands_for_none(monkeypatch):
    """A negative `tokens` is refused also after a call that gives none (whose form is known then)."""
    if tx.load().tx_device_available():
        pytest.skip("there is a GPU")
    monkeypatch.setattr(cache4_module, "_current_stream", lambda device: 0)
    with pytest.raises(tx.TxError) as e:
        read(stream=0)
    assert e.value.code == tx.ERR_NO_DEVICE
    with pytest.raises(ValueError):
        read(stream=0, tokens=-1)


def test_calls_without_a_gpu():
    if tx.load().tx_device_available():
        pytest.skip("there is a GPU")
    for call in (append, attend, read):
        kw = {"workspace": torch.zeros(1 << 23, dtype=torch.uint8)} if call is attend else {}
        with pytest.raises((tx.TxError, RuntimeError)) as e:
            call(stream=0, **kw)
        assert not isinstance(e.value, tx.TxError) or e.value.code in (tx.ERR_NO_DEVICE, tx.ERR_WORKSPACE,
                                                                     tx.ERR_HIP)


def _attn4(**kw):
    base = dict(T=4, B=4, pages=100, table_width=50, Hq=32, Hkv=8, head_dim=128, page_size=16, dtype=tx.BF16,
                cache_type=tx.F4E2M1, causal=1, window=0, ragged=0, sm_scale=0.1, q_st=32 * 256, q_sh=256,
                o_st=32 * 256, o_sh=256, k_sp=16 * 8 * 128, k_st=128, k_sh=16 * 128, v_sp=16 * 8 * 128, v_st=128,
                v_sh=16 * 128, table_s=50)
    scales = dict(mode=tx.SCALE_MX32, reserved=0, k_sp=16 * 8 * 8, k_st=1, k_sh=8 * 16, k_sb=16, v_sp=16 * 8 * 8,
                  v_st=1, v_sh=8 * 16, v_sb=16)
    for k, v in kw.items():
        (scales if k in ("mode", "reserved") or k.endswith("_sb") or k.startswith("s_") else base)[
            k.replace("s_k", "k").replace("s_v", "v")] = v
    d, p = capi.PagedAttn4Desc(capi.PagedAttnDesc(**base), capi.BlockScales(**scales)), capi.PagedAttn4Plan()
    return tx.load().tx_paged_attn4_plan_create(ctypes.byref(d), ctypes.byref(p)), p


@pytest.mark.parametrize("T,B,G,D,rows", [(4, 4, 4, 128, 16), (4, 4, 16, 64, 16), (4, 4, 17, 64, 32),
                                          (8, 1, 4, 64, 32), (9, 1, 4, 64, 128), (9, 1, 4, 96, 32),
                                          (16, 1, 4, 128, 32), (17, 1, 4, 128, 128), (0, 0, 4, 128, 0),
                                          (300, 4, 1, 128, 128)])
def test_form_by_rows(T, B, G, D, rows):
    rc, p = _attn4(T=T, B=B, Hq=2 * G, Hkv=2, ragged=1, q_st=2 * G * 256, o_st=2 * G * 256, head_dim=D)
    D = 128 if D == 128 else 96 if D == 96 else 64  # (the dims that a head is computed in)
    assert rc == tx.OK and p.rows == rows
    assert p.grid_x == p.units and p.slots == 2 * p.units and p.units * 4 <= 65536
    # the arrival counters, and a place for each part: sums, maximum and sum of p of every row
    assert p.workspace_bytes == (65536 + p.slots * rows * (D + 2) * 4 if T else 0)


@pytest.mark.parametrize("kw,code", [
    (dict(mode=tx.SCALE_BLOCK128), tx.ERR_UNSUPPORTED), (dict(reserved=1), tx.ERR_INVALID),
    (dict(k_sb=-1), tx.ERR_INVALID), (dict(s_v_sp=2 ** 62), tx.ERR_UNSUPPORTED),
    (dict(cache_type=tx.F8E4M3), tx.ERR_UNSUPPORTED), (dict(head_dim=120), tx.ERR_UNSUPPORTED),
    (dict(k_st=72), tx.ERR_INVALID), (dict(v_sh=8), tx.ERR_INVALID), (dict(page_size=24), tx.ERR_UNSUPPORTED),
    (dict(T=2 ** 24, B=1, ragged=1, table_width=2 ** 26, table_s=2 ** 26), tx.ERR_UNSUPPORTED)])
def test_plans_refused(kw, code):
    rc, _ = _attn4(**kw)
    assert rc == code, tx.load().tx_get_last_error()


def test_a_plan_changed_by_hand_is_refused():
    rc, p = _attn4()
    assert rc == tx.OK
    p.units -= 1
    assert tx.load().tx_paged_attn4_launch(ctypes.byref(p), *[None] * 13, 0, None) == tx.ERR_INVALID
    for kind in ("append4", "attn4", "read"):
        create = getattr(tx.load(), f"tx_paged_{kind}_plan_create")
        assert create(None, None) == tx.ERR_INVALID


@pytest.mark.parametrize("kind", ["mx", "nv"])
def test_what_the_oracle_holds(kind):
    """The oracle itself: no value is further from its own than half a step of its scale, and what the
    cache can hold stays as it is."""
    g = torch.Generator()
    g.manual_seed(1)
    x = torch.randn(64, 128, generator=g).to(BF).double() * torch.exp(torch.randn(64, 1, generator=g)).double()
    codes, sb = quantise(x, kind, BF)
    y = values(codes, sb, kind)
    unit = scale_values(sb, kind).repeat_interleave(BLOCK[kind], -1)
    assert bool(((x - y).abs() <= unit).all())  # half of the largest step, 2 of 6
    sure = (x / unit).abs() < 2.0
    assert bool(((x - y).abs() <= 0.25 * unit)[sure].all())
    held = LEVELS[torch.randint(0, 8, (8, 32), generator=g)]
    held[:, ::16] = 6.0
    codes, sb = quantise(held, kind, BF)
    assert torch.equal(values(codes, sb, kind), held)
    bad = held.clone()
    bad[0, 0], bad[1, 20] = math.nan, math.inf
    y = values(*quantise(bad, kind, BF), kind)
    assert bool(y[0, :16].isnan().all()) and bool(y[1, 16:].isnan().all()) and torch.equal(y[2:], held[2:])
