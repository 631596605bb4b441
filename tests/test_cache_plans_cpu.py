"""The paged attention's plans, and the module that reads tensors' forms, without a GPU."""
import ctypes
import math

import pytest

import triton_ext_amd as tx
from test_cache_cpu import _attn_plan
from triton_ext_amd import capi

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("T,B,G,rows", [(4, 4, 4, 16), (4, 4, 16, 16), (4, 4, 17, 32), (8, 1, 4, 32),
                                        (9, 1, 4, 128), (0, 0, 4, 0), (300, 4, 1, 128)])
def test_form_by_rows(T, B, G, rows):
    rc, p = _attn_plan(T=T, B=B, Hq=2 * G, Hkv=2, ragged=1, q_st=2 * G * 128, o_st=2 * G * 128)
    assert rc == tx.OK and p.rows == rows
    assert p.grid_x == p.units and p.slots == 2 * p.units
    # the arrival counters, and a place for each part: sums, maximum and sum of p of every row
    assert p.workspace_bytes == (65536 + p.slots * rows * 130 * 4 if T else 0)
    assert p.units * 4 <= 65536


@pytest.mark.parametrize("D,cache,per_cu", [(64, tx.BF16, 2), (80, tx.BF16, 2), (128, tx.F8E4M3, 2),
                                            (256, tx.BF16, 1), (256, tx.F8E4M3, 2)])
def test_workgroups_of_a_large_call(D, cache, per_cu):
    rc, p = _attn_plan(T=64, B=64, head_dim=D, cache_type=cache, table_width=4096, table_s=4096,
                       q_sh=256, q_st=2048, o_sh=256, o_st=2048, k_sh=256, k_st=512, k_sp=8192,
                       v_sh=256, v_st=512, v_sp=8192)
    assert rc == tx.OK and p.units == 256 * per_cu


def test_more_work_than_is_counted_is_refused():
    rc, _ = _attn_plan(T=2 ** 24, B=1, ragged=1, table_width=2 ** 26, table_s=2 ** 26)
    assert rc == tx.ERR_UNSUPPORTED and b"2^31" in tx.load().tx_get_last_error()


def test_forms():
    form = capi.calls().form
    a = torch.zeros(3, 4)
    assert form("x", a, None, 1.5, True, 7, (a, a)) == form("x", torch.ones(3, 4), None, 1.5, True, 7, [a, a])
    seen = {form(*args) for args in (
        ("x",), ("y",), (a,), (a.t(),), (a.half(),), (torch.zeros(4, 3),), (torch.zeros(12),),
        (torch.zeros(3, 8)[:, ::2],), (a, None), (None, a), (1,), (1.0,), (True,), (0,), (0.0,),
        (False,), (None,), ((a,),), ((a, a),), (a, a), ((), a), ("x", "y"), ("xy",), (-0.0,),
        (math.inf,), (torch.zeros(()),), (torch.zeros(0),), (a.to(torch.bfloat16),))}
    assert len(seen) == 28
    assert form(torch.zeros(2, device="meta")) != form(torch.zeros(2))
    for bad in (object(), {}, 2 ** 70, torch.zeros(2, 2).to_sparse()):
        with pytest.raises((TypeError, OverflowError)):
            form(bad)


def test_calls_by_address():
    native = capi.calls()
    a = torch.arange(4)
    assert native.addresses([a, a[1:], None]) == b"".join(
        x.to_bytes(8, "little") for x in (a.data_ptr(), a.data_ptr() + 8, 0))
    got = []
    kind = ctypes.CFUNCTYPE(ctypes.c_int, *[ctypes.c_uint64] * 8)

    def take(*args):
        got.append(args)
        return -3
    fn = kind(take)
    where = ctypes.cast(fn, ctypes.c_void_p).value
    word = b"12345678"
    assert native.call(where, a, None, 5, 2 ** 63, word, a[2:], 0, 9) == -3
    assert got[0][:4] == (a.data_ptr(), 0, 5, 2 ** 63) and got[0][5:] == (a.data_ptr() + 16, 0, 9)
    assert ctypes.string_at(got[0][4], 8) == word
    for bad in ((), (0, a), (None, a), (where, 1.5), (where, -1), (where,) + (a,) * 21):
        with pytest.raises((TypeError, ValueError, OverflowError)):
            native.call(*bad)
    with pytest.raises(TypeError):
        native.addresses(a)
