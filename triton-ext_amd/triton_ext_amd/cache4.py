"""A paged cache held in 4 bits, and any paged cache read back (include/triton_ext/tx_cache4.h).

The forms of paged_append and paged_attention (cache.py) that block scales select, and paged_read.
Codes are uint8 [pages, page_size, Hkv, D / 2], two e2m1 values a byte, the even dim in the low
four bits; block scales are [pages, page_size, Hkv, D / 32] uint8 (e8m0) or [.., D / 16]
float8_e4m3fn, as dot_scaled takes them."""
from . import cache, capi
from .cache import (_append_tokens, _attention_q, _cache_books, _calls, _dense, _dense_last, _forms,
                    _keep, _maker, _plan, _same_device, _tokens)
from .dot import _current_stream, _current_workspace, _there, _tx_of

_NO_SCALES = (0,) * 10


def _code_checks(k_cache, v_cache, k_block_scale, v_block_scale, Hkv, D):
    """Refuses codes and block scales that do not go together, of heads of D dims (None: what the
    codes say)."""
    import torch
    if k_block_scale is None or v_block_scale is None:
        raise ValueError("k_block_scale and v_block_scale go together")
    if (k_cache.dtype != torch.uint8 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape
            or v_cache.dtype != k_cache.dtype):
        raise ValueError("with block scales, k_cache and v_cache must be uint8 codes [pages, "
                         f"page_size, Hkv, D / 2]: {k_cache.dtype} {tuple(k_cache.shape)}, "
                         f"{v_cache.dtype} {tuple(v_cache.shape)}")
    if D is None:
        Hkv, D = k_cache.shape[2], 2 * k_cache.shape[3]
    if tuple(k_cache.shape[2:]) != (Hkv, D // 2) or D % 32:
        raise ValueError(f"the cache holds codes of {tuple(k_cache.shape[2:])}, not ({Hkv}, {D} / 2),"
                         " D a multiple of 32")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the caches' last dimension must be contiguous")
    block = {torch.uint8: 32, torch.float8_e4m3fn: 16}.get(k_block_scale.dtype)
    if block is None:
        raise NotImplementedError(f"block scales of {k_block_scale.dtype}: uint8 (e8m0, of 32 dims) "
                                  "or float8_e4m3fn (of 16)")
    want = tuple(k_cache.shape[:3]) + (D // block,)
    for t, name in ((k_block_scale, "k_block_scale"), (v_block_scale, "v_block_scale")):
        if t.dtype != k_block_scale.dtype or tuple(t.shape) != want:
            raise ValueError(f"{name} must be {k_block_scale.dtype} {want}, got {t.dtype} "
                             f"{tuple(t.shape)}")
    return D


def _head_scales(k_scale, v_scale, Hkv):
    import torch
    for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if t is not None and (t.dtype != torch.float32 or t.shape != (Hkv,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 [{Hkv}] tensor")


def _scales_of(k_block_scale, v_block_scale):
    """tx_block_scales, field by field."""
    if k_block_scale is None:
        return _NO_SCALES
    mode = capi.SCALE_MX32 if k_block_scale.element_size() == 1 and not k_block_scale.is_floating_point() \
        else capi.SCALE_NV16
    return (mode, 0) + k_block_scale.stride() + v_block_scale.stride()


def append(k, v, k_cache, v_cache, page_table, kv_len, cu_q, q, inv_freq, interleaved, scale, k_scale,
           v_scale, k_block_scale, v_block_scale, q_out, stream):
    native = cache._native or _calls()
    form = native.form("append4", k, v, k_cache, v_cache, page_table, kv_len, cu_q, q, inv_freq,
                       bool(interleaved), float(scale), k_scale, v_scale, k_block_scale, v_block_scale,
                       q_out)
    found = _forms.get(form)
    if found is None:
        _append_tokens(k, v, q, inv_freq, q_out)
        T, Hkv, D = k.shape
        _code_checks(k_cache, v_cache, k_block_scale, v_block_scale, Hkv, D)
        _head_scales(k_scale, v_scale, Hkv)
        _cache_books(page_table, kv_len, cu_q, T)
        _same_device(k.device, v=v, k_cache=k_cache, v_cache=v_cache, page_table=page_table,
                     kv_len=kv_len, cu_q=cu_q, q=q, inv_freq=inv_freq, k_scale=k_scale,
                     v_scale=v_scale, k_block_scale=k_block_scale, v_block_scale=v_block_scale,
                     q_out=q_out)
        given = (k, v, kv_len, cu_q, q, inv_freq)
        dense = tuple(None if t is None else f(t) for f, t in zip(
            (_dense_last, _dense_last, _dense, _dense, _dense_last, _dense), given))
        if any(a is not b for a, b in zip(dense, given)):  # copied, and the copies' form looked up
            k, v, kv_len, cu_q, q, inv_freq = dense
            return append(k, v, k_cache, v_cache, page_table, kv_len, cu_q, q, inv_freq, interleaved,
                          scale, k_scale, v_scale, k_block_scale, v_block_scale, q_out, stream)
        Hq, q_st, make = 0, (0, 0, 0, 0), None
        if q is not None:
            make = _maker(q)
            like = make(q) if q_out is None else q_out
            Hq, q_st = q.shape[1], q.stride()[:2] + like.stride()[:2]
        base = capi.PagedAppendDesc(
            T, kv_len.shape[0], k_cache.shape[0], page_table.shape[1], Hq, Hkv, D,
            0 if inv_freq is None else 2 * inv_freq.shape[0], k_cache.shape[1], _tx_of(k.dtype),
            capi.F4E2M1, int(bool(interleaved)), int(cu_q is not None), float(scale),
            *q_st, *k.stride()[:2], *v.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3],
            page_table.stride(0))
        found = _keep(form, (_plan("paged_append4", capi.PagedAppend4Desc, capi.PagedAppend4Plan,
                                   (base, _scales_of(k_block_scale, v_block_scale))), make))
    (launch, plan, _), make = found
    if q is not None and q_out is None:
        q_out = make(q)
    rc = native.call(launch, plan, q, k, v, q_out, k_cache, v_cache, k_block_scale, v_block_scale,
                     page_table, kv_len, cu_q, inv_freq, k_scale, v_scale,
                     _current_stream(k.device) if stream is None else stream)
    if rc:
        capi.check(rc)
    return q_out


def attention(q, k_cache, v_cache, page_table, kv_len, cu_q, sm_scale, causal, window, k_scale, v_scale,
              k_block_scale, v_block_scale, out, return_lse, workspace, stream):
    import torch
    native = cache._native or _calls()
    form = native.form("attention4", q, k_cache, v_cache, page_table, kv_len, cu_q, float(sm_scale),
                       bool(causal), int(window), k_scale, v_scale, k_block_scale, v_block_scale, out)
    found = _forms.get(form)
    if found is None or q.data_ptr() % 16:
        _attention_q(q, out)
        T, Hq, D = q.shape
        _code_checks(k_cache, v_cache, k_block_scale, v_block_scale,
                     k_cache.shape[2] if k_cache.dim() == 4 else 0, D)
        Hkv = k_cache.shape[2]
        _head_scales(k_scale, v_scale, Hkv)
        _cache_books(page_table, kv_len, cu_q, T)
        _same_device(q.device, k_cache=k_cache, v_cache=v_cache, page_table=page_table, kv_len=kv_len,
                     cu_q=cu_q, k_scale=k_scale, v_scale=v_scale, k_block_scale=k_block_scale,
                     v_block_scale=v_block_scale, out=out)
        s0, s1, s2 = q.stride()
        qc = q
        if s2 != 1 or s0 % 8 or s1 % 8 or q.data_ptr() % 16:
            qc = torch.empty(q.shape, dtype=q.dtype, device=q.device).copy_(q)
        dense = (_dense(kv_len), None if cu_q is None else _dense(cu_q))
        if qc is not q or dense[0] is not kv_len or dense[1] is not cu_q:
            return attention(qc, k_cache, v_cache, page_table, *dense, sm_scale, causal, window, k_scale,
                             v_scale, k_block_scale, v_block_scale, out, return_lse, workspace, stream)
        make = _maker(q)
        like = make(q) if out is None else out
        base = capi.PagedAttnDesc(
            T, kv_len.shape[0], k_cache.shape[0], page_table.shape[1], Hq, Hkv, D, k_cache.shape[1],
            _tx_of(q.dtype), capi.F4E2M1, int(bool(causal)), int(window), int(cu_q is not None),
            float(sm_scale), *q.stride()[:2], *like.stride()[:2], *k_cache.stride()[:3],
            *v_cache.stride()[:3], page_table.stride(0))
        found = _keep(form, (_plan("paged_attn4", capi.PagedAttn4Desc, capi.PagedAttn4Plan,
                                   (base, _scales_of(k_block_scale, v_block_scale))), make))
    (launch, plan, needs), make = found
    if out is None:
        out = make(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    if stream is None:
        stream = _current_stream(q.device)
    ws = workspace if workspace is not None else _current_workspace(needs, q.device, stream)
    rc = native.call(launch, plan, q, k_cache, v_cache, k_block_scale, v_block_scale, page_table, kv_len,
                     cu_q, k_scale, v_scale, out, lse, ws,
                     0 if ws is None else ws.numel() * ws.element_size(), stream)
    if rc:
        capi.check(rc)
    return (out, lse) if return_lse else out


def paged_read(k_cache, v_cache, page_table, kv_len, cu_q=None, *, tokens=None, dtype=None, k_scale=None,
               v_scale=None, k_block_scale=None, v_block_scale=None, k_out=None, v_out=None,
               stream=None):
    """Tokens out of a paged cache, as dense k and v [T, Hkv, D]: rows cu_q[b] .. cu_q[b + 1] - 1 are
    the last so many tokens of sequence b (cu_q [B + 1], T = `tokens`; None: one token each, the
    newest).  So cu_q of a paged_append gives the tokens that it wrote, as the cache holds them, and
    the starts of whole lengths whole sequences.

    The cache is of fp16, bf16 or float8_e4m3fn (times k_scale, v_scale, fp32 [Hkv]), or uint8 codes
    under block scales (see paged_append).  dtype is fp16, bf16 or fp32 (None: the cache's own, where
    it has 16 bits): the products are taken in fp32 and rounded once.  Rows of tokens without a
    page, and rows of no sequence, are 0.  k_out and v_out: the tensors to write."""
    device = kv_len.device
    if stream is not None and stream != _current_stream(device):
        return _there(device, stream, paged_read, k_cache, v_cache, page_table, kv_len, cu_q,
                      tokens=tokens, dtype=dtype, k_scale=k_scale, v_scale=v_scale,
                      k_block_scale=k_block_scale, v_block_scale=v_block_scale, k_out=k_out, v_out=v_out)
    import torch
    native = cache._native or _calls()
    form = native.form("read", k_cache, v_cache, page_table, kv_len, cu_q,
                       None if tokens is None else cache.index(tokens), str(dtype), k_scale, v_scale,
                       k_block_scale, v_block_scale, k_out, v_out)
    found = _forms.get(form)
    if found is None:
        T, Hkv, D, dtype = _read_checks(k_cache, v_cache, page_table, kv_len, cu_q, tokens, dtype,
                                        k_scale, v_scale, k_block_scale, v_block_scale, k_out, v_out)
        dense = (_dense(kv_len), None if cu_q is None else _dense(cu_q))
        if dense[0] is not kv_len or dense[1] is not cu_q:
            return paged_read(k_cache, v_cache, page_table, *dense, tokens=tokens, dtype=dtype,
                              k_scale=k_scale, v_scale=v_scale, k_block_scale=k_block_scale,
                              v_block_scale=v_block_scale, k_out=k_out, v_out=v_out, stream=stream)
        rows = (Hkv * D, D)
        found = _keep(form, (_plan(
            "paged_read", capi.PagedReadDesc, capi.PagedReadPlan,
            (T, kv_len.shape[0], k_cache.shape[0], page_table.shape[1], Hkv, D, k_cache.shape[1],
             capi.F4E2M1 if k_block_scale is not None else _tx_of(k_cache.dtype), _tx_of(dtype),
             int(cu_q is not None)) + k_cache.stride()[:3] + v_cache.stride()[:3]
            + (rows if k_out is None else k_out.stride()[:2])
            + (rows if v_out is None else v_out.stride()[:2]) + (page_table.stride(0),)
            + (_scales_of(k_block_scale, v_block_scale),)),
            # what new rows are like: a view of one element, which empty_like makes packed
            torch.empty((), dtype=dtype, device=device).expand(T, Hkv, D), torch.empty_like))
    (launch, plan, _), like, make = found
    if k_out is None:
        k_out = make(like)
    if v_out is None:
        v_out = make(like)
    rc = native.call(launch, plan, k_cache, v_cache, k_block_scale, v_block_scale, page_table, kv_len,
                     cu_q, k_scale, v_scale, k_out, v_out,
                     _current_stream(device) if stream is None else stream)
    if rc:
        capi.check(rc)
    return k_out, v_out


def _read_checks(k_cache, v_cache, page_table, kv_len, cu_q, tokens, dtype, k_scale, v_scale,
                 k_block_scale, v_block_scale, k_out, v_out):
    import torch
    if k_block_scale is not None or v_block_scale is not None:
        D = _code_checks(k_cache, v_cache, k_block_scale, v_block_scale, None, None)
        Hkv = k_cache.shape[2]
    else:
        if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
            raise ValueError("k_cache and v_cache must share one [pages, page_size, Hkv, D] shape and "
                             f"type: {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
        if k_cache.dtype not in (torch.float16, torch.bfloat16, torch.float8_e4m3fn):
            raise NotImplementedError(f"a cache of {k_cache.dtype}: fp16, bf16, float8_e4m3fn, or "
                                      "uint8 codes with block scales")
        Hkv, D = k_cache.shape[2:]
        if D > 1 and (k_cache.stride(3) != 1 or v_cache.stride(3) != 1):
            raise ValueError("the caches' last dimension must be contiguous")
        if k_cache.dtype != torch.float8_e4m3fn and (k_scale is not None or v_scale is not None):
            raise ValueError("k_scale and v_scale are for float8_e4m3fn caches and codes")
    _head_scales(k_scale, v_scale, Hkv)
    if dtype is None:
        if k_out is not None:
            dtype = k_out.dtype
        elif k_cache.dtype in (torch.float16, torch.bfloat16):
            dtype = k_cache.dtype
        else:
            raise ValueError(f"dtype: fp16, bf16 or fp32 for a cache of {k_cache.dtype}")
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise NotImplementedError(f"dtype {dtype}: fp32, fp16 and bf16 are implemented")
    B = kv_len.shape[0] if kv_len.dim() == 1 else 0
    if cu_q is None:
        T = B if tokens is None else cache.index(tokens)
    elif tokens is not None:
        T = cache.index(tokens)
    elif k_out is not None and k_out.dim() == 3:
        T = k_out.shape[0]
    else:
        raise ValueError("cu_q needs `tokens`, the rows to write (nothing is read on the host)")
    if T < 0:
        raise ValueError(f"tokens {T}")
    _cache_books(page_table, kv_len, cu_q, T)
    for t, name in ((k_out, "k_out"), (v_out, "v_out")):
        if t is not None:
            _tokens(t, name, Hkv, D, dtype, T)
            if D > 1 and t.stride(2) != 1:
                raise ValueError(f"{name}: the last dimension must be contiguous")
    _same_device(kv_len.device, k_cache=k_cache, v_cache=v_cache, page_table=page_table, cu_q=cu_q,
                 k_scale=k_scale, v_scale=v_scale, k_block_scale=k_block_scale,
                 v_block_scale=v_block_scale, k_out=k_out, v_out=v_out)
    return T, Hkv, D, dtype
