"""Rotary positions, a paged key/value cache and the attention that reads it, over torch
device tensors (include/triton_ext/tx_cache.h).

A cache is a pair of tensors [pages, page_size, Hkv, D] for k and v, in any order in
memory with D contiguous (a permuted [pages, Hkv, page_size, D] does), its books int32
tensors: page_table [S, W], kv_len [S] and refs [pages] (how many table entries hold a
page).  Token j of sequence b lies in page page_table[b, j // page_size], slot
j % page_size.  A decoding step is

    page_table, kv_len, refs, missing = page_reserve(page_table, kv_len, refs, kv_len + 1, 16)
    q = paged_append(k, v, k_cache, v_cache, page_table, kv_len, q=q, inv_freq=inv_freq)
    o = paged_attention(q, k_cache, v_cache, page_table, kv_len, sm_scale=D ** -0.5)

and a chunk of several new tokens a sequence the same with cu_q, their starts in q, k
and v.  Nothing here reads device memory on the host: every call can be captured into
a graph and replayed with other contents.

stream: the handle of the HIP stream to run on, torch's current one if None.  All of a call is in order
on it: the copies of arguments that the kernels do not take as they lie, and the results, whose memory
is that stream's.  The arguments have to be ready there.

rotary has a gradient in torch's backward pass; the calls on the cache are for generation and have none.
"""
import ctypes
import functools
import math
from operator import index

from . import capi
from .dot import _COUNTERS, _current_stream, _current_workspace, _there, _tx_of

# What a call's checks found for arguments of one form (shapes, strides, types, devices and
# numbers, as bytes), so that a call of the same form goes to the launch at once.  Nothing here
# depends on a tensor's address or contents.
_forms = {}
_native = None


def _calls():
    """The module that makes forms and calls, loaded with the first call."""
    global _native
    if _native is None:
        _native = capi.calls()
    return _native


def _keep(form, found):
    if len(_forms) >= 4096:  # a program of ever new sizes
        _forms.clear()
    _forms[form] = found
    return found


def _plan(kind, desc_type, plan_type, key):
    """The plan of a descriptor with these fields in order, and its launch: (function, address of
    the plan, plan)."""
    p = plan_type()
    capi.check(getattr(capi.load(), f"tx_{kind}_plan_create")(
        ctypes.byref(desc_type(*key)), ctypes.byref(p)))
    return capi.address(f"tx_{kind}_launch"), ctypes.addressof(p), p


def _is_int32(t, name, dims):
    import torch
    if t.dtype != torch.int32 or t.dim() != dims:
        raise ValueError(f"{name} must be an int32 tensor of {dims} dimension(s), got "
                         f"{t.dtype} {tuple(t.shape)}")


def _dense(t):
    return t if t.is_contiguous() else t.contiguous()


def _int32(t, name, dims):
    _is_int32(t, name, dims)
    return _dense(t)


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _dense_last(t):
    """t, or a copy, with its last dimension contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _new(t):
    """A new packed tensor like t."""
    import torch
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _maker(t):
    """What makes new tensors like t, with their last dimension contiguous: empty_like, the
    cheapest call, where it does."""
    import torch
    out = torch.empty_like(t)
    return torch.empty_like if out.stride(-1) == 1 or out.shape[-1] <= 1 else _new


def rotary_frequencies(rot_dim, base=10000.0, *, scaling=None, factor=1.0, context=4096,
                       turns=(1.0, 32.0), device=None):
    """The frequencies of `rot_dim` rotated dims, base^(-2 i / rot_dim), as an fp32 tensor
    [rot_dim // 2], and the factor for cos and sin (`scale` of rotary and paged_append).

    scaling, for contexts `factor` times as long as the `context` trained on: None;
    "linear" (positions divided by factor); "ntk" (base times factor^(rot_dim /
    (rot_dim - 2))); "yarn" (frequencies of fewer than turns[0] turns over the context
    divided by factor, those of more than turns[1] kept, a line between, and a scale
    of 0.1 ln(factor) + 1)."""
    import torch
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim {rot_dim}: an even number of dims")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling {scaling!r}: None, 'linear', 'ntk' or 'yarn'")
    if scaling is not None and not factor >= 1.0:
        raise ValueError(f"factor {factor}: at least 1")
    base = float(base)
    if scaling == "ntk":
        if rot_dim < 4:
            raise ValueError("ntk scaling needs a rot_dim of 4 or more")
        base *= factor ** (rot_dim / (rot_dim - 2))
    f = base ** (-2.0 * torch.arange(rot_dim // 2, dtype=torch.float64) / rot_dim)
    scale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        lo, hi = turns
        keep = ((context * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        f = f / factor * (1 - keep) + f * keep
        scale = 0.1 * math.log(factor) + 1.0
    return f.to(torch.float32).to(device), scale


def rotary(x, positions, inv_freq, *, interleaved=False, scale=1.0, inverse=False, out=None,
           stream=None):
    """Rotary positions: pair i of every head of x goes to (x1 c - x2 s, x2 c + x1 s) with
    c = scale cos(position * inv_freq[i]), s = scale sin(..), the angle in 64 bits.

    x [T, H, D] with positions [T], or [Z, H, N, D] (the layout of attention()) with
    positions [N] or [Z, N]; fp16, bf16 or fp32, any strides with D contiguous;
    positions int32 or int64; inv_freq fp32 [rot_dim / 2] (rotary_frequencies), rot_dim
    <= D: the dims past it are copied.  The pairs are dims (i, i + rot_dim / 2), or
    (2 i, 2 i + 1) when interleaved.  inverse: the transposed map, which takes the
    gradient of the result to that of x; torch's backward pass calls it by itself where x
    requires a gradient (positions and inv_freq get none).  out may be x itself; a result in
    it has no gradient, so an x that requires one is refused."""
    if stream is not None and stream != _current_stream(x.device):
        return _there(x.device, stream, rotary, x, positions, inv_freq, interleaved=interleaved,
                      scale=scale, inverse=inverse, out=out)
    if x.requires_grad and _grad_enabled():
        if out is not None:
            raise ValueError("out takes no gradient: x requires one (x.detach(), or torch.no_grad())")
        return _differentiable()(x, positions, inv_freq, interleaved, scale, inverse)
    native = _native or _calls()
    form = native.form("rotary", x, positions, inv_freq, bool(interleaved), float(scale),
                       bool(inverse), out)
    found = _forms.get(form)
    if found is None:
        _rotary_checks(x, positions, inv_freq, out)
        # what the kernel does not take as it lies is copied, and the copy's form looked up
        xc = _dense_last(x)
        pc, fc = positions.contiguous(), inv_freq.contiguous()
        if xc is not x or pc is not positions or fc is not inv_freq:
            return rotary(xc, pc, fc, interleaved=interleaved, scale=scale, inverse=inverse,
                          out=out, stream=stream)
        make = _maker(x)
        found = _keep(form, (_rotary_plan(x, positions, inv_freq, interleaved, scale, inverse,
                                          make(x) if out is None else out), make))
    (launch, plan, _), make = found
    if out is None:
        out = make(x)
    rc = native.call(launch, plan, x, positions, inv_freq, out,
                     _current_stream(x.device) if stream is None else stream)
    if rc:
        capi.check(rc)
    return out


def _grad_enabled():
    import torch
    return torch.is_grad_enabled()


@functools.lru_cache(None)
def _differentiable():
    """rotary with its gradient."""
    import torch

    class Rotary(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, positions, inv_freq, interleaved, scale, inverse):
            ctx.save_for_backward(positions, inv_freq)
            ctx.how = interleaved, scale, inverse
            return rotary(x, positions, inv_freq, interleaved=interleaved, scale=scale,
                          inverse=inverse)

        @staticmethod
        def backward(ctx, dy):
            interleaved, scale, inverse = ctx.how
            return (rotary(dy, *ctx.saved_tensors, interleaved=interleaved, scale=scale,
                           inverse=not inverse),) + (None,) * 5
    return Rotary.apply


def _rotary_checks(x, positions, inv_freq, out):
    import torch
    if x.dim() not in (3, 4):
        raise ValueError(f"x must be [T, H, D] or [Z, H, N, D], got {tuple(x.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1:
        raise ValueError("inv_freq must be an fp32 vector")
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise NotImplementedError(f"x: fp32, fp16 and bf16 are implemented, got {x.dtype}")
    _same_device(x.device, positions=positions, inv_freq=inv_freq, out=out)
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype
                            or (out.stride(-1) != 1 and out.shape[-1] > 1)):
        raise ValueError("out must be as x, with its last dimension contiguous")
    N = x.shape[0] if x.dim() == 3 else x.shape[2]
    if positions.shape != (N,) and (x.dim() == 3 or positions.shape != (x.shape[0], N)):
        raise ValueError(f"positions must be [{N}]" + (f" or [{x.shape[0]}, {N}]" if x.dim() == 4
                                                       else "") + f", got {tuple(positions.shape)}")


def _rotary_plan(x, positions, inv_freq, interleaved, scale, inverse, out):
    xs, os_ = x.stride(), out.stride()
    if x.dim() == 3:
        (N, H, D), Z = x.shape, 1
        st = (0, xs[0], xs[1], 0, os_[0], os_[1])
    else:
        Z, H, N, D = x.shape
        st = (xs[0], xs[2], xs[1], os_[0], os_[2], os_[1])
    return _plan(
        "rotary", capi.RotaryDesc, capi.RotaryPlan,
        (Z, N, H, D, 2 * inv_freq.shape[0], _tx_of(x.dtype), int(bool(interleaved)),
         int(bool(inverse)), 8 * positions.element_size(), float(scale), 0,
         N if positions.dim() == 2 else 0) + st)


def _cache_checks(k_cache, v_cache, page_table, kv_len, cu_q, k_scale, v_scale, T, Hkv, D, dtype):
    """What paged_append and paged_attention ask alike."""
    import torch
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must share one [pages, page_size, Hkv, D] shape and "
                         f"type: {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if tuple(k_cache.shape[2:]) != (Hkv, D):
        raise ValueError(f"the cache holds heads of {tuple(k_cache.shape[2:])}, not ({Hkv}, {D})")
    if k_cache.dtype != dtype and k_cache.dtype != torch.float8_e4m3fn:
        raise NotImplementedError(f"a cache of {k_cache.dtype} under {dtype}: the same type, or "
                                  "float8_e4m3fn")
    if D > 1 and (k_cache.stride(3) != 1 or v_cache.stride(3) != 1):
        raise ValueError("the caches' last dimension must be contiguous")
    for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if t is None:
            continue
        if k_cache.dtype != torch.float8_e4m3fn:
            raise ValueError(f"{name} is for float8_e4m3fn caches")
        if t.dtype != torch.float32 or t.shape != (Hkv,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous fp32 [{Hkv}] tensor")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or (
            page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be an int32 [sequences, entries] tensor with contiguous "
                         "rows")
    _is_int32(kv_len, "kv_len", 1)
    B = kv_len.shape[0]
    if page_table.shape[0] != B:
        raise ValueError(f"page_table has {page_table.shape[0]} rows, kv_len {B}")
    if cu_q is None:
        if T != B:
            raise ValueError(f"{T} new tokens of {B} sequences: give cu_q")
    else:
        _is_int32(cu_q, "cu_q", 1)
        if cu_q.shape[0] != B + 1:
            raise ValueError(f"cu_q must be [{B + 1}], got {tuple(cu_q.shape)}")


def _tokens(t, name, heads, D, dtype, T):
    """Refuses t unless it is [T, heads, D]."""
    if t.dim() != 3 or tuple(t.shape) != (T, heads, D):
        raise ValueError(f"{name} must be [{T}, {heads}, {D}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}, not {dtype}")


def paged_append(k, v, k_cache, v_cache, page_table, kv_len, cu_q=None, *, q=None, inv_freq=None,
                 interleaved=False, scale=1.0, k_scale=None, v_scale=None, q_out=None,
                 stream=None):
    """New tokens into a paged cache: k, v [T, Hkv, D] go to the pages of their sequences,
    k (and q [T, Hq, D], which is returned, in q_out if given) rotated at the token's
    position first when inv_freq is given (see rotary for interleaved and scale).

    kv_len [B] counts the new tokens too, cu_q [B + 1] says which rows are whose (None:
    one token each): row cu_q[b] + i of sequence b's n is its token kv_len[b] - n + i.
    The pages must be there (page_reserve); a token without one is not written.  fp16 or
    bf16; a float8_e4m3fn cache holds k / k_scale[head] and v / v_scale[head] (fp32 [Hkv];
    None: 1), saturated.  Rows of q from cu_q[B] on come back as they are."""
    if stream is not None and stream != _current_stream(k.device):
        return _there(k.device, stream, paged_append, k, v, k_cache, v_cache, page_table, kv_len,
                      cu_q, q=q, inv_freq=inv_freq, interleaved=interleaved, scale=scale,
                      k_scale=k_scale, v_scale=v_scale, q_out=q_out)
    native = _native or _calls()
    form = native.form("append", k, v, k_cache, v_cache, page_table, kv_len, cu_q, q, inv_freq,
                       bool(interleaved), float(scale), k_scale, v_scale, q_out)
    found = _forms.get(form)
    if found is None:
        _append_checks(k, v, k_cache, v_cache, page_table, kv_len, cu_q, q, inv_freq, k_scale,
                       v_scale, q_out)
        given = (k, v, kv_len, cu_q, q, inv_freq)
        dense = tuple(None if t is None else f(t) for f, t in zip(
            (_dense_last, _dense_last, _dense, _dense, _dense_last, _dense), given))
        if any(a is not b for a, b in zip(dense, given)):  # copied, and the copies' form looked up
            k, v, kv_len, cu_q, q, inv_freq = dense
            return paged_append(k, v, k_cache, v_cache, page_table, kv_len, cu_q, q=q,
                                inv_freq=inv_freq, interleaved=interleaved, scale=scale,
                                k_scale=k_scale, v_scale=v_scale, q_out=q_out, stream=stream)
        T, Hkv, D = k.shape
        Hq, q_st, make = 0, (0, 0, 0, 0), None
        if q is not None:
            make = _maker(q)
            if q_out is None:
                q_out = make(q)
            Hq, q_st = q.shape[1], q.stride()[:2] + q_out.stride()[:2]
        found = _keep(form, (_plan(
            "paged_append", capi.PagedAppendDesc, capi.PagedAppendPlan,
            (T, kv_len.shape[0], k_cache.shape[0], page_table.shape[1], Hq, Hkv, D,
             0 if inv_freq is None else 2 * inv_freq.shape[0], k_cache.shape[1], _tx_of(k.dtype),
             _tx_of(k_cache.dtype), int(bool(interleaved)), int(cu_q is not None), float(scale))
            + q_st + k.stride()[:2] + v.stride()[:2] + k_cache.stride()[:3] + v_cache.stride()[:3]
            + (page_table.stride(0),)), make))
    (launch, plan, _), make = found
    if q is not None and q_out is None:
        q_out = make(q)
    rc = native.call(launch, plan, q, k, v, q_out, k_cache, v_cache, page_table, kv_len, cu_q,
                     inv_freq, k_scale, v_scale,
                     _current_stream(k.device) if stream is None else stream)
    if rc:
        capi.check(rc)
    return q_out


def _append_checks(k, v, k_cache, v_cache, page_table, kv_len, cu_q, q, inv_freq, k_scale, v_scale,
                   q_out):
    import torch
    if k.dim() != 3:
        raise ValueError(f"k must be [T, Hkv, D], got {tuple(k.shape)}")
    T, Hkv, D = k.shape
    dtype = k.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"k: fp16 and bf16 are implemented, got {dtype}")
    _tokens(v, "v", Hkv, D, dtype, T)
    _cache_checks(k_cache, v_cache, page_table, kv_len, cu_q, k_scale, v_scale, T, Hkv, D, dtype)
    _same_device(k.device, v=v, k_cache=k_cache, v_cache=v_cache, page_table=page_table,
                 kv_len=kv_len, cu_q=cu_q, q=q, inv_freq=inv_freq, k_scale=k_scale,
                 v_scale=v_scale, q_out=q_out)
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.dim() != 1):
        raise ValueError("inv_freq must be an fp32 vector")
    if q is None:
        if q_out is not None:
            raise ValueError("q_out without q")
        return
    _tokens(q, "q", q.shape[1] if q.dim() == 3 else 0, D, dtype, T)
    if q_out is not None and (q_out.shape != q.shape or q_out.dtype != dtype
                              or (D > 1 and q_out.stride(2) != 1)):
        raise ValueError("q_out must be as q, with its last dimension contiguous")


def paged_attention(q, k_cache, v_cache, page_table, kv_len, cu_q=None, *, sm_scale, causal=True,
                    window=0, k_scale=None, v_scale=None, out=None, return_lse=False,
                    workspace=None, stream=None):
    """Attention of the new tokens q [T, Hq, D] over a paged cache that holds them already
    (paged_append), Hq a multiple of Hkv (query head h reads key head h // (Hq // Hkv)).

    The new token at position p attends to its sequence's tokens j < kv_len[b] that have
    a page, j <= p if causal, j > p - window if window > 0; one that attends to nothing,
    and rows from cu_q[B] on, get 0.  fp16 or bf16, the cache in q's type or float8_e4m3fn
    (times k_scale, v_scale, fp32 [Hkv]), D a multiple of 8 (e4m3: 16) up to 256.  Returns
    o [T, Hq, D], with return_lse also log2 of the sum of e^(score), fp32 [T, Hq] (-inf
    where nothing is attended to).  cu_q as for paged_append."""
    if stream is not None and stream != _current_stream(q.device):
        return _there(q.device, stream, paged_attention, q, k_cache, v_cache, page_table, kv_len, cu_q,
                      sm_scale=sm_scale, causal=causal, window=window, k_scale=k_scale,
                      v_scale=v_scale, out=out, return_lse=return_lse, workspace=workspace)
    import torch
    native = _native or _calls()
    form = native.form("attention", q, k_cache, v_cache, page_table, kv_len, cu_q, float(sm_scale),
                       bool(causal), int(window), k_scale, v_scale, out)
    found = _forms.get(form)
    if found is None or q.data_ptr() % 16:
        _attention_checks(q, k_cache, v_cache, page_table, kv_len, cu_q, k_scale, v_scale, out)
        s0, s1, s2 = q.stride()
        qc = q
        if q.shape[2] % 8 == 0 and (s2 != 1 or s0 % 8 or s1 % 8 or q.data_ptr() % 16):
            qc = torch.empty(q.shape, dtype=q.dtype, device=q.device).copy_(q)
        given = (kv_len, cu_q)
        dense = (_dense(kv_len), None if cu_q is None else _dense(cu_q))
        if qc is not q or dense[0] is not given[0] or dense[1] is not given[1]:
            return paged_attention(qc, k_cache, v_cache, page_table, *dense, sm_scale=sm_scale,
                                   causal=causal, window=window, k_scale=k_scale, v_scale=v_scale,
                                   out=out, return_lse=return_lse, workspace=workspace,
                                   stream=stream)
        make = _maker(q)
        if out is None:
            out = make(q)
        T, Hq, D = q.shape
        plan = _plan("paged_attn", capi.PagedAttnDesc, capi.PagedAttnPlan,
                     (T, kv_len.shape[0], k_cache.shape[0], page_table.shape[1], Hq,
                      k_cache.shape[2], D, k_cache.shape[1], _tx_of(q.dtype), _tx_of(k_cache.dtype),
                      int(bool(causal)), int(window), int(cu_q is not None), float(sm_scale))
                     + q.stride()[:2] + out.stride()[:2] + k_cache.stride()[:3]
                     + v_cache.stride()[:3] + (page_table.stride(0),))
        found = _keep(form, (plan, make))
    (launch, plan, needs), make = found
    if out is None:
        out = make(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    if stream is None:
        stream = _current_stream(q.device)
    ws = workspace if workspace is not None else _current_workspace(needs, q.device, stream)
    rc = native.call(launch, plan, q, k_cache, v_cache, page_table, kv_len, cu_q, k_scale, v_scale,
                     out, lse, ws, 0 if ws is None else ws.numel() * ws.element_size(), stream)
    if rc:
        capi.check(rc)
    return (out, lse) if return_lse else out


def _attention_checks(q, k_cache, v_cache, page_table, kv_len, cu_q, k_scale, v_scale, out):
    import torch
    if q.dim() != 3:
        raise ValueError(f"q must be [T, Hq, D], got {tuple(q.shape)}")
    T, Hq, D = q.shape
    dtype = q.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"q: fp16 and bf16 are implemented, got {dtype}")
    _cache_checks(k_cache, v_cache, page_table, kv_len, cu_q, k_scale, v_scale, T,
                  k_cache.shape[2] if k_cache.dim() == 4 else 0, D, dtype)
    _same_device(q.device, k_cache=k_cache, v_cache=v_cache, page_table=page_table, kv_len=kv_len,
                 cu_q=cu_q, k_scale=k_scale, v_scale=v_scale, out=out)
    if out is not None and (out.shape != q.shape or out.dtype != dtype or out.stride(2) != 1):
        raise ValueError("out must be as q, with its last dimension contiguous")


# ---------------------------------------------------------------------------
# Pages
# ---------------------------------------------------------------------------

def _page_bytes(t, name, P):
    """(bytes from page to page, bytes of a page) of a cache tensor [P, ...] whose pages
    are each one block of memory."""
    if t.dim() < 2 or t.shape[0] != P:
        raise ValueError(f"{name} must be [{P}, ...] pages, got {tuple(t.shape)}")
    e, n = t.element_size(), 1
    for size, st in sorted(zip(t.shape[1:], t.stride()[1:]), key=lambda x: x[1]):
        if size != 1 and st != n:
            raise ValueError(f"{name}: a page must be one block of memory (strides {t.stride()})")
        n *= size
    return t.stride(0) * e, n * e


class _Pages:
    """The descriptor of calls on pages, and what workspace_for asks of a plan: their scratch
    memory.  The first 64 KiB of a workspace are the arrival counters of other launches."""

    def __init__(self, name, caches, P, device, S=0, W=0, n=0, page_size=1):
        if len(caches) > capi.PAGE_CACHES:
            raise ValueError(f"{len(caches)} caches: at most {capi.PAGE_CACHES} a call")
        d = self.desc = capi.PageDesc()
        d.S, d.W, d.P, d.n, d.page_size, d.caches = S, W, P, n, page_size, len(caches)
        for i, t in enumerate(caches):
            if t.device != device:
                raise ValueError(f"cache {i} is on {t.device}, not on {device}")
            d.stride[i], d.bytes[i] = _page_bytes(t, f"cache {i}", P)
        import torch
        self.new = torch.empty_like  # (of packed books)
        self.count = torch.empty((), dtype=torch.int32, device=device)  # what new counts are like
        self.launch, self.ref, need = capi.address(name), ctypes.addressof(d), ctypes.c_int64(0)
        capi.check(capi.load().tx_page_workspace(ctypes.byref(d), ctypes.byref(need)))
        self.workspace_bytes = _COUNTERS + need.value

    def scratch(self, device, stream):
        return _current_workspace(self, device, stream).data_ptr() + _COUNTERS


def _book_checks(page_table, kv_len, refs, out, **more):
    """Refuses books that do not go together; `more`: int32 vectors, `out` the books to write."""
    _is_int32(page_table, "page_table", 2)
    _is_int32(refs, "refs", 1)
    if kv_len is not None:
        _is_int32(kv_len, "kv_len", 1)
        if kv_len.shape[0] != page_table.shape[0]:
            raise ValueError(f"page_table has {page_table.shape[0]} rows, kv_len "
                             f"{kv_len.shape[0]}")
    for name, t in more.items():
        _is_int32(t, name, 1)
    _same_device(page_table.device, kv_len=kv_len, refs=refs, **more)
    if out is None:
        return
    like = tuple(t for t in (page_table, kv_len, refs) if t is not None)
    if len(out) != len(like):
        raise ValueError(f"out must be {len(like)} tensors")
    for t, u in zip(out, like):
        if t.shape != u.shape or t.dtype != u.dtype or t.device != u.device or not t.is_contiguous():
            raise ValueError(f"out must be contiguous and as the books read: {tuple(t.shape)} "
                             f"{t.dtype} for {tuple(u.shape)} {u.dtype}")


def page_copy(caches, src, dst, *, stream=None):
    """Copies page src[i] of every cache [P, ...] to page dst[i] (int32 [n]).  Entries
    outside [0, P) are skipped; no dst may be another dst, or a src but its own."""
    if stream is not None and stream != _current_stream(src.device):
        return _there(src.device, stream, page_copy, caches, src, dst)
    caches = list(caches)
    src, dst = _int32(src, "src", 1), _int32(dst, "dst", 1)
    if src.shape != dst.shape:
        raise ValueError("src and dst must be of one length")
    if not caches:
        return
    native = _native or _calls()
    form = native.form("copy", src, dst, caches)
    found = _forms.get(form)
    if found is None:
        _same_device(src.device, dst=dst)
        found = _keep(form, _Pages("tx_page_copy", caches, caches[0].shape[0], src.device, n=src.shape[0]))
    capi.check(native.call(found.launch, found.ref, native.addresses(caches), src, dst,
                           _current_stream(src.device) if stream is None else stream))


def page_reserve(page_table, kv_len, refs, new_len, page_size, *, out=None, stream=None):
    """Pages for sequences to grow to new_len [S] tokens (never less than kv_len, at most the
    table's width): free pages (refs 0) in ascending order, for one sequence after
    the other.  Returns page_table, kv_len, refs, and how many pages were missing (an
    int32 scalar on the device; those entries are -1).  out: the three tensors to write,
    which may be those read."""
    if stream is not None and stream != _current_stream(refs.device):
        return _there(refs.device, stream, page_reserve, page_table, kv_len, refs, new_len, page_size,
                      out=out)
    native = _native or _calls()
    page_size = index(page_size)
    form = native.form("reserve", page_table, kv_len, refs, new_len, page_size, out)
    found = _forms.get(form)
    if found is None:
        _book_checks(page_table, kv_len, refs, out, new_len=new_len)
        if new_len.shape != kv_len.shape:
            raise ValueError("new_len must be as kv_len")
        given = (page_table, kv_len, refs, new_len)
        dense = tuple(map(_dense, given))
        if any(a is not b for a, b in zip(dense, given)):
            return page_reserve(*dense, page_size, out=out, stream=stream)
        found = _keep(form, _Pages("tx_page_reserve", (), refs.shape[0], refs.device, *page_table.shape,
                                   page_size=page_size))
    t, n, r = tuple(map(found.new, (page_table, kv_len, refs))) if out is None else out
    device = refs.device
    missing = found.new(found.count)
    if stream is None:
        stream = _current_stream(device)
    rc = native.call(found.launch, found.ref, page_table, kv_len, refs, new_len, t, n, r, missing,
                     found.scratch(device, stream), stream)
    if rc:
        capi.check(rc)
    return t, n, r, missing


def page_fork(caches, page_table, kv_len, refs, parent, child, *, out=None, stream=None):
    """Sequences child[i] (empty rows, each named once) become copies of parent[i] that share
    its pages; a last page that is not full is copied, in every cache [P, page_size, ...],
    to a free one.  Returns page_table, kv_len, refs and the missing pages, as page_reserve."""
    if stream is not None and stream != _current_stream(refs.device):
        return _there(refs.device, stream, page_fork, caches, page_table, kv_len, refs, parent, child,
                      out=out)
    caches = list(caches)
    native = _native or _calls()
    form = native.form("fork", page_table, kv_len, refs, parent, child, out, caches)
    found = _forms.get(form)
    if found is None:
        _book_checks(page_table, kv_len, refs, out, parent=parent, child=child)
        if parent.shape != child.shape:
            raise ValueError("parent and child must be of one length")
        if not caches:
            raise ValueError("page_fork needs the caches: the size of a page is theirs")
        given = (page_table, kv_len, refs, parent, child)
        dense = tuple(map(_dense, given))
        if any(a is not b for a, b in zip(dense, given)):
            return page_fork(caches, *dense, out=out, stream=stream)
        pages = _Pages("tx_page_fork", caches, refs.shape[0], refs.device, *page_table.shape, parent.shape[0],
                       caches[0].shape[1])
        for i, c in enumerate(caches):
            if c.shape[1] != caches[0].shape[1]:
                raise ValueError(f"cache {i} has pages of {c.shape[1]} tokens, cache 0 of "
                                 f"{caches[0].shape[1]}")
        found = _keep(form, pages)
    t, n, r = tuple(map(found.new, (page_table, kv_len, refs))) if out is None else out
    device = refs.device
    missing = found.new(found.count)
    if stream is None:
        stream = _current_stream(device)
    rc = native.call(found.launch, found.ref, native.addresses(caches), page_table, kv_len, refs,
                     parent, child, t, n, r, missing, found.scratch(device, stream), stream)
    if rc:
        capi.check(rc)
    return t, n, r, missing


def page_free(page_table, kv_len, refs, drop, page_size, *, out=None, stream=None):
    """Sequences with drop[s] (bool [S]) give their pages back and become empty.  Returns
    page_table, kv_len, refs; out as for page_reserve."""
    if stream is not None and stream != _current_stream(refs.device):
        return _there(refs.device, stream, page_free, page_table, kv_len, refs, drop, page_size,
                      out=out)
    import torch
    native = _native or _calls()
    page_size = index(page_size)
    form = native.form("free", page_table, kv_len, refs, drop, page_size, out)
    found = _forms.get(form)
    if found is None:
        _book_checks(page_table, kv_len, refs, out)
        if drop.dtype not in (torch.bool, torch.uint8) or drop.shape != kv_len.shape:
            raise ValueError("drop must be a bool tensor as long as kv_len")
        _same_device(refs.device, drop=drop)
        given = (page_table, kv_len, refs, drop)
        dense = tuple(map(_dense, given))
        if any(a is not b for a, b in zip(dense, given)):
            return page_free(*dense, page_size, out=out, stream=stream)
        found = _keep(form, _Pages("tx_page_free", (), refs.shape[0], refs.device, *page_table.shape,
                                   page_size=page_size))
    t, n, r = tuple(map(found.new, (page_table, kv_len, refs))) if out is None else out
    rc = native.call(found.launch, found.ref, page_table, kv_len, refs, drop, t, n, r,
                     _current_stream(refs.device) if stream is None else stream)
    if rc:
        capi.check(rc)
    return t, n, r


def page_compact(caches, page_table, refs, *, out=None, stream=None):
    """Moves the pages in use (refs > 0) together: with U of them, those from U on go, in
    order, to the free ones below U, in every cache [P, ...] and in the books.  Returns
    page_table, refs and how many were moved (an int32 scalar on the device)."""
    if stream is not None and stream != _current_stream(refs.device):
        return _there(refs.device, stream, page_compact, caches, page_table, refs, out=out)
    caches = list(caches)
    native = _native or _calls()
    form = native.form("compact", page_table, refs, out, caches)
    found = _forms.get(form)
    if found is None:
        _book_checks(page_table, None, refs, out)
        dense = _dense(page_table), _dense(refs)
        if dense[0] is not page_table or dense[1] is not refs:
            return page_compact(caches, *dense, out=out, stream=stream)
        found = _keep(form, _Pages("tx_page_compact", caches, refs.shape[0], refs.device, *page_table.shape))
    t, r = tuple(map(found.new, (page_table, refs))) if out is None else out
    device = refs.device
    moved = found.new(found.count)
    if stream is None:
        stream = _current_stream(device)
    rc = native.call(found.launch, found.ref, native.addresses(caches), page_table, refs, t, r,
                     moved, found.scratch(device, stream), stream)
    if rc:
        capi.check(rc)
    return t, r, moved
