"""Inputs and 64-bit oracles of the paged cache's tests (CPU tensors; the kernels get copies).

Tolerances count roundings: u(t) = finfo(t).eps / 2 is what one rounding to t is off by, and
F = 2^-24 that of fp32.
"""
import math

import torch

F = 2.0 ** -24
E4M3 = torch.float8_e4m3fn


def u(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype)


def rotate64(x, pos, inv_freq, interleaved, scale, inverse=False):
    """x [..., H, D] of positions pos [...]: result and what its error is measured by,
    the sum of the pair's magnitudes."""
    x = x.double()
    half = inv_freq.numel()
    a = pos.double()[..., None] * inv_freq.double()  # 64 bits: both factors have 24 bits or fewer
    c, s = (torch.cos(a) * scale)[..., None, :], (torch.sin(a) * scale)[..., None, :]
    if inverse:
        s = -s
    y, mag = x.clone(), torch.zeros_like(x)
    i, j = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved
            else (slice(0, half), slice(half, 2 * half)))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    mag[..., i] = mag[..., j] = (x[..., i].abs() + x[..., j].abs()) * abs(scale)
    return y, mag


def rotate_bound(y, mag, dtype):
    """One rounding of the result, and of fp32: the reduced angle (2^-25 of half a turn
    is under 4 F radians), sine or cosine (2 F), times scale, product and sum (1 F each)."""
    return u(dtype) * y.abs() + 9 * F * mag + 2.0 ** -24 * (dtype == torch.float16)


def check(got, ref, bound, what=""):
    got = got.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    inf = ~torch.isfinite(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: where the oracle is not finite"
    off = (got - ref).abs()[~inf] - bound.expand_as(ref)[~inf]
    assert not torch.isnan(off).any(), f"{what}: NaN"
    assert off.numel() == 0 or float(off.max()) <= 0, (
        f"{what}: {int((off > 0).sum())} of {off.numel()} values are off by up to "
        f"{float(off.max()):.3g} more than they may be")


class Cache:
    """A cache of sequences of these lengths on the CPU, poisoned with NaN wherever no token
    lies, its pages in random order."""

    def __init__(self, seed, lens, page, Hkv, D, dtype, cache, layout="nhd", spare=3, width=0,
                 holes=()):
        g = self.g = gen(seed)
        need = [-(-x // page) for x in lens]
        self.P = sum(need) + spare
        self.page, self.Hkv, self.D, self.lens, self.cache = page, Hkv, D, list(lens), cache
        order = torch.randperm(self.P, generator=g).to(torch.int32)
        self.W = width or max(need + [1])
        self.table = torch.full((len(lens), self.W), -1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            ids = order[at:at + k]
            self.table[b, :min(k, self.W)] = ids[:self.W]
            at += k
        for b, e, value in holes:
            self.table[b, e] = value
        shape = (self.P, Hkv, page, D) if layout == "hnd" else (self.P, page, Hkv, D)
        self.k, self.v = (self.empty(shape, cache, layout) for _ in range(2))
        self.k_scale = self.v_scale = None
        if cache == E4M3:
            self.k_scale = torch.rand(Hkv, generator=g) / 64 + 1 / 128
            self.v_scale = torch.rand(Hkv, generator=g) / 64 + 1 / 128
        self.kv_len = torch.tensor(lens, dtype=torch.int32)

    @staticmethod
    def empty(shape, cache, layout):
        t = torch.full(shape, math.nan).to(cache)
        return t.permute(0, 2, 1, 3) if layout == "hnd" else t

    def place(self, b, j):
        """(page, slot) of token j of sequence b, or None."""
        e = j // self.page
        if j < 0 or e >= self.W:
            return None
        p = int(self.table[b, e])
        return (p, j % self.page) if 0 <= p < self.P else None

    def fill(self, amp=1.0):
        """N(0, amp) in the place of every token."""
        for t in (self.k, self.v):
            for b, n in enumerate(self.lens):
                x = randn(self.g, n, self.Hkv, self.D) * amp
                if self.cache == E4M3:
                    x = (x * 64).clamp(-448, 448)
                x = x.to(self.cache)
                for e in range(-(-n // self.page)):
                    at = self.place(b, e * self.page)
                    if at is None:
                        continue
                    m = min(self.page, n - e * self.page)
                    t.view(t.dtype)[at[0], :m] = x[e * self.page:e * self.page + m]
        return self

    def rows(self, which, b):
        """All of sequence b's tokens in 64 bits, and which of them have a page."""
        t, scale = (self.k, self.k_scale) if which == "k" else (self.v, self.v_scale)
        n = max(self.lens[b], 0)
        x = torch.zeros(n, self.Hkv, self.D, dtype=torch.float64)
        ok = torch.zeros(n, dtype=torch.bool)
        for e in range(-(-n // self.page)):
            at = self.place(b, e * self.page)
            if at is not None:
                m = min(self.page, n - e * self.page)
                x[e * self.page:e * self.page + m] = t[at[0]].to(torch.float64)[:m]
                ok[e * self.page:e * self.page + m] = True
        return (x if scale is None else x * scale.double()[:, None]), ok

    def to(self, device):
        return dict(k_cache=_like(self.k, device), v_cache=_like(self.v, device),
                    page_table=self.table.to(device), kv_len=self.kv_len.to(device),
                    k_scale=None if self.k_scale is None else self.k_scale.to(device),
                    v_scale=None if self.v_scale is None else self.v_scale.to(device))


def _like(t, device):
    """A copy on `device` that keeps the order in memory."""
    if t.is_contiguous():
        return t.to(device)
    return t.permute(0, 2, 1, 3).contiguous().to(device).permute(0, 2, 1, 3)


def starts(n):
    return torch.tensor([0] + torch.tensor(n).cumsum(0).tolist(), dtype=torch.int32)


def attend64(q, c, n, causal, window, scale):
    """o, lse and their bounds for q [T, Hq, D] (rows past sum(n) attend to nothing)."""
    T, Hq, D = q.shape
    G = Hq // c.Hkv
    o = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    bo, bl = torch.zeros_like(o), torch.zeros_like(lse)
    un, at = u(q.dtype), 0
    for b, k in enumerate(n):
        K, ok = c.rows("k", b)
        V, _ = c.rows("v", b)
        L = K.shape[0]
        j = torch.arange(L)
        for h in range(c.Hkv if L and k else 0):
            x = q[at:at + k, h * G:(h + 1) * G].double()  # [k, G, D]
            s = (x.reshape(-1, D) @ K[:, h].T).view(k, G, L) * scale
            # a score: D + 2 roundings of fp32 of the sum of magnitudes
            es = (x.abs().reshape(-1, D) @ K[:, h].abs().T).view(k, G, L) * scale * (D + 2) * F
            pos = (c.lens[b] - k + torch.arange(k))[:, None]
            seen = ok.expand(k, L).clone()
            if causal:
                seen &= j <= pos
            if window:
                seen &= j > pos - window
            s = s.masked_fill(~seen[:, None, :], -math.inf)
            m = s.amax(-1, keepdim=True)
            some = torch.isfinite(m)
            p = torch.exp(s - m.masked_fill(~some, 0.0))
            total = p.sum(-1, keepdim=True)
            p = p / total.masked_fill(total == 0, 1.0)
            rows, hs = slice(at, at + k), slice(h * G, (h + 1) * G)
            o[rows, hs] = p @ V[:, h]
            es = es.masked_fill(~seen[:, None, :], 0.0).amax(-1, keepdim=True)
            # a weight: its score and the maximum's, the exponential (3 F of it, F of the exponent,
            # under 64 where it counts), the sums over keys, then one rounding to q's type
            e = 2 * es + (3 + 64 + 2 * math.log2(L + 1) + 16) * F
            A = p @ V[:, h].abs()
            bo[rows, hs] = (e + un) * A + (un + 4 * F) * o[rows, hs].abs() + 1e-30
            if q.dtype == torch.float16:  # weights and results below fp16's normal range
                bo[rows, hs] += 2.0 ** -25 * (1 + V[:, h].abs().sum(0))
            lse[rows, hs] = ((m + total.log()) / math.log(2.0))[..., 0]
            bl[rows, hs] = (e[..., 0] / math.log(2.0)) + 4 * F * lse[rows, hs].abs().nan_to_num(
                posinf=0.0)
        at += k
    return o, lse, bo, bl
