"""4-bit paged caches for the tests, and 64-bit oracles of what they hold (CPU tensors; the kernels
get copies).  Every value of a block is looked for among the fifteen that it may become."""
import math

import torch

from cachecase import E4M3, Cache, randn

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BLOCK = {"mx": 32, "nv": 16}
RANGE = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}


def scale_bytes(a, kind, dtype):
    """The scale bytes of blocks whose largest magnitudes are a (64 bits; NaN where not finite)."""
    if kind == "mx":
        lo, hi = RANGE[dtype]
        e = torch.full(a.shape, float(lo), dtype=torch.float64)
        for x in range(lo, hi):  # one up while 7 * 2^e is too small
            e = torch.where(a > 7.0 * 2.0 ** x, float(x + 1), e)
        return torch.where(a.isfinite(), e + 127, 255.0).to(torch.uint8)
    s = (a / 6).float().clamp(2.0 ** -9, 448.0).to(E4M3).view(torch.uint8)
    return torch.where(a.isfinite(), s, torch.tensor(0x7f, dtype=torch.uint8))


def scale_values(b, kind):
    if kind == "nv":
        return b.view(E4M3).to(torch.float64)
    return torch.where(b == 255, math.nan, torch.pow(2.0, b.double() - 127))


def nearest(m):
    """The code of |y| / scale: nearest, ties to the even code, saturated."""
    d = (m.clamp(max=6.0)[..., None] - LEVELS).abs()
    best = d.amin(-1, keepdim=True)
    tied = d == best
    odd = torch.arange(8) % 2 == 1
    return (tied & ~(odd & (tied.sum(-1, keepdim=True) > 1))).to(torch.int8).argmax(-1)


def quantise(y, kind, dtype):
    """Codes [..., D / 2] and scale bytes [..., D / block] of y [..., D] (64 bits)."""
    z = y.unflatten(-1, (-1, BLOCK[kind]))
    bad = ~z.isfinite().all(-1)
    a = torch.where(bad, math.nan, z.abs().amax(-1))
    b = scale_bytes(a, kind, dtype)
    unit = scale_values(b, kind)[..., None]
    z = torch.where(bad[..., None], 0.0, z)
    code = nearest(z.abs() / unit.nan_to_num(1.0)) + 8 * (torch.signbit(z) & ~bad[..., None])
    code = code.to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, b


def values(codes, b, kind):
    """What they stand for."""
    table = torch.cat((LEVELS, -LEVELS))
    x = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    return (x.unflatten(-1, (-1, BLOCK[kind])) * scale_values(b, kind)[..., None]).flatten(-2)


class Cache4(Cache):
    """As Cache, held in 4 bits: wherever no token lies, random codes under scales of NaN."""

    def __init__(self, seed, lens, page, Hkv, D, dtype, kind, layout="nhd", spare=3, width=0, holes=(),
                 scaled=False):
        super().__init__(seed, lens, page, Hkv, D, dtype, dtype, layout, spare, width, holes)
        self.kind, self.dtype, self.layout = kind, dtype, layout
        n, B = self.P, D // BLOCK[kind]
        self.k, self.v = (torch.randint(0, 256, (n, page, Hkv, D // 2), generator=self.g, dtype=torch.uint8)
                          for _ in range(2))
        self.kb, self.vb = (torch.full((n, page, Hkv, B), 255 if kind == "mx" else 0x7f, dtype=torch.uint8)
                            for _ in range(2))
        if scaled:  # a head's own factors (powers of two: quotients stay as they are)
            self.k_scale = 2.0 ** torch.randint(-3, 4, (Hkv,), generator=self.g).float()
            self.v_scale = 2.0 ** torch.randint(-3, 4, (Hkv,), generator=self.g).float()

    def put(self, which, b, j, codes, scales):
        at = self.place(b, j)
        if at is not None:
            (self.k if which == "k" else self.v)[at] = codes
            (self.kb if which == "k" else self.vb)[at] = scales

    def fill(self, amp=1.0):
        """N(0, amp) in the place of every token."""
        for t, s in ((self.k, self.kb), (self.v, self.vb)):
            for b, n in enumerate(self.lens):
                codes, scales = quantise(randn(self.g, max(n, 0), self.Hkv, self.D).double() * amp, self.kind,
                                         self.dtype)
                for e in range(-(-n // self.page)):
                    at = self.place(b, e * self.page)
                    if at is None:
                        continue
                    m = min(self.page, n - e * self.page)
                    t[at[0], :m] = codes[e * self.page:e * self.page + m]
                    s[at[0], :m] = scales[e * self.page:e * self.page + m]
        return self

    def rows(self, which, b):
        """All of sequence b's tokens in 64 bits, and which of them have a page."""
        t, s, scale = ((self.k, self.kb, self.k_scale) if which == "k"
                       else (self.v, self.vb, self.v_scale))
        n = max(self.lens[b], 0)
        x = torch.zeros(n, self.Hkv, self.D, dtype=torch.float64)
        ok = torch.zeros(n, dtype=torch.bool)
        for e in range(-(-n // self.page)):
            at = self.place(b, e * self.page)
            if at is not None:
                m = min(self.page, n - e * self.page)
                x[e * self.page:e * self.page + m] = values(t[at[0]], s[at[0]], self.kind)[:m]
                ok[e * self.page:e * self.page + m] = True
        return (x if scale is None else x * scale.double()[:, None]), ok

    def to(self, device):
        kind = torch.uint8 if self.kind == "mx" else E4M3

        def moved(t, order, back):
            if self.layout == "hnd":
                return t.permute(order).contiguous().to(device).permute(back)
            return t.to(device)
        codes = [moved(t, (0, 2, 1, 3), (0, 2, 1, 3)) for t in (self.k, self.v)]
        scales = [moved(t, (0, 2, 3, 1), (0, 3, 1, 2)).view(kind) for t in (self.kb, self.vb)]
        return dict(k_cache=codes[0], v_cache=codes[1], k_block_scale=scales[0],
                    v_block_scale=scales[1], page_table=self.table.to(device),
                    kv_len=self.kv_len.to(device),
                    k_scale=None if self.k_scale is None else self.k_scale.to(device),
                    v_scale=None if self.v_scale is None else self.v_scale.to(device))


# Appends whose tokens have more than 256 threads, the last workgroup of a token fewer than there are
# rotated pairs, with a head of q or k in it: n, lens, Hq, Hkv, D, rot, page, dtype, layout, interleaved.
MANY_THREADS = [
    ([1, 1, 1], [5, 70, 3000], 16, 2, 256, 256, 16, torch.bfloat16, "hnd", False),
    ([1, 1], [9, 33], 32, 2, 128, 128, 64, torch.float16, "nhd", False),
    ([2, 1], [40, 7], 32, 1, 128, 128, 16, torch.bfloat16, "hnd", False),
    ([1, 3], [6, 50], 16, 1, 128, 128, 16, torch.bfloat16, "hnd", True),
    ([600], [700], 64, 8, 256, 256, 16, torch.bfloat16, "hnd", False),  # fewer threads than heads
    ([990, 10], [990, 500], 31, 17, 256, 80, 16, torch.float16, "hnd", False),  # halves end inside a block
    ([990, 10], [990, 500], 31, 17, 256, 76, 16, torch.bfloat16, "nhd", False),
]
