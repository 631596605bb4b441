"""A paged key/value cache, the attention that reads it, and rotary positions, as cases to time
and to compare.

Every case is one pass through one path:

  path   "rotary"   positions rotated into the heads of x, or (inverse) the gradient of that
         "append"   new tokens: q and k rotated, k and v written into the pages of their sequences
         "attend"   a chunk of new tokens of each sequence (one token: decode) over its pages
         "reserve"  pages for the tokens to come
         "fork"     sequences that share their parent's pages, the last one copied
         "compact"  sequences freed, and the pages that are left moved together

Sizes are those of this repository's benchmark and tests where it has them: heads of 64 and 128
(32 of them, 4096 tokens, batch 4), batches of 1 .. 64 rows for decode, prompts of 1000 .. 4096
tokens; page sizes and group sizes are generic.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-ext_amd")
_DEV = "cuda:0"
_TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
          "e4m3": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


def _tx():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import triton_ext_amd
    return triton_ext_amd


def _rotary(N, H, D, rot, dtype, interleaved, inverse, layout="nhd", Z=1, scaling="", start=0):
    return {"path": "rotary", "Z": Z, "N": N, "H": H, "D": D, "rot": rot, "dtype": dtype,
            "interleaved": interleaved, "inverse": inverse, "layout": layout, "scaling": scaling,
            "start": start}


def _append(B, tokens, context, Hq, Hkv, D, rot, page, dtype, cache, interleaved=False,
            scaling="", layout="nhd"):
    """`tokens` new tokens in all over B sequences, that hold up to `context` tokens already."""
    return {"path": "append", "B": B, "tokens": tokens, "context": context, "Hq": Hq, "Hkv": Hkv,
            "D": D, "rot": rot, "page": page, "dtype": dtype, "cache": cache,
            "interleaved": interleaved, "scaling": scaling, "layout": layout}


def _attend(B, q_lo, q_hi, kv_lo, kv_hi, Hq, Hkv, D, page, dtype, cache, window=0, causal=True,
            layout="nhd", lse=False):
    """B sequences of q_lo .. q_hi new tokens and kv_lo .. kv_hi tokens in all."""
    return {"path": "attend", "B": B, "q_lo": q_lo, "q_hi": q_hi, "kv_lo": kv_lo, "kv_hi": kv_hi,
            "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "cache": cache,
            "window": window, "causal": causal, "layout": layout, "lse": lse}


def _pages(path, S, W, P, page, Hkv=8, D=128, caches=0, children=0, dtype="bf16"):
    return {"path": path, "S": S, "W": W, "P": P, "page": page, "Hkv": Hkv, "D": D,
            "caches": caches, "children": children, "dtype": dtype}


def listed():
    return [
        # q and k heads of 16 sequences in one decode step: latency counts
        {"name": "rotary_step16", **_rotary(16, 40, 128, 128, "bf16", False, False, start=5000)},
        # the gradient of q in a training step, at the attention benchmark's shape, a partly
        # rotated head in interleaved pairs
        {"name": "rotary_grad_4096", **_rotary(4096, 32, 64, 32, "fp16", True, True, "zhnd", 4)},
        # the new tokens of a decode step of 48 sequences go into the cache
        {"name": "append_step48", **_append(48, 48, 8000, 32, 8, 128, 128, 16, "bf16", "bf16")},
        # prompts of some thousand tokens, positions scaled for a long context, an 8-bit cache
        {"name": "append_prompts_e4m3", **_append(7, 9001, 30000, 32, 8, 128, 128, 64, "bf16",
                                                  "e4m3", scaling="yarn")},
        # one user, a short conversation: the smallest attention call
        {"name": "attend_one_1500", **_attend(1, 1, 1, 1500, 1500, 16, 4, 64, 16, "bf16", "bf16")},
        # a serving batch: 32 sequences of very different lengths, one token each
        {"name": "attend_batch32", **_attend(32, 1, 1, 100, 16384, 32, 8, 128, 16, "bf16", "bf16")},
        # a few very long contexts in an 8-bit cache, several drafted tokens to verify
        {"name": "attend_long_e4m3", **_attend(4, 4, 4, 60000, 131072, 32, 8, 128, 64, "fp16",
                                               "e4m3")},
        # long prompts taken in chunks of 2048
        {"name": "attend_chunk2048", **_attend(2, 2048, 2048, 8192, 16384, 32, 8, 128, 64, "bf16",
                                               "bf16")},
        # decode and prompt chunks in one batch, a sliding window, a head of k and v per head of q
        {"name": "attend_mixed_window", **_attend(24, 1, 300, 300, 8000, 16, 16, 64, 16, "fp16",
                                                  "fp16", window=1024, layout="hnd", lse=True)},
        # the bookkeeping before each decode step
        {"name": "reserve_step256", **_pages("reserve", 256, 512, 65536, 16)},
        # beams: each of 8 sequences forks into 8, a model of 4 layers
        {"name": "fork_beams64", **_pages("fork", 96, 64, 1024, 64, caches=8, children=56)},
        # half of the sequences end; the cache is made dense again
        {"name": "compact_half", **_pages("compact", 64, 256, 4096, 16, caches=4)},
    ]


# ---------------------------------------------------------------------------
# More cases of the same ranges
# ---------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    Hkv = rng.choice([1, 2, 4, 8, 8, 5, 16])
    G = rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    return (Hkv * G, Hkv) if Hkv * G <= 64 else (Hkv, Hkv)


def draw(rng):
    while True:
        path = rng.choice(["rotary", "rotary", "append", "append", "attend", "attend", "attend",
                           "attend", "reserve", "fork", "compact"])
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        page = rng.choice([8, 16, 16, 32, 64, 128])
        layout = rng.choice(["nhd", "nhd", "hnd"])
        D = rng.choice([64, 64, 128, 128, 96, 80, 256])
        if path == "rotary":
            rot = rng.choice([D, D, D // 2, 32])
            zhnd = rng.random() < 0.5
            c = _rotary(_log(rng, 1, 8192), rng.choice([1, 8, 12, 32, 40]), D, rot,
                        rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5,
                        rng.random() < 0.4, "zhnd" if zhnd else "nhd",
                        rng.choice([1, 2, 4]) if zhnd else 1,
                        rng.choice(["", "linear", "ntk", "yarn"]), rng.choice([0, 0, 100000]))
            if c["Z"] * c["N"] * c["H"] * D <= 4 * 4096 * 32 * 64:
                return c
        elif path == "append":
            Hq, Hkv = _heads(rng)
            B = _log(rng, 1, 64)
            c = _append(B, max(B, _log(rng, 1, 9000)), _log(rng, 1, 30000), Hq, Hkv, D,
                        rng.choice([D, D // 2]), page, dtype, rng.choice([dtype, dtype, "e4m3"]),
                        rng.random() < 0.4, rng.choice(["", "linear", "yarn"]), layout)
            if c["tokens"] * Hq * D <= 9001 * 32 * 128 and B * c["context"] * Hkv * D <= 1 << 29:
                return c
        elif path == "attend":
            Hq, Hkv = _heads(rng)
            cache = rng.choice([dtype, dtype, "e4m3"])
            kind = rng.choice(["decode", "decode", "few", "chunk"])
            if kind == "chunk":
                B, q_hi = rng.choice([1, 1, 2, 3]), _log(rng, 64, 2048)
            else:
                B, q_hi = _log(rng, 1, 48), 1 if kind == "decode" else _log(rng, 2, 16)
            q_lo = rng.choice([q_hi, max(1, q_hi // 3)])
            kv_hi = max(q_hi, _log(rng, 16, 16384 if kind == "chunk" else 131072))
            kv_lo = rng.choice([q_hi, kv_hi, max(q_hi, kv_hi // 2)])
            c = _attend(B, q_lo, q_hi, kv_lo, kv_hi, Hq, Hkv, D, page, dtype, cache,
                        rng.choice([0, 0, 0, 100, 4096]), rng.random() < 0.85, layout,
                        rng.random() < 0.3)
            if (B * q_hi * Hq * kv_hi * D <= 2 * 2048 * 32 * 16384 * 128
                    and B * kv_hi * Hkv * D <= 32 * 16384 * 8 * 128):
                return c
        elif path == "reserve":
            S = _log(rng, 1, 256)
            W = _log(rng, 4, 512)
            return _pages("reserve", S, W, max(64, S * W // 2), page)
        else:
            S, Hkv = _log(rng, 2, 64), rng.choice([1, 2, 4, 8])
            W = _log(rng, 4, 64)
            n = rng.choice([1, 2, 5, 8])
            c = _pages(path, 2 * S if path == "fork" else S, W, S * W + 37, page, Hkv, D, n,
                       rng.randint(1, S) if path == "fork" else 0, dtype)
            if c["P"] * page * Hkv * D * n <= 4096 * 16 * 8 * 128 * 4:
                return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _gens(seed):
    """For values on the GPU, and for the order of pages."""
    d, h = torch.Generator(device=_DEV), torch.Generator()
    d.manual_seed(int(seed))
    h.manual_seed(int(seed) + 1)
    return d, h


def _sizes(c):
    """The new tokens and the lengths of a case's sequences: its own, whatever the seed."""
    h = torch.Generator()
    h.manual_seed(7)
    if c["path"] == "append":
        n = _parts(h, c["B"], c["tokens"])
        return n, [x + y for x, y in zip(n, _spread(h, c["B"], 0, c["context"]))]
    n = _spread(h, c["B"], c["q_lo"], c["q_hi"])
    return n, [max(x, y) for x, y in zip(n, _spread(h, c["B"], c["kv_lo"], c["kv_hi"]))]


def _held(c):
    """The same of the sequences whose pages are kept in order."""
    h = torch.Generator()
    h.manual_seed(7)
    S, W, P, page = c["S"], c["W"], c["P"], c["page"]
    if c["path"] == "reserve":  # a third of the pool is held
        return _spread(h, S, 1, max(1, min(W * page - 1, P * page // (3 * S))))
    if c["path"] == "fork":  # sequences in the first slots, their children in free ones after them
        live = S - c["children"]
        most = max(1, min(W, (P - c["children"]) // max(live, 1)) * page - 1)
        return _spread(h, live, 1, most) + [0] * c["children"]
    return _spread(h, S, max(1, min(W, P // S) * page // 2), max(1, min(W, P // S) * page))


def _randn(g, *shape, dtype=torch.float32):
    out = torch.empty(shape, dtype=dtype, device=_DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):  # the 32-bit draws of a large cache, in pieces
        piece = flat[i:i + (1 << 28)]
        piece.copy_(torch.randn(piece.shape, generator=g, device=_DEV))
    return out


def _spread(h, count, lo, hi):
    """`count` lengths of lo .. hi, spread over their logarithm, hi among them."""
    if lo == hi:
        return [hi] * count
    u = torch.rand(count, generator=h).tolist()
    got = [int(round(math.exp(math.log(max(lo, 1)) + x * (math.log(hi) - math.log(max(lo, 1)))))) for x in u]
    got[count // 2] = hi
    return got


def _parts(h, count, total):
    """`total` tokens over `count` sequences, one each at least, in unequal parts."""
    w = torch.rand(count, generator=h) + 0.05
    n = [1 + int(x) for x in (w / w.sum() * (total - count)).floor().tolist()]
    n[0] += total - sum(n)
    return n


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _starts(n):
    got = [0]
    for x in n:
        got.append(got[-1] + x)
    return got


def _tables(h, lens, page, spare=1.1, width=0):
    """A page table for sequences of these lengths, their pages scattered over the pool."""
    need = [-(-x // page) for x in lens]
    P = int(sum(need) * spare) + 3
    order = torch.randperm(P, generator=h).to(torch.int32)
    W = max(width, max(need), 1)
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, P


def _cache(g, P, page, Hkv, D, kind, layout):
    """[P, page, Hkv, D], in the order of `layout` in memory ("hnd": a head's tokens together)."""
    shape = (P, Hkv, page, D) if layout == "hnd" else (P, page, Hkv, D)
    if kind == "e4m3":  # N(0, 1) at the scale below
        c = torch.empty(shape, dtype=torch.float8_e4m3fn, device=_DEV)
        step = max(1, (1 << 27) // (page * Hkv * D))
        for i in range(0, P, step):
            c[i:i + step] = (torch.randn((min(step, P - i),) + shape[1:], generator=g, device=_DEV)
                             * 64.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        c = _randn(g, *shape, dtype=_TORCH[kind])
    return c.permute(0, 2, 1, 3) if layout == "hnd" else c


def _frequencies(rot, scaling):
    """base^(-2 i / rot) in fp32, scaled for long contexts, and the factor on cos and sin."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    base, factor, context = 10000.0, 8.0, 4096.0
    if scaling == "ntk":
        base *= factor ** (rot / max(rot - 2, 1))
    f = base ** (-2.0 * i / rot)
    scale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        turns = context * f / (2 * math.pi)  # of one frequency over the trained context
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f / factor * (1 - keep) + f * keep
        scale = 0.1 * math.log(factor) + 1.0
    return f.to(torch.float32).to(_DEV), scale


def prepare(case, seed):
    c = dict(case)
    g, h = _gens(seed)
    path = c["path"]
    s = {"path": path, "case": c}
    if path == "rotary":
        dt = _TORCH[c["dtype"]]
        s["inv_freq"], s["scale"] = _frequencies(c["rot"], c["scaling"])
        if c["layout"] == "zhnd":
            s["x"] = _randn(g, c["Z"], c["H"], c["N"], c["D"], dtype=dt)
            s["positions"] = torch.arange(c["start"], c["start"] + c["N"], dtype=torch.int32,
                                          device=_DEV)
        else:  # the q and k heads of a fused projection, whose v heads follow
            s["x"] = _randn(g, c["N"], c["H"] + 8, c["D"], dtype=dt)[:, :c["H"]]
            s["positions"] = torch.randint(c["start"], c["start"] + 8192, (c["N"],),
                                           generator=h).to(torch.int32).to(_DEV)
        return s
    if path in ("append", "attend"):
        B, page, Hq, Hkv, D = (c[k] for k in ("B", "page", "Hq", "Hkv", "D"))
        dt = _TORCH[c["dtype"]]
        n, lens = _sizes(c)
        T = sum(n)
        table, P = _tables(h, lens, page)
        s.update(n=n, lens=lens, page_table=table.to(_DEV), kv_len=_int(lens),
                 cu_q=_int(_starts(n)) if max(n) > 1 or min(n) < 1 else None)
        s["k_cache"] = _cache(g, P, page, Hkv, D, c["cache"], c["layout"])
        s["v_cache"] = _cache(g, P, page, Hkv, D, c["cache"], c["layout"])
        s["k_scale"] = s["v_scale"] = None
        if c["cache"] == "e4m3":
            s["k_scale"] = (torch.rand(Hkv, generator=g, device=_DEV) + 0.5) / 64.0
            s["v_scale"] = (torch.rand(Hkv, generator=g, device=_DEV) + 0.5) / 64.0
        qkv = _randn(g, T, Hq + 2 * Hkv, D, dtype=dt)  # as a fused projection leaves them
        if path == "append":
            s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
            s["inv_freq"], s["scale"] = _frequencies(c["rot"], c["scaling"])
        else:
            s["q"] = qkv[:, :Hq].contiguous()  # as the rotation leaves it
        return s
    S, W, P, page = c["S"], c["W"], c["P"], c["page"]
    lens = _held(c)
    need = [-(-x // page) for x in lens]
    order = torch.randperm(P, generator=h).to(torch.int32)
    table, refs, at = torch.full((S, W), -1, dtype=torch.int32), torch.zeros(P, dtype=torch.int32), 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        refs[order[at:at + k].long()] = 1
        at += k
    s.update(page_table=table.to(_DEV), kv_len=_int(lens), refs=refs.to(_DEV))
    s["caches"] = [_randn(g, P, page, c["Hkv"], c["D"], dtype=_TORCH[c["dtype"]])
                   for _ in range(c["caches"])]
    if path == "reserve":
        s["new_len"] = _int([min(x + 1, W * page) for x in lens])  # one token more each
    elif path == "fork":
        k = c["children"]
        s["parent"] = torch.randint(0, S - k, (k,), generator=h).to(torch.int32).to(_DEV)
        s["child"] = (S - k + torch.randperm(k, generator=h)).to(torch.int32).to(_DEV)
    else:
        s["drop"] = (torch.arange(S) % 2 == 0).to(_DEV)
    return s


# ---------------------------------------------------------------------------
# The paths, in elementary operations
# ---------------------------------------------------------------------------

def _rotate(x, positions, inv_freq, interleaved, scale, inverse):
    """x [..., D] in fp32 with angles [..., rot / 2] = position * inv_freq broadcast over it."""
    a = positions.double()[..., None] * inv_freq.double()
    cos, sin = (torch.cos(a) * scale).float(), (torch.sin(a) * scale).float()
    if inverse:
        sin = -sin
    rot = 2 * inv_freq.numel()
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        x1, x2 = r[..., 0::2], r[..., 1::2]
        y = torch.stack((x1 * cos - x2 * sin, x2 * cos + x1 * sin), dim=-1).flatten(-2)
    else:
        x1, x2 = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), dim=-1)
    return torch.cat((y, rest), dim=-1)


def _places(s):
    """Of every new token: its sequence, its place among that one's new tokens, its position."""
    B, T = len(s["n"]), s["q"].shape[0]
    if s["cu_q"] is None:
        seq = torch.arange(B, device=_DEV)
        return seq, torch.zeros_like(seq), s["kv_len"].long() - 1
    cu = s["cu_q"].long()
    seq = torch.repeat_interleave(torch.arange(B, device=_DEV), cu.diff(), output_size=T)
    off = torch.arange(T, device=_DEV) - cu[seq]
    return seq, off, s["kv_len"].long()[seq] - cu.diff()[seq] + off


def _plain_rotary(s):
    c, x = s["case"], s["x"].float()
    p = s["positions"] if c["layout"] == "zhnd" else s["positions"][:, None]
    return _rotate(x, p, s["inv_freq"], c["interleaved"], s["scale"], c["inverse"]).to(s["x"].dtype)


def _plain_append(s):
    c = s["case"]
    seq, _, pos = _places(s)
    page = s["page_table"][seq, pos // c["page"]].long()
    slot = pos % c["page"]
    q, k = (_rotate(s[t].float(), pos[:, None], s["inv_freq"], c["interleaved"], s["scale"], False)
            for t in ("q", "k"))
    v = s["v"].float()
    for new, cache, scale in ((k, s["k_cache"], s["k_scale"]), (v, s["v_cache"], s["v_scale"])):
        if scale is not None:
            new = (new / scale[:, None]).clamp(-448.0, 448.0)
            cache.view(torch.uint8)[page, slot] = new.to(cache.dtype).view(torch.uint8)
        else:
            cache[page, slot] = new.to(cache.dtype)
    return {"q": q.to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    c = s["case"]
    B, Hq, Hkv, D, page = (c[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    G, Q, W = Hq // Hkv, max(s["n"]), s["page_table"].shape[1]
    seq, off, pos = _places(s)
    pages = s["page_table"].long().clamp_min(0)
    L = W * page

    def keys(cache, scale):  # [B, Hkv, L, D]
        x = (cache.view(torch.uint8)[pages].view(cache.dtype) if scale is not None
             else cache[pages]).float().reshape(B, L, Hkv, D)
        if scale is not None:
            x = x * scale[:, None]
        held = torch.arange(L, device=_DEV) < s["kv_len"][:, None]
        return x.masked_fill(~held[:, :, None, None], 0.0).transpose(1, 2).contiguous()

    q = torch.zeros((B, Q, Hq, D), device=_DEV)
    q[seq, off] = s["q"].float()
    q = q.view(B, Q, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Q * G, D)
    scores = torch.matmul(q, keys(s["k_cache"], s["k_scale"]).transpose(2, 3)) * D ** -0.5
    n = (s["cu_q"].diff() if s["cu_q"] is not None else torch.ones_like(s["kv_len"]))
    at = (s["kv_len"] - n)[:, None] + torch.arange(Q, device=_DEV)  # positions [B, Q]
    j = torch.arange(L, device=_DEV)
    seen = (j < s["kv_len"][:, None])[:, None, :]
    if c["causal"]:
        seen = seen & (j <= at[:, :, None])
    if c["window"]:
        seen = seen & (j > at[:, :, None] - c["window"])
    seen = seen.expand(B, Q, L)[:, None, :, None, :].expand(B, 1, Q, G, L).reshape(B, 1, Q * G, L)
    scores.masked_fill_(~seen, -math.inf)
    m = scores.amax(dim=-1, keepdim=True)
    p = scores.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, keys(s["v_cache"], s["v_scale"])) / total.masked_fill(total == 0, 1.0)
    back = lambda t: t.view(B, Hkv, Q, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Q, Hq, -1)[seq, off]  # noqa: E731
    out = back(o).to(s["q"].dtype)
    if not c["lse"]:
        return out
    return {"o": out, "lse": back((m + total.log()) / math.log(2.0))[..., 0].contiguous()}


def _take(refs, wanted):
    """For every true place of `wanted`, in order, the next free page in order (-1: none left),
    and how many free pages there were too few."""
    P = refs.numel()
    free = refs == 0
    rank = torch.where(free, free.cumsum(0) - 1, P)
    pages = torch.full((P + 1,), -1, dtype=torch.int64, device=refs.device)
    pages.scatter_(0, rank, torch.arange(P, device=refs.device))
    pages[P] = -1
    turn = (wanted.flatten().cumsum(0) - 1).clamp(0, P).view(wanted.shape)
    pages.masked_fill_(torch.arange(P + 1, device=refs.device) >= free.sum(), -1)
    got = torch.where(wanted, pages[turn], -1)
    return got, (wanted.sum() - free.sum()).clamp_min(0).to(torch.int32)


def _plain_reserve(s):
    page, table, refs = s["case"]["page"], s["page_table"], s["refs"]
    S, W = table.shape
    w = torch.arange(W, device=_DEV)
    length = torch.maximum(s["kv_len"], s["new_len"].clamp_max(W * page))
    wanted = ((w >= ((s["kv_len"] + page - 1) // page)[:, None])
              & (w < ((length + page - 1) // page)[:, None]))
    got, missing = _take(refs, wanted)
    refs = torch.cat((refs, refs.new_zeros(1)))
    refs = refs.index_add(0, torch.where(got >= 0, got, refs.numel() - 1).flatten(),
                          (got >= 0).to(torch.int32).flatten())[:-1]
    return {"page_table": torch.where(wanted, got.to(torch.int32), table), "kv_len": length,
            "refs": refs, "missing": missing}


def _plain_fork(s):
    page, table, refs = s["case"]["page"], s["page_table"], s["refs"]
    parent, child = s["parent"].long(), s["child"].long()
    length = s["kv_len"][parent]
    used = (length + page - 1) // page
    w = torch.arange(table.shape[1], device=_DEV)
    rows = torch.where(w < used[:, None], table[parent], -1)
    open_ = length % page != 0
    got, missing = _take(refs, open_)
    last = (used - 1).clamp_min(0).long()[:, None]
    old = rows.gather(1, last)[:, 0].long()
    new = torch.where(open_, got, old)
    rows = rows.scatter(1, last, new.to(torch.int32)[:, None])
    refs = refs.index_add(0, rows.clamp_min(0).long().flatten(), (rows >= 0).to(torch.int32).flatten())
    for cache in s["caches"]:  # a page kept is copied onto itself
        cache[new] = cache[old]
    return {"page_table": table.index_copy(0, child, rows),
            "kv_len": s["kv_len"].index_copy(0, child, length), "refs": refs, "missing": missing,
            "caches": s["caches"]}


def _plain_compact(s):
    page, table, refs = s["case"]["page"], s["page_table"], s["refs"]
    drop = s["drop"]
    used = (s["kv_len"] + page - 1) // page
    w = torch.arange(table.shape[1], device=_DEV)
    gone = drop[:, None] & (w < used[:, None]) & (table >= 0)
    refs = refs.index_add(0, table.clamp_min(0).long().flatten(), -gone.to(torch.int32).flatten())
    table = table.masked_fill(drop[:, None], -1)
    length = s["kv_len"].masked_fill(drop, 0)
    P = refs.numel()
    page_id = torch.arange(P, device=_DEV)
    live = refs > 0
    count = live.sum()
    source = (live & (page_id >= count)).nonzero()[:, 0]
    target = (~live & (page_id < count)).nonzero()[:, 0]
    moved = page_id.index_copy(0, source, target)
    table = torch.where(table >= 0, moved[table.clamp_min(0).long()].to(torch.int32), table)
    refs = refs.index_copy(0, target, refs[source]).index_fill(0, source, 0)
    for cache in s["caches"]:
        cache[target] = cache[source]
    return {"page_table": table, "kv_len": length, "refs": refs,
            "moved": (live & (page_id >= count)).sum().to(torch.int32), "caches": s["caches"]}


_PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend,
          "reserve": _plain_reserve, "fork": _plain_fork, "compact": _plain_compact}


# ---------------------------------------------------------------------------
# The same by this package
# ---------------------------------------------------------------------------

def _own_rotary(tx, s, c):
    return tx.rotary(s["x"], s["positions"], s["inv_freq"], interleaved=c["interleaved"],
                     scale=s["scale"], inverse=c["inverse"])


def _own_append(tx, s, c):
    q = tx.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_len"],
                        s["cu_q"], q=s["q"], inv_freq=s["inv_freq"],
                        interleaved=c["interleaved"], scale=s["scale"], k_scale=s["k_scale"],
                        v_scale=s["v_scale"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attend(tx, s, c):
    r = tx.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_len"],
                           s["cu_q"], sm_scale=c["D"] ** -0.5, causal=c["causal"],
                           window=c["window"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                           return_lse=c["lse"])
    return {"o": r[0], "lse": r[1]} if c["lse"] else r


def _own_reserve(tx, s, c):
    table, length, refs, missing = tx.page_reserve(s["page_table"], s["kv_len"], s["refs"],
                                                   s["new_len"], c["page"])
    return {"page_table": table, "kv_len": length, "refs": refs, "missing": missing}


def _own_fork(tx, s, c):
    table, length, refs, missing = tx.page_fork(s["caches"], s["page_table"], s["kv_len"],
                                                s["refs"], s["parent"], s["child"])
    return {"page_table": table, "kv_len": length, "refs": refs, "missing": missing,
            "caches": s["caches"]}


def _own_compact(tx, s, c):
    table, length, refs = tx.page_free(s["page_table"], s["kv_len"], s["refs"], s["drop"],
                                       c["page"])
    table, refs, moved = tx.page_compact(s["caches"], table, refs)
    return {"page_table": table, "kv_len": length, "refs": refs, "moved": moved,
            "caches": s["caches"]}


_OWN = {"rotary": _own_rotary, "append": _own_append, "attend": _own_attend,
        "reserve": _own_reserve, "fork": _own_fork, "compact": _own_compact}


def run(state):
    if own:
        return _OWN[state["path"]](_tx(), state, state["case"])
    return _PLAIN[state["path"]](state)


# ---------------------------------------------------------------------------
# Work, and the results in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    c, path = case, case["path"]
    if path == "rotary":
        n = c["Z"] * c["N"] * c["H"]
        return {"bytes": 2 * n * c["D"] * _SIZE[c["dtype"]] + 4 * c["N"], "flops": 3 * n * c["rot"]}
    if path == "append":
        e, T = _SIZE[c["dtype"]], c["tokens"]
        return {"bytes": T * c["D"] * (2 * c["Hq"] * e + 2 * c["Hkv"] * (e + _SIZE[c["cache"]])),
                "flops": 3 * T * (c["Hq"] + c["Hkv"]) * c["rot"]}
    if path == "attend":
        pairs = span = T = 0
        for n, length in zip(*_sizes(c)):
            first = length - n  # the first new token's position
            T += n
            span += min(length, c["window"] + n - 1) if c["window"] else length
            for p in range(first, length):
                to = p + 1 if c["causal"] else length
                pairs += to - max(0, p - c["window"] + 1) if c["window"] else to
        return {"bytes": 2 * T * c["Hq"] * c["D"] * _SIZE[c["dtype"]]
                + 2 * span * c["Hkv"] * c["D"] * _SIZE[c["cache"]],
                "flops": 4 * pairs * c["Hq"] * c["D"]}
    books = 8 * (c["S"] * c["W"] + c["S"] + c["P"])
    one = c["page"] * c["Hkv"] * c["D"] * _SIZE[c["dtype"]] * c["caches"]
    held = [-(-x // c["page"]) for x in _held(c)]
    if path == "compact":  # of the pages that are left, those that lie past the hole they fill
        left = sum(held[1::2])
        return {"bytes": books + 2 * one * left * (1 - left / c["P"]), "flops": 0}
    return {"bytes": books + 2 * one * c["children"], "flops": 0}


def _exact_angles(positions, inv_freq, scale):
    a = torch.outer(positions.double().flatten(), inv_freq.double())
    return torch.complex(torch.cos(a), torch.sin(a)) * scale


def _exact_turn(x, turns, interleaved):
    """The pairs of x [N, H, D] as complex numbers, times turns [N, rot / 2]."""
    x = x.double()
    half = turns.shape[1]
    y = x.clone()
    first, second = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved
                     else (slice(0, half), slice(half, 2 * half)))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turns[:, None, :]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rotary(c, s):
    turns = _exact_angles(s["positions"], s["inv_freq"], s["scale"])
    if c["inverse"]:
        turns = turns.conj()
    if c["layout"] != "zhnd":
        return _exact_turn(s["x"], turns, c["interleaved"])
    return torch.stack([_exact_turn(x.transpose(0, 1), turns, c["interleaved"]).transpose(0, 1)
                        for x in s["x"]])


def _exact_append(c, s):
    first = _starts(s["n"])
    q = torch.empty(s["q"].shape, dtype=torch.float64, device=_DEV)
    caches = {t: s[t].to(torch.float64) for t in ("k_cache", "v_cache")}
    for b, (n, length) in enumerate(zip(s["n"], s["lens"])):
        rows = slice(first[b], first[b] + n)
        at = torch.arange(length - n, length, device=_DEV)
        turns = _exact_angles(at, s["inv_freq"], s["scale"])
        q[rows] = _exact_turn(s["q"][rows], turns, c["interleaved"])
        new = {"k_cache": _exact_turn(s["k"][rows], turns, c["interleaved"]),
               "v_cache": s["v"][rows].double()}
        page = s["page_table"][b][torch.div(at, c["page"], rounding_mode="floor")].long()
        for t, x in new.items():
            if s["k_scale"] is not None:
                x = (x / s[t[0] + "_scale"].double()[:, None]).clamp(-448.0, 448.0)
            caches[t][page, at % c["page"]] = x
    return {"q": q, **caches}


def _exact_attend(c, s):
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]
    G, first = Hq // Hkv, _starts(s["n"])
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=_DEV)
    for b, (n, length) in enumerate(zip(s["n"], s["lens"])):
        ids = s["page_table"][b, :-(-length // page)].long()
        j = torch.arange(length, device=_DEV)
        for h in range(Hkv):
            def side(name, scale):
                one = s[name][:, :, h]  # [P, page, D]
                x = (one.view(torch.uint8)[ids].view(one.dtype) if scale is not None else one[ids])
                x = x.reshape(-1, D)[:length].double()
                return x if scale is None else x * scale[h].double()
            K, V = side("k_cache", s["k_scale"]), side("v_cache", s["v_scale"])
            step = max(1, (1 << 27) // max(1, length * G))
            for i in range(0, n, step):
                t = torch.arange(i, min(n, i + step), device=_DEV)
                rows = first[b] + t
                x = s["q"][rows][:, h * G:(h + 1) * G].double().reshape(-1, D)
                z = x @ K.T.contiguous() / math.sqrt(D)
                pos = (length - n + t).repeat_interleave(G)[:, None]
                bad = torch.zeros(z.shape, dtype=torch.bool, device=_DEV)
                if c["causal"]:
                    bad |= j > pos
                if c["window"]:
                    bad |= j <= pos - c["window"]
                z[bad] = -math.inf
                e = torch.logsumexp(z, dim=1)
                w = torch.exp(z - e.masked_fill(e == -math.inf, 0.0)[:, None])
                o[rows, h * G:(h + 1) * G] = (w @ V).view(-1, G, D)
                lse[rows, h * G:(h + 1) * G] = (e / math.log(2.0)).view(-1, G)
    return {"o": o, "lse": lse} if c["lse"] else o


def exact(case, seed):
    c = dict(case)
    if c["path"] not in ("rotary", "append", "attend"):
        return None  # pages are moved and counted, not computed
    return {"rotary": _exact_rotary, "append": _exact_append,
            "attend": _exact_attend}[c["path"]](c, prepare(c, seed))
