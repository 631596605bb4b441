"""A paged key/value cache held in 4 bits, as cases to time and to compare: tokens quantised as they
are written, read back, and the attention over what the cache holds.

Every case is one pass through one path:

  path   "append"   new tokens: q and k rotated, k and v quantised into the pages of their sequences,
                    and read back as the values that the cache now holds of them
         "read"     whole sequences out of the cache, as dense tensors
         "attend"   a chunk of new tokens of each sequence (one token: decode) over its pages

The cache holds e2m1 codes, two a byte (the even dim in the low four bits), and scales: "mx", one
e8m0 byte of 32 dims (2^(byte - 127)), or "nv", one e4m3 value of 16.  Of a block with the largest
magnitude a, mx takes the least e with a <= 7 * 2^e (within [-125, 125] for bf16 tokens, [-23, 13] for
fp16), nv e4m3(a / 6) (within [2^-9, 448]); x / scale goes to the nearest code, ties to the even one,
saturated at 6.

Sizes are those of this repository's benchmark and tests where it has them: heads of 64, 128 and
256, batches of 1 .. 64 rows for decode, prompts of 1000 .. 4096 tokens; page sizes and group sizes
are generic.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-ext_amd")
_DEV = "cuda:0"
_TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}
_BLOCK = {"mx": 32, "nv": 16}
_RANGE = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}


def _tx():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import triton_ext_amd
    return triton_ext_amd


def _append(B, tokens, context, Hq, Hkv, D, rot, page, dtype, kind, interleaved=False, scaling="",
            layout="hnd"):
    """`tokens` new tokens in all over B sequences, that hold up to `context` tokens already."""
    return {"path": "append", "B": B, "tokens": tokens, "context": context, "Hq": Hq, "Hkv": Hkv,
            "D": D, "rot": rot, "page": page, "dtype": dtype, "kind": kind,
            "interleaved": interleaved, "scaling": scaling, "layout": layout}


def _read(B, kv_lo, kv_hi, Hkv, D, page, dtype, kind, layout="hnd"):
    """B sequences of kv_lo .. kv_hi tokens, all of each."""
    return {"path": "read", "B": B, "kv_lo": kv_lo, "kv_hi": kv_hi, "Hkv": Hkv, "D": D, "page": page,
            "dtype": dtype, "kind": kind, "layout": layout}


def _attend(B, q_lo, q_hi, kv_lo, kv_hi, Hq, Hkv, D, page, dtype, kind, window=0, causal=True,
            layout="hnd", lse=False):
    """B sequences of q_lo .. q_hi new tokens and kv_lo .. kv_hi tokens in all."""
    return {"path": "attend", "B": B, "q_lo": q_lo, "q_hi": q_hi, "kv_lo": kv_lo, "kv_hi": kv_hi,
            "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "kind": kind,
            "window": window, "causal": causal, "layout": layout, "lse": lse}


def listed():
    return [
        # the new tokens of a decode step of 48 sequences: latency counts
        {"name": "append4_step48", **_append(48, 48, 8000, 32, 8, 128, 128, 16, "bf16", "mx")},
        # prompts of some thousand tokens, positions scaled for a long context, the finer scales
        {"name": "append4_prompts", **_append(7, 9001, 30000, 32, 8, 128, 128, 64, "bf16", "nv",
                                              scaling="yarn")},
        # chunks of a smaller model's prompts: partly rotated heads of 64, pages as they are allocated
        {"name": "append4_heads64", **_append(3, 2001, 4000, 16, 16, 64, 32, 16, "fp16", "mx",
                                              interleaved=True, layout="nhd")},
        # one short conversation leaves the cache (to another device, or to be extended in 16 bits)
        {"name": "read4_one_1500", **_read(1, 1500, 1500, 4, 64, 16, "fp16", "nv")},
        # long contexts leave the cache
        {"name": "read4_long", **_read(4, 20000, 60000, 8, 128, 16, "bf16", "mx")},
        # one user, a short conversation: the smallest attention call
        {"name": "attend4_one_1500", **_attend(1, 1, 1, 1500, 1500, 16, 4, 64, 16, "bf16", "mx")},
        # a serving batch: 32 sequences of very different lengths, one token each
        {"name": "attend4_batch32", **_attend(32, 1, 1, 100, 16384, 32, 8, 128, 16, "bf16", "mx")},
        # a few very long contexts, several drafted tokens to verify
        {"name": "attend4_long", **_attend(4, 4, 4, 60000, 131072, 32, 8, 128, 64, "fp16", "nv")},
        # heads of 256, eight of q on one of k and v, one token each
        {"name": "attend4_heads256", **_attend(8, 1, 1, 5000, 32768, 16, 2, 256, 32, "bf16", "nv")},
        # long prompts taken in chunks of 2048
        {"name": "attend4_chunk2048", **_attend(2, 2048, 2048, 8192, 16384, 32, 8, 128, 64, "bf16",
                                                "mx")},
        # decode and prompt chunks in one batch, a sliding window, a head of k and v per head of q,
        # pages as they are allocated
        {"name": "attend4_mixed_window", **_attend(24, 1, 300, 300, 8000, 16, 16, 64, 16, "fp16",
                                                   "mx", window=1024, layout="nhd", lse=True)},
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
        path = rng.choice(["append", "append", "read", "attend", "attend", "attend"])
        dtype, kind = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["mx", "nv"])
        page = rng.choice([8, 16, 16, 32, 64, 128])
        layout = rng.choice(["hnd", "hnd", "nhd"])
        D = rng.choice([64, 64, 128, 128, 128, 96, 256])
        Hq, Hkv = _heads(rng)
        if path == "append":
            B = _log(rng, 1, 64)
            c = _append(B, max(B, _log(rng, 1, 9000)), _log(rng, 1, 30000), Hq, Hkv, D,
                        rng.choice([D, D // 2]), page, dtype, kind, rng.random() < 0.4,
                        rng.choice(["", "linear", "yarn"]), layout)
            if c["tokens"] * Hq * D <= 9001 * 32 * 128 and B * c["context"] * Hkv * D <= 1 << 29:
                return c
        elif path == "read":
            hi = _log(rng, 1, 60000)
            c = _read(_log(rng, 1, 48), rng.choice([hi, max(1, hi // 4)]), hi, Hkv, D, page, dtype,
                      kind, layout)
            if c["B"] * hi * Hkv * D <= 4 * 60000 * 8 * 128:
                return c
        else:
            form = rng.choice(["decode", "decode", "few", "chunk"])
            if form == "chunk":
                B, q_hi = rng.choice([1, 1, 2, 3]), _log(rng, 64, 2048)
            else:
                B, q_hi = _log(rng, 1, 48), 1 if form == "decode" else _log(rng, 2, 16)
            q_lo = rng.choice([q_hi, max(1, q_hi // 3)])
            kv_hi = max(q_hi, _log(rng, 16, 16384 if form == "chunk" else 131072))
            kv_lo = rng.choice([q_hi, kv_hi, max(q_hi, kv_hi // 2)])
            c = _attend(B, q_lo, q_hi, kv_lo, kv_hi, Hq, Hkv, D, page, dtype, kind,
                        rng.choice([0, 0, 0, 100, 4096]), rng.random() < 0.85, layout,
                        rng.random() < 0.3)
            if (B * q_hi * Hq * kv_hi * D <= 2 * 2048 * 32 * 16384 * 128
                    and B * kv_hi * Hkv * D <= 32 * 16384 * 8 * 128):
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


def _spread(h, count, lo, hi):
    """`count` lengths of lo .. hi, spread over their logarithm, hi among them."""
    if lo == hi:
        return [hi] * count
    u = torch.rand(count, generator=h).tolist()
    lo, span = math.log(max(lo, 1)), math.log(hi) - math.log(max(lo, 1))
    got = [int(round(math.exp(lo + x * span))) for x in u]
    got[count // 2] = hi
    return got


def _parts(h, count, total):
    """`total` tokens over `count` sequences, one each at least, in unequal parts."""
    w = torch.rand(count, generator=h) + 0.05
    n = [1 + int(x) for x in (w / w.sum() * (total - count)).floor().tolist()]
    n[0] += total - sum(n)
    return n


def _sizes(c):
    """The tokens of the pass and the lengths of a case's sequences: its own, whatever the seed."""
    h = torch.Generator()
    h.manual_seed(7)
    if c["path"] == "append":
        n = _parts(h, c["B"], c["tokens"])
        return n, [x + y for x, y in zip(n, _spread(h, c["B"], 0, c["context"]))]
    if c["path"] == "read":
        lens = _spread(h, c["B"], c["kv_lo"], c["kv_hi"])
        return lens, lens
    n = _spread(h, c["B"], c["q_lo"], c["q_hi"])
    return n, [max(x, y) for x, y in zip(n, _spread(h, c["B"], c["kv_lo"], c["kv_hi"]))]


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _starts(n):
    got = [0]
    for x in n:
        got.append(got[-1] + x)
    return got


def _tables(h, lens, page):
    """A page table for sequences of these lengths, their pages scattered over the pool."""
    need = [-(-x // page) for x in lens]
    P = int(sum(need) * 1.1) + 3
    order = torch.randperm(P, generator=h).to(torch.int32)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, P


def _cache(g, P, c):
    """Codes [P, page, Hkv, D / 2] and scales [P, page, Hkv, D / block] of N(0, 1) values: "hnd", a
    head's tokens together in memory (of the scales, those of one block of dims), or "nhd", dense."""
    page, Hkv, D, block = c["page"], c["Hkv"], c["D"], _BLOCK[c["kind"]]
    codes = torch.empty((P, Hkv, page, D // 2), dtype=torch.uint8, device=_DEV)
    scales = torch.empty((P, Hkv, page, D // block), device=_DEV,
                         dtype=torch.uint8 if c["kind"] == "mx" else torch.float8_e4m3fn)
    step = max(1, (1 << 26) // (page * Hkv * D))
    for i in range(0, P, step):
        x = torch.randn((min(step, P - i), Hkv, page, D), generator=g, device=_DEV)
        codes[i:i + step], scales[i:i + step] = _quantise(x, c["kind"], _TORCH[c["dtype"]])
    codes = codes.permute(0, 2, 1, 3)
    if c["layout"] == "hnd":
        return codes, scales.permute(0, 1, 3, 2).contiguous().permute(0, 3, 1, 2)
    return codes.contiguous(), scales.permute(0, 2, 1, 3).contiguous()


def _frequencies(rot, scaling):
    """10000^(-2 i / rot) in fp32, scaled for contexts 8 times as long, and the factor on cos and sin."""
    f = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    scale = 1.0
    if scaling == "linear":
        f = f / 8.0
    elif scaling == "yarn":
        turns = 4096.0 * f / (2 * math.pi)  # of one frequency over the trained context
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f / 8.0 * (1 - keep) + f * keep
        scale = 0.1 * math.log(8.0) + 1.0
    return f.to(torch.float32).to(_DEV), scale


def prepare(case, seed):
    c = dict(case)
    g, h = _gens(seed)
    n, lens = _sizes(c)
    T, dt = sum(n), _TORCH[c["dtype"]]
    table, P = _tables(h, lens, c["page"])
    s = {"case": c, "n": n, "lens": lens, "T": T, "page_table": table.to(_DEV), "kv_len": _int(lens),
         "cu_q": _int(_starts(n)) if max(n) > 1 or min(n) < 1 else None}
    s["k_cache"], s["k_block_scale"] = _cache(g, P, c)
    s["v_cache"], s["v_block_scale"] = _cache(g, P, c)
    if c["path"] != "read":
        Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
        # as a fused projection leaves them
        qkv = torch.randn((T, Hq + 2 * Hkv, D), generator=g, device=_DEV).to(dt)
        if c["path"] == "append":
            s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
            s["inv_freq"], s["scale"] = _frequencies(c["rot"], c["scaling"])
        else:
            s["q"] = qkv[:, :Hq].contiguous()  # as the rotation leaves it
    return s


# ---------------------------------------------------------------------------
# The paths, in elementary operations
# ---------------------------------------------------------------------------

def _quantise(x, kind, dtype):
    """Codes, two a byte, and scales of fp32 (or fp64) values [..., D]."""
    y = x.unflatten(-1, (-1, _BLOCK[kind]))
    a = y.abs().amax(dim=-1)
    if kind == "mx":
        f, e = torch.frexp(a)  # a = f 2^e, f in [1/2, 1)
        lo, hi = _RANGE[dtype]
        e = (e - 3 + (f > 0.875).to(e.dtype)).clamp(lo, hi)
        e = torch.where(a > 0, e, lo)
        y, scales = torch.ldexp(y, -e[..., None]), (e + 127).to(torch.uint8)
    else:
        scales = (a / 6.0).clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn)
        y = y / scales.to(y.dtype)[..., None]
    m = y.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5)
            + (m >= 3.5) + (m > 5.0))
    code = (code + 8 * torch.signbit(y)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scales


def _values(codes, scales, kind):
    """What codes [..., D / 2] and scales [..., D / block] stand for, in fp32."""
    e2m1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=_DEV)
    e2m1 = torch.cat((e2m1, -e2m1))
    x = e2m1[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).int()]
    factor = torch.exp2(scales.float() - 127.0) if kind == "mx" else scales.float()
    return (x.unflatten(-1, (-1, _BLOCK[kind])) * factor[..., None]).flatten(-2)


def _pages_of(t, pages):
    """t[pages], also of a type that torch does not index."""
    return t.view(torch.uint8)[pages].view(t.dtype) if t.dtype != torch.uint8 else t[pages]


def _rotate(x, positions, inv_freq, interleaved, scale):
    """x [..., D] in fp32 with angles [..., rot / 2] = position * inv_freq broadcast over it."""
    a = positions.double()[..., None] * inv_freq.double()
    cos, sin = (torch.cos(a) * scale).float(), (torch.sin(a) * scale).float()
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
    """Of every token of the pass: its sequence, its place among that one's, its position."""
    B, T = len(s["n"]), s["T"]
    if s["cu_q"] is None:
        seq = torch.arange(B, device=_DEV)
        return seq, torch.zeros_like(seq), s["kv_len"].long() - 1
    cu = s["cu_q"].long()
    seq = torch.repeat_interleave(torch.arange(B, device=_DEV), cu.diff(), output_size=T)
    off = torch.arange(T, device=_DEV) - cu[seq]
    return seq, off, s["kv_len"].long()[seq] - cu.diff()[seq] + off


def _plain_read(s):
    c = s["case"]
    seq, _, pos = _places(s)
    page, slot = s["page_table"][seq, pos // c["page"]].long(), pos % c["page"]

    def side(t):
        scales = s[t + "_block_scale"]
        held = scales.view(torch.uint8)[page, slot].view(scales.dtype)
        return _values(s[t + "_cache"][page, slot], held, c["kind"]).to(_TORCH[c["dtype"]])
    return {"k": side("k"), "v": side("v")}


def _plain_append(s):
    c = s["case"]
    seq, _, pos = _places(s)
    page, slot = s["page_table"][seq, pos // c["page"]].long(), pos % c["page"]
    q, k = (_rotate(s[t].float(), pos[:, None], s["inv_freq"], c["interleaved"], s["scale"])
            for t in ("q", "k"))

    def write(t, x):
        codes, scales = _quantise(x, c["kind"], s["q"].dtype)
        s[t + "_cache"][page, slot] = codes
        s[t + "_block_scale"].view(torch.uint8)[page, slot] = scales.view(torch.uint8)
    write("k", k)
    write("v", s["v"].float())
    return {"q": q.to(s["q"].dtype), **_plain_read(s)}


def _plain_attend(s):
    c = s["case"]
    B, Hq, Hkv, D, page = (c[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    G, Q, W = Hq // Hkv, max(s["n"]), s["page_table"].shape[1]
    seq, off, _ = _places(s)
    pages = s["page_table"].long().clamp_min(0)
    L = W * page

    def keys(t):  # [B, Hkv, L, D]
        x = _values(s[t + "_cache"][pages], _pages_of(s[t + "_block_scale"], pages), c["kind"])
        x = x.reshape(B, L, Hkv, D)
        held = torch.arange(L, device=_DEV) < s["kv_len"][:, None]
        return x.masked_fill(~held[:, :, None, None], 0.0).transpose(1, 2).contiguous()

    q = torch.zeros((B, Q, Hq, D), device=_DEV)
    q[seq, off] = s["q"].float()
    q = q.view(B, Q, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Q * G, D)
    scores = torch.matmul(q, keys("k").transpose(2, 3)) * D ** -0.5
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
    o = torch.matmul(p, keys("v")) / total.masked_fill(total == 0, 1.0)

    def back(t):
        return t.view(B, Hkv, Q, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Q, Hq, -1)[seq, off]
    out = back(o).to(s["q"].dtype)
    if not c["lse"]:
        return out
    return {"o": out, "lse": back((m + total.log()) / math.log(2.0))[..., 0].contiguous()}


_PLAIN = {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}


# ---------------------------------------------------------------------------
# The same by this package
# ---------------------------------------------------------------------------

def _own_read(tx, s, c):
    k, v = tx.paged_read(s["k_cache"], s["v_cache"], s["page_table"], s["kv_len"], s["cu_q"],
                         tokens=s["T"], dtype=_TORCH[c["dtype"]], k_block_scale=s["k_block_scale"],
                         v_block_scale=s["v_block_scale"])
    return {"k": k, "v": v}


def _own_append(tx, s, c):
    q = tx.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_len"],
                        s["cu_q"], q=s["q"], inv_freq=s["inv_freq"], interleaved=c["interleaved"],
                        scale=s["scale"], k_block_scale=s["k_block_scale"],
                        v_block_scale=s["v_block_scale"])
    return {"q": q, **_own_read(tx, s, c)}


def _own_attend(tx, s, c):
    r = tx.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_len"],
                           s["cu_q"], sm_scale=c["D"] ** -0.5, causal=c["causal"],
                           window=c["window"], k_block_scale=s["k_block_scale"],
                           v_block_scale=s["v_block_scale"], return_lse=c["lse"])
    return {"o": r[0], "lse": r[1]} if c["lse"] else r


_OWN = {"append": _own_append, "read": _own_read, "attend": _own_attend}


def run(state):
    c = state["case"]
    return _OWN[c["path"]](_tx(), state, c) if own else _PLAIN[c["path"]](state)


# ---------------------------------------------------------------------------
# Work, and the results in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    c, D = case, case["D"]
    token = 2 * c["Hkv"] * (D // 2 + D // _BLOCK[c["kind"]])  # bytes of k and v in the cache
    if c["path"] == "append":
        T = c["tokens"]
        return {"bytes": T * (2 * D * (2 * c["Hq"] + 4 * c["Hkv"]) + token),
                "flops": 3 * T * (c["Hq"] + c["Hkv"]) * c["rot"]}
    n, lens = _sizes(c)
    if c["path"] == "read":
        return {"bytes": sum(lens) * (token + 2 * 2 * c["Hkv"] * D), "flops": 0}
    pairs = span = 0
    for k, length in zip(n, lens):
        first = length - k  # the first new token's position
        span += min(length, c["window"] + k - 1) if c["window"] else length
        for p in range(first, length):
            to = p + 1 if c["causal"] else length
            pairs += to - max(0, p - c["window"] + 1) if c["window"] else to
    return {"bytes": 2 * sum(n) * c["Hq"] * D * 2 + span * token, "flops": 4 * pairs * c["Hq"] * D}


_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values(codes, scales):
    """Codes [..., D / 2] and their scales [..., blocks] as numbers of 64 bits."""
    x = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device=_DEV)
    for half in (0, 1):
        nibble = codes.to(torch.int16) // (16 if half else 1) % 16
        value = torch.zeros(nibble.shape, dtype=torch.float64, device=_DEV)
        for i, m in enumerate(_MAGNITUDES):
            value += m * ((nibble == i).double() - (nibble == i + 8).double())
        x[..., half::2] = value
    if scales.dtype == torch.uint8:
        factor = torch.pow(2.0, scales.double() - 127)
    else:
        factor = scales.to(torch.float64)
    return x * factor.repeat_interleave(x.shape[-1] // scales.shape[-1], dim=-1)


def _exact_rounded(x, c):
    """The values that the cache holds of x [N, H, D]: the nearest of the fifteen in each block."""
    size = _BLOCK[c["kind"]]
    blocks = x.reshape(x.shape[:-1] + (x.shape[-1] // size, size))
    top = blocks.abs().max(dim=-1, keepdim=True).values
    if c["kind"] == "mx":
        lo, hi = (-125, 125) if c["dtype"] == "bf16" else (-23, 13)
        e = torch.ceil(torch.log2(top / 7.0))
        e = e - (top <= 7.0 * torch.pow(2.0, e - 1)).double()  # (where the logarithm was rounded)
        e = e + (top > 7.0 * torch.pow(2.0, e)).double()
        unit = torch.pow(2.0, e.clamp(lo, hi))
    else:
        unit = (top / 6.0).float().clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn).double()
    m = (blocks.abs() / unit).clamp(max=6.0)
    step = torch.pow(2.0, torch.floor(torch.log2(m.clamp(min=1.0)))) / 2  # of e2m1 from m on
    return (torch.sign(blocks) * torch.round(m / step) * step * unit).reshape(x.shape)


def _exact_tokens(s, t, b, length, h):
    """Head h of sequence b's tokens [length, D]."""
    ids = s["page_table"][b, :-(-length // s["case"]["page"])].long()
    scales = s[t + "_block_scale"]
    held = scales.view(torch.uint8)[:, :, h][ids].contiguous().view(scales.dtype)
    codes = s[t + "_cache"][:, :, h][ids]
    return _exact_values(codes, held).reshape(-1, s["case"]["D"])[:length]


def _exact_read(c, s):
    out = {t: torch.empty((s["T"], c["Hkv"], c["D"]), dtype=torch.float64, device=_DEV)
           for t in ("k", "v")}
    first = _starts(s["n"])
    for b, length in enumerate(s["lens"]):
        for h in range(c["Hkv"]):
            for t in out:
                out[t][first[b]:first[b + 1], h] = _exact_tokens(s, t, b, length, h)
    return out


def _exact_turn(x, at, s, c):
    """The pairs of x [N, H, D] at positions `at` as complex numbers, turned."""
    a = torch.outer(at.double(), s["inv_freq"].double())
    turns = torch.complex(torch.cos(a), torch.sin(a)) * s["scale"]
    y, half = x.double(), turns.shape[1]
    first, second = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if c["interleaved"]
                     else (slice(0, half), slice(half, 2 * half)))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turns[:, None, :]
    y = y.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_append(c, s):
    first = _starts(s["n"])
    q = torch.empty(s["q"].shape, dtype=torch.float64, device=_DEV)
    k = torch.empty(s["k"].shape, dtype=torch.float64, device=_DEV)
    for b, (n, length) in enumerate(zip(s["n"], s["lens"])):
        rows = slice(first[b], first[b] + n)
        at = torch.arange(length - n, length, device=_DEV)
        q[rows] = _exact_turn(s["q"][rows], at, s, c)
        k[rows] = _exact_rounded(_exact_turn(s["k"][rows], at, s, c), c)
    return {"q": q, "k": k, "v": _exact_rounded(s["v"].double(), c)}


def _exact_attend(c, s):
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    G, first = Hq // Hkv, _starts(s["n"])
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=_DEV)
    for b, (n, length) in enumerate(zip(s["n"], s["lens"])):
        j = torch.arange(length, device=_DEV)
        for h in range(Hkv):
            K, V = (_exact_tokens(s, t, b, length, h) for t in ("k", "v"))
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
    return {"append": _exact_append, "read": _exact_read,
            "attend": _exact_attend}[c["path"]](c, prepare(c, seed))
