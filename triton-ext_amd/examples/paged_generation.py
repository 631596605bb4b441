"""Generation from a paged key/value cache: a few layers of attention with random weights.

    python triton-ext_amd/examples/paged_generation.py [--sequences 4] [--tokens 32] [--beams 2]

Prompts of different lengths go through in chunks, each of them then forks into beams that share
its pages, and all beams take one token a step, in a HIP graph that is captured once and
replayed as the sequences grow.  At the end every other beam is freed and the cache made
dense again.  Prints the step's time, and what the pages did.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import triton_ext_amd as tx  # noqa: E402


class Decoder:
    """`layers` layers of y = x + Wo attention(Wqkv x / rms), with a paged cache each."""

    def __init__(self, layers=2, width=512, Hq=8, Hkv=2, D=64, pages=256, page=16, rows=16,
                 entries=64, dtype=torch.bfloat16, cache_dtype=None, device="cuda", seed=0):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.Hq, self.Hkv, self.D, self.page = Hq, Hkv, D, page

        def weight(n, k):
            return torch.randn(n, k, generator=g, device=device).mul_(k ** -0.5).to(dtype)
        self.qkv = [weight((Hq + 2 * Hkv) * D, width) for _ in range(layers)]
        self.out = [weight(width, Hq * D) for _ in range(layers)]
        kind = cache_dtype or dtype
        self.k, self.v = ([torch.zeros(pages, page, Hkv, D, dtype=kind, device=device)
                           for _ in range(layers)] for _ in range(2))
        self.scale = (torch.full((Hkv,), 1 / 64, device=device)
                      if kind == torch.float8_e4m3fn else None)
        self.inv_freq, self.rope_scale = tx.rotary_frequencies(D, device=device)
        self.table = torch.full((rows, entries), -1, dtype=torch.int32, device=device)
        self.length = torch.zeros(rows, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)

    def reserve(self, more):
        """Room for `more` [rows] new tokens of each sequence, in place."""
        self.missing = tx.page_reserve(self.table, self.length, self.refs, self.length + more,
                                       self.page, out=(self.table, self.length, self.refs))[3]

    def forward(self, x, rows, cu_q=None):
        """x [T, width], the new tokens of sequences `rows` (a slice), already reserved."""
        H, G, D = self.Hq, self.Hkv, self.D
        table, length = self.table[rows], self.length[rows]
        for qkv, out, k, v in zip(self.qkv, self.out, self.k, self.v):
            h = x.float()
            h = (h * h.square().mean(-1, keepdim=True).add(1e-6).rsqrt()).to(x.dtype)
            y = (h @ qkv.t()).view(x.shape[0], H + 2 * G, D)
            q = tx.paged_append(y[:, H:H + G], y[:, H + G:], k, v, table, length, cu_q,
                                q=y[:, :H], inv_freq=self.inv_freq, scale=self.rope_scale,
                                k_scale=self.scale, v_scale=self.scale)
            o = tx.paged_attention(q, k, v, table, length, cu_q, sm_scale=D ** -0.5,
                                   k_scale=self.scale, v_scale=self.scale)
            x = x + o.reshape(x.shape[0], H * D) @ out.t()
        return x

    def fork(self, parent, child):
        """Sequences `child` continue `parent`, in every layer's cache."""
        self.missing = tx.page_fork(self.k + self.v, self.table, self.length, self.refs, parent,
                                    child, out=(self.table, self.length, self.refs))[3]

    def free(self, drop):
        tx.page_free(self.table, self.length, self.refs, drop, self.page,
                     out=(self.table, self.length, self.refs))

    def compact(self):
        return tx.page_compact(self.k + self.v, self.table, self.refs,
                               out=(self.table, self.refs))[2]


def generate(sequences=4, tokens=32, beams=2, chunk=64, width=512, device="cuda", seed=0, **kw):
    """Runs all of it; returns the decoder, the inputs of every row and its outputs."""
    rows = sequences * beams
    d = Decoder(width=width, rows=rows, device=device, seed=seed, **kw)
    g = torch.Generator(device=device)
    g.manual_seed(seed + 1)
    dtype = d.qkv[0].dtype
    lengths = [17 + 41 * i % 150 for i in range(sequences)]
    prompts = [torch.randn(n, width, generator=g, device=device).to(dtype) for n in lengths]
    fed, got = [[] for _ in range(rows)], [[] for _ in range(rows)]

    # prompts, a chunk of each at a time
    done = [0] * sequences
    while any(a < n for a, n in zip(done, lengths)):
        take = [min(chunk, n - a) for a, n in zip(done, lengths)]
        more = torch.tensor(take + [0] * (rows - sequences), dtype=torch.int32, device=device)
        cu = torch.nn.functional.pad(more[:sequences].cumsum(0, dtype=torch.int32), (1, 0))
        d.reserve(more)
        x = torch.cat([p[a:a + t] for p, a, t in zip(prompts, done, take)])
        y = d.forward(x, slice(0, sequences), cu).split(take)
        for i, part in enumerate(y):
            got[i].append(part)
        done = [a + t for a, t in zip(done, take)]
    for i in range(sequences):
        fed[i].append(prompts[i])

    # beams
    parent = torch.arange(sequences, device=device, dtype=torch.int32).repeat_interleave(beams - 1)
    child = torch.arange(sequences, rows, device=device, dtype=torch.int32)
    if beams > 1:
        d.fork(parent, child)
        for p, c in zip(parent.tolist(), child.tolist()):
            fed[c], got[c] = list(fed[p]), list(got[p])

    # a step, captured once
    x = torch.empty(rows, width, dtype=dtype, device=device)
    one = torch.ones(rows, dtype=torch.int32, device=device)

    def step():
        d.reserve(one)
        return d.forward(x, slice(0, rows))

    books = [t.clone() for t in (d.table, d.length, d.refs)]  # a first step outside the capture
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.zero_()
        step()
    torch.cuda.current_stream().wait_stream(side)
    for t, u in zip((d.table, d.length, d.refs), books):
        t.copy_(u)  # .. whose tokens are forgotten
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = step()
    start = time.perf_counter()
    for _ in range(tokens):
        x.copy_(torch.randn(rows, width, generator=g, device=device))
        graph.replay()
        for r in range(rows):
            fed[r].append(x[r:r + 1].clone())
            got[r].append(y[r:r + 1].clone())
    torch.cuda.synchronize()
    d.step_ms = (time.perf_counter() - start) / max(tokens, 1) * 1e3
    return d, [torch.cat(f) for f in fed], [torch.cat(o) for o in got]


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--beams", type=int, default=2)
    a = ap.parse_args()
    d, fed, _ = generate(a.sequences, a.tokens, a.beams)
    used = int((d.refs > 0).sum())
    print(f"{len(fed)} sequences of {min(map(len, fed))} .. {max(map(len, fed))} tokens in {used} "
          f"pages of {d.page} ({int((d.refs > 1).sum())} of them shared), {d.step_ms:.2f} ms a step")
    d.free(torch.arange(len(fed), device="cuda") % 2 == 1)
    moved = d.compact()
    print(f"every other one freed: {int((d.refs > 0).sum())} pages left, {int(moved)} of them moved")


if __name__ == "__main__":
    main()
