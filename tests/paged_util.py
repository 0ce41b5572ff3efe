"""Helpers of the paged-cache and norm tests: batches of sequences, caches in pages and plain 64-bit results (not a test
module)."""
from __future__ import annotations

import numpy as np

import vva

DT = {vva.F16: "float16", vva.BF16: "bfloat16", vva.F32: "float32"}
# half a step of a type relative to the value, and the smallest step
HALF = {vva.F16: 2.0 ** -11, vva.BF16: 2.0 ** -8, vva.F32: 2.0 ** -24}
TINY = {vva.F16: 2.0 ** -25, vva.BF16: 0.0, vva.F32: 0.0}


def dtype(torch, t):
    return getattr(torch, DT[t])


class Pages:
    """A K and a V pool and a batch of sequences (n new tokens, L keys) in it: pages in random order, every slot and table
    entry that no sequence owns filled with `stale` and ids outside the pool."""

    def __init__(self, torch, lens, Hq, Hkv, d, type_, page, seed, stale=float("nan"), extra_rows=0, width=0, slot_major=False,
                 n_pages=0, scale=1.0):
        self.torch, self.lens, self.Hq, self.Hkv, self.d, self.type, self.page = torch, lens, Hq, Hkv, d, type_, page
        dt = dtype(torch, type_)
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        used = [-(-L // page) for _, L in lens]
        n_pages = max(n_pages, sum(used) + 3)
        rng = np.random.default_rng(seed)
        ids = rng.permutation(n_pages)[:sum(used)].astype(np.int32)
        if n_pages > 2 * sum(used) + 3:                     # a huge pool: the pages at its far end
            ids = (n_pages - 1 - rng.permutation(sum(used))).astype(np.int32)
        table = np.full((len(lens), max([width, 1] + used)), 0x7ffffff0, np.int32)
        at = 0
        for s, u in enumerate(used):
            table[s, :u] = ids[at:at + u]
            at += u
        self.table_host = table
        shape = (n_pages, page, Hkv, d) if slot_major else (n_pages, Hkv, page, d)
        huge = n_pages * page * Hkv * d > 1 << 28
        pools = [torch.empty(shape, dtype=dt, device="cuda") for _ in range(2)]
        if not huge:
            for p in pools:
                p.fill_(stale)
        self.k, self.v = [p.transpose(1, 2) if slot_major else p for p in pools]
        for s, (_, L) in enumerate(lens):
            for p in (self.k, self.v):
                for i in range(used[s]):
                    m = min(page, L - i * page)
                    p[int(table[s, i]), :, :m] = (torch.randn(Hkv, m, d, generator=self.gen, device="cuda") * scale).to(dt)
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.n_tok = int(self.starts[-1])
        self.rows = self.n_tok + extra_rows
        self.q_start = torch.from_numpy(self.starts).cuda()
        self.kv_len = torch.tensor([L for _, L in lens], dtype=torch.int32, device="cuda")
        self.table = torch.from_numpy(table).cuda()
        self.q = (torch.randn(max(self.rows, 1), Hq, d, generator=self.gen, device="cuda") * scale).to(dt)
        self.max_new = max([1] + [n for n, _ in lens])

    def batch(self, max_new=0):
        return vva.Batch(self.q_start, self.kv_len, self.table, max_new or self.max_new)

    def keys(self, s, pool, kvh):
        """Rows [0, L) of sequence s and kv head kvh, in 64 bits."""
        L = self.lens[s][1]
        ids = [int(i) for i in self.table_host[s, :-(-L // self.page)]]
        return pool[ids, kvh].reshape(-1, self.d)[:L].double()


def attention(P: Pages, scale, q=None):
    """(64-bit result, how far a correct result may be off) of every packed row, from the definition.

    A row is sum_j p_j v_j / sum_j p_j with p in the pages' type (half a step u of p_j, and in F16 half the smallest step
    where p_j, whose largest is at least 1, is below the normal range), its scores in F32 sums of d products (each within
    (d + 2) 2^-24 of the sum of their magnitudes; an error of a score is one of p_j relative to it; exp2, its argument's
    rounding and the sums add a few 2^-24 more), and rounded once to the output type."""
    torch = P.torch
    q = P.q if q is None else q
    u, tiny = HALF[P.type], TINY[P.type]
    ref = torch.zeros(P.rows, P.Hq, P.d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(ref)
    G = P.Hq // P.Hkv
    for s, (n, L) in enumerate(P.lens):
        if n == 0 or L == 0:
            continue
        r0 = int(P.starts[s])
        j = torch.arange(L, device="cuda")
        seen = j[None, :] <= (L - n + torch.arange(n, device="cuda"))[:, None]
        none = ~seen.any(-1, keepdim=True)
        for h in range(P.Hq):
            k, v = P.keys(s, P.k, h // G), P.keys(s, P.v, h // G)
            qh = q[r0:r0 + n, h].double()
            sc = (qh @ k.t().contiguous()) * scale
            mag = (qh.abs() @ k.abs().t().contiguous()) * scale
            sc = sc.masked_fill(~seen, -float("inf"))
            m = sc.amax(-1, keepdim=True).masked_fill(none, 0.0)
            p = torch.exp(sc - m)
            den = p.sum(-1, keepdim=True).masked_fill(none, 1.0)
            out = (p @ v) / den
            # the score's error, and 2^-24 of the exponent's argument, relative to p
            rel = u + 2.0 ** -23 * (8 + (P.d + 2) * mag.masked_fill(~seen, 0.0) + (sc - m).abs().masked_fill(~seen, 0.0))
            e = (rel * p + tiny * seen) / den
            ref[r0:r0 + n, h] = out
            tol[r0:r0 + n, h] = 1.01 * (e @ v.abs() + e.sum(-1, keepdim=True) * out.abs()) + u * out.abs() + tiny
    return ref, tol


def check_rows(got, ref, tol, what=""):
    d = (got.double() - ref).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((d / tol.clamp(min=1e-30)).nan_to_num(1e9).max()):.3g} "
                                 f"times the tolerance, first at {bad.nonzero()[0].tolist()}")
