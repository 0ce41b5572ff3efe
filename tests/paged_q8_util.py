"""Helpers of the tests over Q8_0 pages: batches in pools of codes and scales, and plain 64-bit results (not a test module)."""
from __future__ import annotations

import numpy as np

import vva
from paged_util import HALF, TINY, dtype


def parts(raw, d):
    """Codes [n_pages, Hkv, page, d] and scales [n_pages, Hkv, d / 32, page] of pages, as views of their bytes."""
    page = raw.shape[2] // (d // 32 * 34)
    import torch
    codes = raw[..., :page * d].view(torch.int8).unflatten(2, (page, d))
    return codes, raw[..., page * d:].view(torch.float16).unflatten(2, (d // 32, page))


def values(raw, d):
    """What the pages stand for, in 64 bits: [n_pages, Hkv, page, d]."""
    codes, scales = parts(raw, d)
    return codes.double() * scales.double().transpose(-1, -2).repeat_interleave(32, -1)


class Q8Pages:
    """A K and a V pool of Q8_0 pages and a batch of sequences (n new tokens, L keys) in it: pages in random order; every
    slot and table entry that no sequence owns holds NaN scales, wild codes and ids outside the pool."""

    def __init__(self, torch, lens, Hq, Hkv, d, io, page, seed, extra_rows=0, width=0, n_pages=0, scale=1.0, head_major=False):
        self.torch, self.lens, self.Hq, self.Hkv, self.d, self.type, self.page = torch, lens, Hq, Hkv, d, io, page
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        used = [-(-L // page) for _, L in lens]
        n_pages = max(n_pages, sum(used) + 3)
        rng = np.random.default_rng(seed)
        ids = rng.permutation(n_pages)[:sum(used)].astype(np.int32)
        self.huge = n_pages > 2 * sum(used) + 3            # a huge pool: the pages at its far end
        if self.huge:
            ids = (n_pages - 1 - rng.permutation(sum(used))).astype(np.int32)
        table = np.full((len(lens), max([width, 1] + used)), 0x7ffffff0, np.int32)
        at = 0
        for s, u in enumerate(used):
            table[s, :u] = ids[at:at + u]
            at += u
        self.table_host = table
        run = page * d // 32 * 34
        self.raw = []
        for _ in range(2):
            shape = (Hkv, n_pages, run + 32) if head_major else (n_pages, Hkv, run)
            raw = torch.empty(shape, dtype=torch.uint8, device="cuda")
            self.raw.append(raw.transpose(0, 1)[..., :run] if head_major else raw)
        if not self.huge:
            for raw in self.raw:
                codes, scales = parts(raw, d)
                codes.copy_(torch.randint(-128, 128, codes.shape, generator=self.gen, device="cuda", dtype=torch.int8))
                scales.fill_(float("nan"))
        for s, (_, L) in enumerate(lens):
            for raw in self.raw:
                for i in range(used[s]):
                    m = min(page, L - i * page)
                    one = raw[int(table[s, i]):int(table[s, i]) + 1]
                    codes, scales = parts(one, d)
                    codes[0, :, :m] = torch.randint(-127, 128, (Hkv, m, d), generator=self.gen, device="cuda", dtype=torch.int8)
                    # values of about the size of `scale`, the blocks' scales an octave apart
                    u = torch.rand(Hkv, d // 32, m, generator=self.gen, device="cuda")
                    scales[0, :, :, :m] = (scale / 80 * 2.0 ** (u - 0.5)).half()
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.n_tok = int(self.starts[-1])
        self.rows = self.n_tok + extra_rows
        self.q_start = torch.from_numpy(self.starts).cuda()
        self.kv_len = torch.tensor([L for _, L in lens], dtype=torch.int32, device="cuda")
        self.table = torch.from_numpy(table).cuda()
        self.q = (torch.randn(max(self.rows, 1), Hq, d, generator=self.gen, device="cuda") * scale).to(dtype(torch, io))
        self.max_new = max([1] + [n for n, _ in lens])

    @property
    def k(self):
        return vva.q8_pages(self.raw[0], self.d)

    @property
    def v(self):
        return vva.q8_pages(self.raw[1], self.d)

    def batch(self, max_new=0):
        return vva.Batch(self.q_start, self.kv_len, self.table, max_new or self.max_new)

    def keys(self, s, which, kvh):
        """Rows [0, L) of sequence s and kv head kvh, in 64 bits."""
        L = self.lens[s][1]
        ids = [int(i) for i in self.table_host[s, :-(-L // self.page)]]
        return values(self.raw[which][ids][:, kvh:kvh + 1], self.d).reshape(-1, self.d)[:L]

    def places(self):
        """(page, slot) of each packed token, None before key 0, and its index."""
        place, index = [], []
        for s, (n, L) in enumerate(self.lens):
            for j in range(L - n, L):
                index.append(j)
                place.append((int(self.table_host[s, j // self.page]), j % self.page) if j >= 0 else None)
        return place, index


def attention(P: Q8Pages, scale, q=None):
    """(64-bit result, how far a correct result may be off) of every packed row, from the definition.

    K, V and q go into the products as F16: half a step u of each value, and half of F16's smallest step.  The probabilities
    are F16 too (u of p_j, and half the smallest step where p_j, whose largest is at least 1, is below the normal range); a
    score is an F32 sum of d products (within (d + 2) 2^-24 of the sum of their magnitudes), and an error of it is one of
    p_j relative to it; exp2, its argument's rounding and the sums add a few 2^-24 more.  The result is rounded once."""
    torch = P.torch
    q = P.q if q is None else q
    u, tiny, step = HALF[vva.F16], TINY[vva.F16], 2.0 ** -25
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
            k, v = P.keys(s, 0, h // G), P.keys(s, 1, h // G)
            qh = q[r0:r0 + n, h].double()
            sc = (qh @ k.t().contiguous()) * scale
            mag = (qh.abs() @ k.abs().t().contiguous()) * scale
            small = step * scale * (qh.abs().sum(-1, keepdim=True) + k.abs().sum(-1)[None, :])
            sc = sc.masked_fill(~seen, -float("inf"))
            m = sc.amax(-1, keepdim=True).masked_fill(none, 0.0)
            p = torch.exp(sc - m)
            den = p.sum(-1, keepdim=True).masked_fill(none, 1.0)
            out = (p @ v) / den
            err = (u * mag + small + 2.0 ** -23 * (8 + (P.d + 2) * mag)).masked_fill(~seen, 0.0)
            err = err + 2.0 ** -23 * (sc - m).abs().masked_fill(~seen, 0.0)
            # the largest score is off too, and the others are measured from it: of no account, it divides out
            e = ((u + torch.expm1(err)) * p + tiny * seen) / den
            ref[r0:r0 + n, h] = out
            tol[r0:r0 + n, h] = (1.01 * (e @ v.abs() + e.sum(-1, keepdim=True) * out.abs() + (p / den) @ (u * v.abs() + step)) +
                                 HALF[P.type] * out.abs() + TINY[P.type])
    return ref, tol


def quantise(x: np.ndarray):
    """Codes and scales of F32 rows [..., d] by the rule of the Q8_0 caches, each step in F32."""
    b = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    d = np.abs(b).max(-1, keepdims=True) / np.float32(127)
    with np.errstate(divide="ignore"):
        z = b * np.where(d > 0, np.float32(1) / d, np.float32(0))
    low = np.floor(np.abs(z))
    codes = np.sign(z) * (low + (np.abs(z) - low >= 0.5))
    with np.errstate(over="ignore"):                      # scales beyond F16 are infinite
        return codes.astype(np.int8).reshape(x.shape), d[..., 0].astype(np.float16)
