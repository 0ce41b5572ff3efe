"""Few rows over Q8_0 pages with F16 q and results: K and V go into the products with what their rounding to F16 leaves.

scale * code has up to 18 bits, F16 keeps 11.  The pages here hold pairs of values whose F16 parts cancel exactly, so that
what is left of a score or of a result is the rest alone; every value, product and sum is exact in F32 then."""
import numpy as np
import pytest

import vva
from paged_q8_util import Q8Pages, parts
from paged_util import HALF, TINY, check_rows

pytestmark = pytest.mark.gpu

# new tokens of a sequence, query heads, kv heads, head dim: at most 16 rows of a sequence and kv head, then 17 to 32
ROWS = [(1, 1, 1, 128), (1, 14, 2, 64), (1, 28, 4, 128), (16, 2, 2, 64), (1, 16, 1, 128),
        (1, 17, 1, 128), (4, 14, 2, 64), (4, 28, 4, 128), (32, 1, 1, 64), (2, 32, 2, 128)]
# beside a sequence of many rows: the second's are in F16 tiles, only the first is looked at
MIXED = [([(1, 300), (90, 200)], 14, 2, 64), ([(1, 300), (90, 200)], 28, 4, 128), ([(4, 1200), (50, 60)], 14, 2, 64)]


def clear(P, which, s):
    """Zeros in all keys of sequence s; returns set(j, head, block, scale, {dim: code})."""
    codes, scales = parts(P.raw[which], P.d)
    L = P.lens[s][1]
    for j in range(L):
        at, slot = int(P.table_host[s, j // P.page]), j % P.page
        codes[at, :, slot], scales[at, :, :, slot] = 0, 1.0

    def put(j, head, block, scale, values):
        at, slot = int(P.table_host[s, j // P.page]), j % P.page
        row = codes[at, head, slot, 32 * block:32 * block + 32]
        for i, c in values.items():
            row[i] = c
        scales[at, head, block, slot] = scale
    return put


def split(rng):
    """A scale and a code whose product, 17 or 18 bits and odd, F16 cannot hold; the product rounded to F16."""
    scale = float(1024 + 2 * int(rng.integers(0, 512)) + 1) * 2.0 ** -11
    code = int(rng.integers(32, 64)) * 2 + 1
    top = float(np.float16(scale * code))
    assert top != scale * code
    return scale, code, top


def results(P, s, scale, rest):
    """64-bit results of sequence s (on the CPU), and how far a correct one may be off: a probability is rounded to F16 (u, and
    half the smallest step where p_j, whose largest is at least 1, is below the normal range), the scores' scaling, exp2 and the
    quotient are a few 2^-24, the result is rounded once.  rest False: K and V rounded to F16 instead."""
    torch = P.torch
    n, L = P.lens[s]
    r0, G = int(P.starts[s]), P.Hq // P.Hkv
    u, tiny = HALF[vva.F16], TINY[vva.F16]
    seen = torch.arange(L)[None, :] <= (L - n + torch.arange(n))[:, None]
    ref = torch.zeros(n, P.Hq, P.d, dtype=torch.float64)
    tol = torch.zeros_like(ref)
    for h in range(P.Hq):
        k, v = (P.keys(s, w, h // G).cpu() for w in (0, 1))
        if not rest:
            k, v = k.half().double(), v.half().double()
        sc = (P.q[r0:r0 + n, h].double().cpu() @ k.t().contiguous() * scale).masked_fill(~seen, -float("inf"))
        d = sc - sc.amax(-1, keepdim=True)
        p = torch.exp(d)
        den = p.sum(-1, keepdim=True)
        out = (p @ v) / den
        # p of equal scores is a power of two, which F16 holds
        flat = bool((d.masked_fill(~seen, 0.0) == 0).all())
        e = ((0.0 if flat else u + 2.0 ** -21) * p + (0.0 if flat else tiny) * seen) / den
        ref[:, h] = out
        tol[:, h] = 1.01 * (e @ v.abs() + e.sum(-1, keepdim=True) * out.abs()) + (u + 2.0 ** -22) * out.abs() + tiny
    return ref, tol


def check(ctx, P, s, scale, hit):
    """The call's rows of sequence s against their definition; without the rests the result would be off in every head."""
    torch = P.torch
    ref, tol = results(P, s, scale, True)
    plain, _ = results(P, s, scale, False)
    off = (plain - ref).abs() > 2 * tol
    assert bool((off.all() if hit == "all" else off.any(-1).all())), "the pages do not show the rests"
    out = torch.full_like(P.q, 77.0)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), scale, out)
    torch.cuda.synchronize()
    r0, n = int(P.starts[s]), P.lens[s][0]
    check_rows(out[r0:r0 + n].cpu(), ref, tol, f"{P.lens[s]}")


def fill_values(P, s, rng):
    """q of zeros, and V of two keys that every row sees: scale * code, and its F16 value with the other sign."""
    n, L = P.lens[s]
    put = clear(P, 1, s)
    for head in range(P.Hkv):
        for b in range(P.d // 32):
            i, j = rng.choice(L - n + 1, 2, replace=False)
            scale, code, top = split(rng)
            signs = rng.choice([-1, 1], 32)
            put(int(i), head, b, scale, {x: int(code * signs[x]) for x in range(32)})
            put(int(j), head, b, top, {x: int(-signs[x]) for x in range(32)})


def fill_keys(P, s, rng):
    """q of ones, and keys whose scores are the rest of one dim's value: another dim, of another block, takes its F16 part away.
    The rests are a fifth of their largest size at least, of one sign at every second key."""
    n, L = P.lens[s]
    put = clear(P, 0, s)
    for head in range(P.Hkv):
        for j in range(L):
            x, y = rng.choice(P.d // 32, 2, replace=False)
            scale, code, top = split(rng)
            while abs(scale * code - top) < 2.0 ** -7:
                scale, code, top = split(rng)
            sign = 1 if (scale * code > top) == (j % 2 == 0) else -1
            put(j, head, int(x), scale, {int(rng.integers(32)): sign * code})
            put(j, head, int(y), top, {int(rng.integers(32)): -sign})


@pytest.mark.parametrize("n,Hq,Hkv,d", ROWS)
def test_what_f16_leaves_of_values(ctx, torch_gpu, n, Hq, Hkv, d):
    print(n, Hq, Hkv, d, flush=True)
    P = Q8Pages(torch_gpu, [(n, n + 1), (n, n + 39), (n, n + 700)], Hq, Hkv, d, vva.F16, 16, seed=n + Hq)
    P.q.zero_()
    rng = np.random.default_rng(Hq)
    for s in range(3):
        fill_values(P, s, rng)
    for s in range(3):
        check(ctx, P, s, 0.125, "all")


@pytest.mark.parametrize("n,Hq,Hkv,d", ROWS)
def test_what_f16_leaves_of_keys(ctx, torch_gpu, n, Hq, Hkv, d):
    print(n, Hq, Hkv, d, flush=True)
    P = Q8Pages(torch_gpu, [(n, n + 1), (n, n + 39), (n, n + 200)], Hq, Hkv, d, vva.F16, 16, seed=n + Hq)
    P.q.fill_(1.0)
    rng = np.random.default_rng(Hq)
    for s in range(3):
        fill_keys(P, s, rng)
    for s in range(3):
        check(ctx, P, s, 64.0, "any")


@pytest.mark.parametrize("lens,Hq,Hkv,d", MIXED)
def test_what_f16_leaves_beside_many_rows(ctx, torch_gpu, lens, Hq, Hkv, d):
    print(lens, Hq, Hkv, d, flush=True)
    for fill, ones, scale, hit in ((fill_values, 0.0, 0.125, "all"), (fill_keys, 1.0, 64.0, "any")):
        P = Q8Pages(torch_gpu, lens, Hq, Hkv, d, vva.F16, 16, seed=d)
        P.q.fill_(ones)
        fill(P, 0, np.random.default_rng(d))
        check(ctx, P, 0, scale, hit)
