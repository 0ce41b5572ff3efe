"""Packed tokens over a cache in Q8_0 pages (vva_paged_rope_append, vva_paged_attn, vva_paged_read) against plain 64-bit
results, at the lengths and layouts where they can go wrong: no tokens, no keys, one key, tiles and pages that end inside each
other, stale slots, strided pages, long caches, scales that are not finite, captured steps that grow."""
import numpy as np
import pytest

import vva
from paged_q8_util import Q8Pages, attention, parts, quantise, values
from paged_util import HALF, TINY, Pages, check_rows, dtype
from test_gpu_paged import SETS, rope_table

pytestmark = pytest.mark.gpu

H7, H15, H05 = (28, 4, 128), (12, 2, 128), (14, 2, 64)


def run_attn(ctx, P, scale=None, max_new=0, out=None):
    torch = P.torch
    scale = P.d ** -0.5 if scale is None else scale
    out = torch.full_like(P.q, 77.0) if out is None else out
    ctx.paged_attn(P.q, P.k, P.v, P.batch(max_new), scale, out)
    torch.cuda.synchronize()
    ref, tol = attention(P, scale)
    check_rows(out[:P.n_tok], ref[:P.n_tok], tol[:P.n_tok], f"{P.lens[:4]}")
    assert bool((out[P.n_tok:] == 77.0).all()), "rows of no sequence were written"
    return out


# ------------------------------------------------------------------ append

def append(ctx, P, io, q_type=None, pos=None, n_pos=None, scale=1.0):
    """The call on random rows, checked against the 64-bit rotation and rounding; every other slot has to stay as it was."""
    torch, d = P.torch, P.d
    q_type = P.type if q_type is None else q_type
    rng = np.random.default_rng(P.rows)
    mk = lambda H: torch.from_numpy((rng.standard_normal((P.rows, H, d)) * scale).astype(np.float32)).cuda().to(dtype(torch, io))  # noqa: E731
    q, k, v = mk(P.Hq), mk(P.Hkv), mk(P.Hkv)
    n_pos = n_pos or max([1] + [L for _, L in P.lens])
    table = rope_table(ctx, torch, n_pos, d)
    q_out = torch.full((P.rows, P.Hq, d), 77.0, dtype=dtype(torch, q_type), device="cuda")
    place, index = P.places()
    own = [p for p in place if p is not None]
    pg, sl = torch.tensor([p for p, _ in own], dtype=torch.long).cuda(), torch.tensor([x for _, x in own], dtype=torch.long).cuda()
    before = None if P.huge else [r.clone() for r in P.raw]
    ctx.paged_rope_append(q, k, v, table, P.batch(), P.k, P.v, q_out, pos=pos)
    torch.cuda.synchronize()
    at = torch.tensor(index, dtype=torch.long).cuda() if pos is None else pos.long()[:P.n_tok]
    inside = (at >= 0) & (at < n_pos)
    cs = table[at.clamp(0, n_pos - 1)].double()
    c, sn = cs[:, None, :d // 2], cs[:, None, d // 2:]

    def turned(x):
        a, b = x[:P.n_tok].double().split(d // 2, -1)
        mag = torch.cat([a.abs() * c.abs() + b.abs() * sn.abs(), a.abs() * sn.abs() + b.abs() * c.abs()], -1)
        return torch.cat([a * c - b * sn, a * sn + b * c], -1), mag

    qr, qm = turned(q)
    check_rows(q_out[:P.n_tok][inside], qr[inside], HALF[q_type] * qr[inside].abs() * 1.001 + 2.0 ** -23 * qm[inside] + 2.0 ** -25, "q")
    assert bool(torch.isnan(q_out[:P.n_tok][~inside]).all())
    assert bool((q_out[P.n_tok:] == 77.0).all())
    kr, km = turned(k)
    live = torch.tensor([p is not None for p in place], dtype=torch.bool).cuda()
    ok = inside[live]
    codes, scales = parts(P.raw[0], d)
    codes, scales = codes[pg, :, sl].double(), scales[pg, :, :, sl].double()
    y, mag = kr[live], km[live].unflatten(-1, (-1, 32)).amax(-1)
    D = y.unflatten(-1, (-1, 32)).abs().amax(-1) / 127
    # two products and their sum off by 2^-23 of their magnitude, then F32 quotients; the F16 scale rounded once
    assert bool(((scales - D).abs()[ok] <= (HALF[vva.F16] * D + 2.0 ** -25 + 2.0 ** -22 * mag / 127)[ok] * 1.001).all()), "scales of k"
    z = y / D.repeat_interleave(32, -1).clamp(min=1e-300)
    off = 0.5 + 127 * 2.0 ** -21 * (1 + (mag / D.clamp(min=1e-300) / 127)).repeat_interleave(32, -1)
    assert bool(((codes - z).abs()[ok] <= off[ok]).all()), "codes of k"
    assert bool(torch.isnan(scales[~ok]).all()), "k of positions outside the table"
    vc, vs = quantise(v[:P.n_tok][live].float().cpu().numpy())
    codes, scales = parts(P.raw[1], d)
    assert bool((codes[pg, :, sl].cpu() == torch.from_numpy(vc)).all()) and bool((scales[pg, :, :, sl].cpu() == torch.from_numpy(vs)).all())
    if before:
        for raw, b in zip(P.raw, before):
            for x, y in zip(parts(raw, d), parts(b, d)):
                if x.dtype == torch.int8:
                    y[pg, :, sl] = x[pg, :, sl]
                else:
                    y[pg, :, :, sl] = x[pg, :, :, sl]
            assert torch.equal(raw, b), "a slot of no new token was written"
    return q, k, v, q_out


@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("heads,t,page,io", [(H7, vva.F16, 16, vva.F32), (H05, vva.BF16, 32, vva.BF16), (H15, vva.F16, 64, vva.F16),
                                             (H05, vva.F16, 1024, vva.F32)])
def test_append_of_packed_sequences(ctx, torch_gpu, name, heads, t, page, io):
    print(name, heads, t, page, io, flush=True)
    append(ctx, Q8Pages(torch_gpu, SETS[name], *heads, t, page, seed=3, extra_rows=2), io)


def test_append_positions_and_q_types(ctx, torch_gpu):
    torch = torch_gpu
    for q_type in (vva.F32, vva.BF16, vva.F16):
        P = Q8Pages(torch, [(5, 20), (1, 3)], *H05, vva.F16, 16, seed=3, extra_rows=1)
        pos = torch.tensor([7, 0, 99, 100, -1, 2 ** 31 - 1, 5], dtype=torch.int32, device="cuda")
        append(ctx, P, vva.F32, q_type=q_type, pos=pos, n_pos=100)


@pytest.mark.parametrize("scale", [1e-3, 3e4])
@pytest.mark.parametrize("heads", [H7, H05])
def test_append_small_and_large_rows(ctx, torch_gpu, scale, heads):
    append(ctx, Q8Pages(torch_gpu, [(20, 50), (1, 3)], *heads, vva.F16, 16, seed=3, head_major=True), vva.F32, q_type=vva.F32, scale=scale)


def test_append_blocks_of_zeros_and_not_finite(ctx, torch_gpu):
    """Blocks of zeros, of values below the smallest scale, above the largest one, with an infinity, with a NaN."""
    torch = torch_gpu
    P = Q8Pages(torch, [(6, 6)], 2, 1, 128, vva.F16, 16, seed=1)
    v = torch.randn(6, 1, 128, device="cuda")
    v[0, 0, 32:64] = 0.0
    v[1, 0, 64:96] *= 1e-7
    v[2, 0, 0:32] *= 1e9
    v[3, 0, 96:128][5] = float("inf")
    v[4, 0, 0:32][31] = float("nan")
    v[5, 0, 32:64][0] = -float("inf")
    k = torch.zeros(6, 1, 128, device="cuda")
    q = torch.zeros(6, 2, 128, device="cuda")
    ctx.paged_rope_append(q, k, v, rope_table(ctx, torch, 6, 128), P.batch(), P.k, P.v, torch.empty_like(q))
    torch.cuda.synchronize()
    page = int(P.table_host[0, 0])
    (kc, ks), (vc, vs) = [parts(r[page:page + 1], 128) for r in P.raw]
    assert not bool(kc[0, :, :6].any()) and not bool(ks[0, :, :, :6].any())
    bad = torch.zeros(4, 6, dtype=torch.bool)
    for t, b in ((3, 3), (4, 0), (5, 1)):
        bad[b, t] = True
    got = vs[0, 0, :, :6].cpu()
    assert torch.equal(got.isnan(), bad)
    assert float(got[1, 0]) == 0.0 and float(got[2, 1]) == 0.0 and float(got[0, 2]) == float("inf")
    codes = vc[0, 0, :6].cpu().view(6, 4, 32)
    assert bool((codes[bad.t()] == 1).all())
    want, scales = quantise(v.nan_to_num(0, 0, 0).cpu().numpy())
    fine = ~bad.t()
    fine[2, 0] = False                                     # F16 has no such scale
    assert bool((codes[fine] == torch.from_numpy(want).view(6, 4, 32)[fine]).all())
    assert bool((got.t()[fine] == torch.from_numpy(scales).view(6, 4)[fine]).all())


def test_append_drops_tokens_without_a_page(ctx, torch_gpu):
    torch = torch_gpu
    P = Q8Pages(torch, [(3, 20), (2, 35), (3, 2)], *H05, vva.BF16, 16, seed=3)
    for bad in (-1, 10 ** 6, -2 ** 31):
        table = P.table_host.copy()
        table[1, 2] = bad                                   # keys 32 .. of the second sequence: both its new tokens
        P.table = torch.from_numpy(table).cuda()
        before = [r.clone() for r in P.raw]
        rows = [torch.randn(8, h, 64, device="cuda") for h in (14, 2, 2)]
        q_out = torch.empty(8, 14, 64, device="cuda")
        ctx.paged_rope_append(*rows, rope_table(ctx, torch, 40, 64), P.batch(), P.k, P.v, q_out)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(q_out[:5]).all())
        assert bool(torch.isnan(q_out[5]).all()) and bool(torch.isfinite(q_out[6:]).all())   # the third begins before key 0
        own = {(int(table[0, j // 16]), j % 16) for j in range(17, 20)} | {(int(table[2, 0]), j) for j in range(2)}
        for a, b in zip(P.raw, before):
            (ca, _), (cb, _) = parts(a, 64), parts(b, 64)
            assert {tuple(x) for x in (ca != cb).any(-1).any(1).nonzero().tolist()} == own


# -------------------------------------------------------------------- read

def read(ctx, P, k_type, v_type, pages=None, strided=False):
    """The call, checked against the pages' values: scale times code is exact in 64 bits and in F32, then rounded once."""
    torch = P.torch
    outs = []
    for t in (k_type, v_type):
        wide = torch.full((P.rows, P.Hkv + 1, P.d + 16), 77.0, dtype=dtype(torch, t or vva.F32), device="cuda")
        outs.append(None if t is None else wide[:, 1:, 8:8 + P.d] if strided else torch.full((P.rows, P.Hkv, P.d), 77.0, dtype=wide.dtype, device="cuda"))
        outs.append(wide)
    kp, vp = (P.k, P.v) if pages is None else pages
    ctx.paged_read(P.batch(), kp, vp, k=outs[0], v=outs[2])
    torch.cuda.synchronize()
    place, _ = P.places()
    for which, out, wide in ((0, outs[0], outs[1]), (1, outs[2], outs[3])):
        if out is None:
            continue
        for i, p in enumerate(place):
            if p is None:
                assert bool(torch.isnan(out[i]).all()), i
        rows = [i for i, p in enumerate(place) if p is not None]
        pg, sl = torch.tensor([place[i][0] for i in rows], dtype=torch.long).cuda(), torch.tensor([place[i][1] for i in rows], dtype=torch.long).cuda()
        if pages is None:
            codes, scales = parts(P.raw[which], P.d)       # of the rows alone: a pool may be large
            want = codes[pg, :, sl].double() * scales[pg, :, :, sl].double().repeat_interleave(32, -1)
        else:
            want = pages[which][pg, :, sl].double()
        want = want.float().to(out.dtype)
        got = out[rows]
        assert bool(((got == want) | (got.isnan() & want.isnan())).all())
        assert bool((out[P.n_tok:] == 77.0).all()), "rows of no sequence were written"
        if strided:
            wide[:, 1:, 8:8 + P.d] = 77.0
            assert bool((wide == 77.0).all()), "memory beside the rows was written"


@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("heads,page,kt,vt", [(H7, 16, vva.F32, vva.F32), (H05, 32, vva.BF16, vva.F16), (H15, 64, vva.F16, None),
                                              (H05, 1024, None, vva.F32), ((3, 3, 64), 128, vva.BF16, vva.BF16)])
def test_read_of_packed_sequences(ctx, torch_gpu, name, heads, page, kt, vt):
    print(name, heads, page, kt, vt, flush=True)
    read(ctx, Q8Pages(torch_gpu, SETS[name], *heads, vva.F16, page, seed=4, extra_rows=3), kt, vt)


def test_read_strided_rows_and_whole_sequences(ctx, torch_gpu):
    for lens in ([(1, 1)], [(70, 70), (333, 333), (5, 5)], [(1, 40)] * 70 + [(17, 17)]):
        P = Q8Pages(torch_gpu, lens, *H7, vva.F16, 16, seed=4, extra_rows=5, head_major=True)
        read(ctx, P, vva.F32, vva.BF16, strided=True)


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
def test_read_of_16_bit_pages(ctx, torch_gpu, t):
    torch = torch_gpu
    for slot_major in (False, True):
        P = Pages(torch, [(3, 20), (70, 70), (0, 9), (2, 1)], *H05, t, 16, seed=4, extra_rows=2, slot_major=slot_major)
        P.places = Q8Pages.places.__get__(P)
        read(ctx, P, vva.F32, t, pages=(P.k, P.v))
        read(ctx, P, vva.F16 + vva.BF16 - t, None, pages=(P.k, P.v))


def test_read_of_bad_pages_gives_nan(ctx, torch_gpu):
    torch = torch_gpu
    P = Q8Pages(torch, [(40, 40), (20, 35)], *H05, vva.F16, 16, seed=4)
    for bad in (-1, 10 ** 6, -2 ** 31):
        P.table = torch.from_numpy(P.table_host).cuda()
        P.table[1, 1] = bad                                 # keys 16 .. 31 of the second sequence
        k = torch.empty(60, 2, 64, device="cuda")
        ctx.paged_read(P.batch(), P.k, P.v, k=k)
        torch.cuda.synchronize()
        nan = k.isnan().all(-1).all(-1).cpu()
        assert nan.tolist() == [False] * 40 + [16 <= j < 32 for j in range(15, 35)]
        assert not bool(k[~nan.cuda()].isnan().any())


def test_batches_that_point_outside_are_cut(ctx, torch_gpu):
    """Starts past the rows, falling starts, lengths past the table: no row beyond the tensors is touched."""
    torch = torch_gpu
    P = Q8Pages(torch, [(2, 40), (3, 50)], *H05, vva.F16, 16, seed=14)
    ref, tol = attention(P, 0.125)
    for starts, lens, good in [([0, 2, 99], [40, 50], slice(0, 2)), ([0, 2, -5], [40, 50], slice(0, 2)),
                               ([-7, 2, 5], [40, 50], slice(0, 5)), ([0, 2, 5], [40, 2 ** 30], slice(0, 2)),
                               ([0, 2, 5], [-3, 50], slice(2, 5))]:
        P.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        P.kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        out = torch.full((9, 14, 64), 5.0, dtype=P.q.dtype, device="cuda")
        rows = torch.full((2, 9, 2, 64), 5.0, device="cuda")
        ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.125, out[:5])
        ctx.paged_read(P.batch(), P.k, P.v, k=rows[0, :5], v=rows[1, :5])
        torch.cuda.synchronize()
        check_rows(out[good], ref[good], tol[good], f"{starts} {lens}")
        assert bool((out[5:] == 5.0).all()) and bool((rows[:, 5:] == 5.0).all())
    for m in (1, 2, 40):                                    # max_new below what a sequence brings: its later rows are left
        P = Q8Pages(torch, [(2, 40), (50, 60)], *H05, vva.F16, 16, seed=15)
        out = torch.full_like(P.q, 5.0)
        ctx.paged_attn(P.q, P.k, P.v, P.batch(m), 0.125, out)
        torch.cuda.synchronize()
        ref, tol = attention(P, 0.125)
        check_rows(out[:min(m, 2)], ref[:min(m, 2)], tol[:min(m, 2)])
        check_rows(out[2:2 + m], ref[2:2 + m], tol[2:2 + m])
        assert bool((out[2 + m:] == 5.0).all())


# --------------------------------------------------------------- attention

@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("heads,t,page", [(H7, vva.F16, 16), (H05, vva.BF16, 32), (H15, vva.BF16, 64), (H05, vva.F16, 128)])
def test_attention_of_packed_sequences(ctx, torch_gpu, name, heads, t, page):
    print(name, heads, t, page, flush=True)
    run_attn(ctx, Q8Pages(torch_gpu, SETS[name], *heads, t, page, seed=len(name) + page, extra_rows=3))


@pytest.mark.parametrize("Hq,Hkv,d", [(1, 1, 64), (8, 8, 128), (8, 1, 64), (32, 1, 128), (33, 1, 64), (40, 2, 64), (3, 3, 64)])
@pytest.mark.parametrize("lens", [[(1, 77), (1, 300)], [(3, 200), (60, 90)]])
def test_attention_head_layouts(ctx, torch_gpu, Hq, Hkv, d, lens):
    print(Hq, Hkv, lens, flush=True)
    run_attn(ctx, Q8Pages(torch_gpu, lens, Hq, Hkv, d, vva.F16, 16, seed=Hq, extra_rows=1))


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("n,Hq,Hkv,d", [(1, 16, 1, 128), (1, 17, 1, 128), (2, 8, 1, 64), (2, 16, 2, 64), (1, 1, 1, 128), (2, 9, 1, 64),
                                        (4, 8, 1, 128), (16, 2, 2, 64), (32, 3, 3, 128), (17, 1, 1, 64)])
def test_attention_of_one_to_thirty_two_rows(ctx, torch_gpu, n, Hq, Hkv, d, t):
    """Rows of a sequence and kv head on both sides of 16, tiles in one piece and in many."""
    print(n, Hq, Hkv, d, t, flush=True)
    run_attn(ctx, Q8Pages(torch_gpu, [(n, 40), (n, n), (n, 1500), (n, 257), (n, 7001)], Hq, Hkv, d, t, 32, seed=n + Hq, extra_rows=0))


@pytest.mark.parametrize("heads,t", [(H7, vva.BF16), (H05, vva.F16)])
def test_single_tokens_of_many_sequences(ctx, torch_gpu, heads, t):
    """More sequences than lanes of a wave, in one kernel for single tokens."""
    run_attn(ctx, Q8Pages(torch_gpu, [(1, 1 + (97 * i) % 1301) for i in range(130)], *heads, t, 16, seed=7))


@pytest.mark.parametrize("lens,heads,t,page", [
    ([(1, 20011)], H7, vva.F16, 16),
    ([(1, 9000), (1, 40), (2, 6001)], H7, vva.BF16, 1024),
    ([(512, 5000)], H7, vva.F16, 64),
    ([(100, 3000), (1, 12000)], H05, vva.BF16, 16),
])
def test_attention_over_long_caches(ctx, torch_gpu, lens, heads, t, page):
    print(lens, heads, t, page, flush=True)
    run_attn(ctx, Q8Pages(torch_gpu, lens, *heads, t, page, seed=5))


def test_attention_of_the_most_sequences(ctx, torch_gpu):
    rng = np.random.default_rng(3)
    lens = [(int(rng.integers(0, 3)), int(rng.integers(3, 50))) for _ in range(1024)]
    P = Q8Pages(torch_gpu, lens, 4, 2, 64, vva.F16, 16, seed=4)
    run_attn(ctx, P)
    read(ctx, P, vva.F32, vva.F32)
    append(ctx, P, vva.F32)


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("lens", [[(1, 100), (2, 40)], [(50, 130), (1, 10)]])
def test_attention_strided_pages_and_rows(ctx, torch_gpu, t, lens):
    """Pools of a head's pages with gaps between them, q inside wider rows, out rows of a wider buffer."""
    torch = torch_gpu
    P = Q8Pages(torch, lens, *H7, t, 32, seed=9, head_major=True, extra_rows=2)
    wide = torch.zeros(P.rows, 28 + 8, 128, dtype=P.q.dtype, device="cuda")
    wide[:, :28] = P.q
    P.q = wide[:, :28]
    buf = torch.full((P.rows, 30, 128), 77.0, dtype=P.q.dtype, device="cuda")
    run_attn(ctx, P, out=buf[:, 1:29])
    assert bool((buf[:, 0] == 77.0).all()) and bool((buf[:, 29] == 77.0).all())


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("lens", [[(1, 300), (1, 5)], [(90, 200)]])
@pytest.mark.parametrize("scale", [1.0, 1e-3, 6.0])
def test_attention_flat_and_peaked(ctx, torch_gpu, t, lens, scale):
    run_attn(ctx, Q8Pages(torch_gpu, lens, *H05, t, 16, seed=11), scale=scale)


@pytest.mark.parametrize("heads", [H7, H05])
@pytest.mark.parametrize("lens", [[(1, 300)], [(60, 200)]])
@pytest.mark.parametrize("size", [1e-4, 60.0])
def test_attention_sizes_of_values(ctx, torch_gpu, heads, lens, size):
    """Caches and q of values far from 1."""
    run_attn(ctx, Q8Pages(torch_gpu, lens, *heads, vva.F16, 16, seed=12, scale=size), scale=min(1.0, size ** -2) * 0.1)


@pytest.mark.parametrize("lens", [[(1, 200)], [(2, 70), (33, 100)], [(64, 64)]])
def test_rising_scores(ctx, torch_gpu, lens):
    """Each key's score well above all before it: the running maximum moves with every tile."""
    P = Q8Pages(torch_gpu, lens, *H05, vva.F16, 16, seed=2)
    codes, scales = parts(P.raw[0], 64)
    for s, (n, L) in enumerate(lens):
        for j in range(L):
            at = int(P.table_host[s, j // 16])
            codes[at, :, j % 16] = 64
            scales[at, :, :, j % 16] = 0.0003 * (j + 1)
    P.q.fill_(1.0)
    run_attn(ctx, P, scale=0.5)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("lens", [[(4, 70)], [(60, 200)], [(300, 300)]])
@pytest.mark.parametrize("heads", [H05, H15])
def test_value_scale_that_is_not_finite_stays_with_the_rows_that_see_it(ctx, torch_gpu, lens, bad, heads):
    """A block of V of the newest tokens: the tokens before them do not see it, the other dims neither."""
    torch = torch_gpu
    P = Q8Pages(torch, lens, *heads, vva.F16, 16, seed=6)
    n, L = lens[0]
    _, scales = parts(P.raw[1], P.d)
    hit = [L - 1, L - 3]                                   # tokens n - 1 and n - 3
    kept = [scales[int(P.table_host[0, j // 16]), :, 1, j % 16].clone() for j in hit]
    for j in hit:
        scales[int(P.table_host[0, j // 16]), :, 1, j % 16] = bad
    out = torch.empty_like(P.q)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.125, out)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out[:n - 3]).all())
    assert not bool(torch.isfinite(out[n - 3:, :, 32:64]).any())
    keep = [i for i in range(P.d) if not 32 <= i < 64]
    assert bool(torch.isfinite(out[:, :, keep]).all())
    for j, x in zip(hit, kept):
        scales[int(P.table_host[0, j // 16]), :, 1, j % 16] = x
    ref, tol = attention(P, 0.125)
    check_rows(out[:n - 3], ref[:n - 3], tol[:n - 3])
    check_rows(out[:, :, keep], ref[:, :, keep], tol[:, :, keep])


@pytest.mark.parametrize("lens,heads", [([(1, 70), (1, 33), (1, 2000)], H7), ([(4, 70), (2, 1)], H05), ([(4, 40)], H7), ([(60, 200), (1, 75)], H05), ([(300, 310)], H7)])
@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
def test_what_lies_behind_a_sequence_does_not_change_a_bit(ctx, torch_gpu, lens, heads, t):
    """Slots behind the keys: NaN scales, large ones, zeros; and later tokens' values past F16 leave the rows before them."""
    torch = torch_gpu
    P = Q8Pages(torch, lens, *heads, t, 16, seed=5)
    outs = []
    for scale in (float("nan"), 6e4, 0.0, float("inf")):
        for s, (_, L) in enumerate(lens):
            if L % 16:
                for raw in P.raw:
                    parts(raw, P.d)[1][int(P.table_host[s, L // 16]), :, :, L % 16:] = scale
        outs.append(run_attn(ctx, P))
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    n, L = lens[0]
    if n > 1:
        for raw in P.raw:                                  # the last token's own row
            parts(raw, P.d)[1][int(P.table_host[0, (L - 1) // 16]), :, :, (L - 1) % 16] = 6e4
        out = torch.empty_like(P.q)
        ctx.paged_attn(P.q, P.k, P.v, P.batch(), P.d ** -0.5, out)
        torch.cuda.synchronize()
        assert torch.equal(out[:n - 1], outs[0][:n - 1])


@pytest.mark.parametrize("lens", [[(4, 70)], [(60, 200)]])
def test_key_scale_that_is_not_finite_reaches_the_rows_that_see_it(ctx, torch_gpu, lens):
    torch = torch_gpu
    for bad in (float("nan"), float("inf")):
        P = Q8Pages(torch, lens, *H05, vva.F16, 16, seed=6)
        n, L = lens[0]
        ref, tol = attention(P, 0.125)
        codes, scales = parts(P.raw[0], 64)
        codes[int(P.table_host[0, (L - 2) // 16]), :, (L - 2) % 16, :32] = 0     # 0 * inf
        scales[int(P.table_host[0, (L - 2) // 16]), :, 0, (L - 2) % 16] = bad
        out = torch.empty_like(P.q)
        ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.125, out)
        torch.cuda.synchronize()
        check_rows(out[:n - 2], ref[:n - 2], tol[:n - 2])
        assert bool(out[n - 2:].isnan().all())


def test_values_beyond_f16_are_infinite(ctx, torch_gpu):
    """One key whose V block is 127 * 600: infinite in F16, and so for the rows that see it."""
    torch = torch_gpu
    for lens in ([(1, 40)], [(40, 40)]):
        P = Q8Pages(torch, lens, *H05, vva.BF16, 16, seed=6)
        codes, scales = parts(P.raw[1], 64)
        at = int(P.table_host[0, 0])
        codes[at, :, 0, :32] = 127
        scales[at, :, 0, 0] = 600.0
        out = torch.empty_like(P.q)
        ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.125, out)
        torch.cuda.synchronize()
        assert bool((out[:, :, :32] == float("inf")).all()) and bool(torch.isfinite(out[:, :, 32:]).all())


def test_shared_prefix_pages(ctx, torch_gpu):
    torch = torch_gpu
    P = Q8Pages(torch, [(1, 100), (3, 90)], *H15, vva.BF16, 16, seed=8)
    P.table_host[1, :4] = P.table_host[0, :4]
    P.table = torch.from_numpy(P.table_host).cuda()
    run_attn(ctx, P)
    read(ctx, P, vva.F32, vva.F32)


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
@pytest.mark.parametrize("lens", [[(1, 100), (1, 90), (1, 70)], [(40, 100), (50, 90), (2, 70)]])
def test_page_id_outside_the_pool_gives_nan(ctx, torch_gpu, bad, lens):
    torch = torch_gpu
    P = Q8Pages(torch, lens, *H05, vva.F16, 16, seed=13)
    table = P.table_host.copy()
    table[1, 2] = bad
    P.table = torch.from_numpy(table).cuda()
    out = torch.empty_like(P.q)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.125, out)
    torch.cuda.synchronize()
    ref, tol = attention(P, 0.125)
    a, b = int(P.starts[1]), int(P.starts[2])
    check_rows(out[:a], ref[:a], tol[:a])
    check_rows(out[b:], ref[b:], tol[b:])
    assert bool(torch.isnan(out[a:b]).all())


@pytest.mark.parametrize("lens,max_new,pad", [([(1, 100), (40, 300)], 40, 39), ([(0, 0), (3, 70), (64, 64)], 64, 125),
                                              ([(2, 33), (0, 9), (1, 1)], 2, 3), ([(4, 900)], 80, 76)])
@pytest.mark.parametrize("heads", [H7, H05])
def test_batch_padded_to_its_rows(ctx, torch_gpu, lens, max_new, pad, heads):
    P = Q8Pages(torch_gpu, lens, *heads, vva.F16, 16, seed=6, extra_rows=pad)
    assert P.rows == len(lens) * max_new
    run_attn(ctx, P, max_new=max_new)


RAGGED = [(1, (97 * i) % 401) for i in range(100)] + [(90, 500), (0, 9), (40, 77)]


@pytest.mark.parametrize("lens,heads,max_new", [
    (RAGGED, H7, 0), (RAGGED, H05, 0), ([(1, 20000), (2, 7000), (200, 300)], H7, 0), ([(1, 40), (300, 6000), (1, 1)], H05, 0),
    ([(1, 9000), (1, 3), (2, 70)], H7, 40), ([(1, 64 * i + 1) for i in range(30)], H15, 64),
    ([(1, 300), (1, 70), (50, 80), (4, 4)], (300, 300, 64), 0), ([(1, 5000), (40, 900)], (8, 8, 128), 0),
    ([(1, 32 * i) for i in range(1, 9)] + [(33, 33)], H05, 0), ([(2500, 2500)], H05, 0), ([(700, 900), (800, 800), (90, 90)], (32, 1, 64), 0),
    ([(9, 2683)] * 3, H7, 0), ([(64, 4160)], H7, 0), ([(40, 40), (7, 7), (300, 310), (0, 8), (33, 1000)], H15, 0), ([(60, 0), (50, 20)], H7, 0),
])
def test_few_rows_beside_many(ctx, torch_gpu, lens, heads, max_new):
    print(lens[:3], heads, max_new, flush=True)
    P = Q8Pages(torch_gpu, lens, *heads, vva.BF16, 16, seed=len(lens), extra_rows=1)
    out = run_attn(ctx, P, max_new=max_new)
    again = torch_gpu.full_like(P.q, 77.0)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(max_new), P.d ** -0.5, again)
    torch_gpu.cuda.synchronize()
    assert torch_gpu.equal(out, again)


def test_pool_beyond_32_bit_offsets(ctx, torch_gpu):
    """Pools of 5 GiB: the pages at their far end."""
    torch = torch_gpu
    for lens in ([(1, 50), (2, 33)], [(70, 120)]):
        P = Q8Pages(torch, lens, 4, 2, 128, vva.F16, 16, seed=1, n_pages=5 * 2 ** 30 // (2 * 16 * 136))
        assert int(P.table_host[0, 0]) * 2 * 16 * 136 > 2 ** 32
        run_attn(ctx, P)
        append(ctx, P, vva.F32)
        read(ctx, P, vva.F32, vva.F32)
        del P
        torch.cuda.empty_cache()


# ------------------------------------------- together, in graphs, on streams

def test_captured_step_grows_with_its_batch(ctx, torch_gpu):
    """Append, attention and reading back the new rows, captured once, replayed while every sequence grows by a token."""
    torch = torch_gpu
    lens = [(1, 60), (1, 400), (1, 5), (2, 130)]
    P = Q8Pages(torch, lens, *H7, vva.F16, 16, seed=21, width=40, n_pages=60)
    free = sorted(set(range(P.raw[0].shape[0])) - set(int(x) for x in P.table_host.flatten()))
    for s in range(4):                                      # a page to grow into
        P.table_host[s, -(-lens[s][1] // 16)] = free[s]
    P.table = torch.from_numpy(P.table_host).cuda()
    rows = [torch.empty(5, h, 128, device="cuda") for h in (28, 4, 4)]
    rope = rope_table(ctx, torch, 700, 128)
    q_out = torch.empty(5, 28, 128, dtype=torch.float16, device="cuda")
    out = torch.empty_like(q_out)
    back = torch.empty(2, 5, 4, 128, device="cuda")
    batch = P.batch()

    def fill(r):
        for x, seed in zip(rows, (1, 2, 3)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * r + seed)))

    def step():
        ctx.paged_rope_append(*rows, rope, batch, P.k, P.v, q_out)
        ctx.paged_attn(q_out, P.k, P.v, batch, 128 ** -0.5, out)
        ctx.paged_read(batch, P.k, P.v, k=back[0], v=back[1])

    fill(0)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    default = torch.cuda.current_stream()
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream())
            step()
    finally:
        ctx.set_stream(default)
    for r in range(4):
        fill(r)
        out.fill_(float("nan"))
        back.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        P.lens = [(n, L + r) for n, L in lens]
        ref, tol = attention(P, 128 ** -0.5, q=q_out)
        check_rows(out, ref, tol, f"replay {r}")
        codes, scales = quantise(rows[2].cpu().numpy())
        want = codes.astype(np.float64) * np.repeat(scales.astype(np.float64), 32, -1)
        assert np.array_equal(back[1].double().cpu().numpy(), want)
        place, _ = P.places()
        keys = torch.stack([values(P.raw[0][p:p + 1], 128)[0, :, s] for p, s in place])
        assert torch.equal(back[0].double(), keys)
        eager = torch.empty_like(out)
        ctx.paged_attn(q_out, P.k, P.v, batch, 128 ** -0.5, eager)
        torch.cuda.synchronize()
        assert torch.equal(eager, out), r
        P.kv_len += 1                                       # the captured pointers stay


def test_one_captured_call_for_every_kind_of_batch(ctx, torch_gpu):
    """128 token rows for 8 sequences, captured once: prompts, single tokens, both, nothing, whatever the batch says."""
    torch = torch_gpu
    P = Q8Pages(torch, [(0, 1200)] * 8, *H7, vva.BF16, 16, seed=12, extra_rows=128)
    batch = vva.Batch(P.q_start, P.kv_len, P.table, 100)
    out = torch.zeros_like(P.q)
    ctx.paged_attn(P.q, P.k, P.v, batch, 0.09, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    default = torch.cuda.current_stream()
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream())
            ctx.paged_attn(P.q, P.k, P.v, batch, 0.09, out)
    finally:
        ctx.set_stream(default)
    ones = [(1, L) for L in (1200, 1, 64, 700, 33, 1199, 5, 90)]
    for lens in (ones, [(100, 1100)] + ones[:5], [(50, 50), (28, 900)] + [(0, 0)] * 6, [(0, 3)] * 8, ones[:7] + [(0, 0)],
                 [(4, 1000)] * 8, [(5, 600)] * 8, [(99, 99)] + [(1, 1000), (2, 1000)] + [(0, 0)] * 5, ones):
        P.lens = lens + [(0, 0)] * (8 - len(lens))
        P.starts = np.concatenate([[0], np.cumsum([n for n, _ in P.lens])]).astype(np.int32)
        P.n_tok = int(P.starts[-1])
        P.q_start.copy_(torch.from_numpy(P.starts))
        P.kv_len.copy_(torch.tensor([L for _, L in P.lens], dtype=torch.int32))
        out.fill_(77.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        ref, tol = attention(P, 0.09)
        check_rows(out[:P.n_tok], ref[:P.n_tok], tol[:P.n_tok], f"{lens}")
        assert bool((out[P.n_tok:] == 77.0).all())


def test_a_sequence_moves_to_a_resident_cache(ctx, torch_gpu):
    """Prompts appended, read back, uploaded into a resident Q8_0 cache: the same blocks, as each block's largest code is 127."""
    torch = torch_gpu
    P = Q8Pages(torch, [(40, 40), (7, 7)], *H7, vva.F16, 16, seed=3)
    append(ctx, P, vva.F32)
    k, v = (torch.empty(47, 4, 128, device="cuda") for _ in range(2))
    ctx.paged_read(P.batch(), P.k, P.v, k=k, v=v)
    torch.cuda.synchronize()
    kv = vva.KVCache(ctx, 1, 4, 128, 64, 1, vva.Q8_0)
    kv.upload(0, 0, 0, k[:40].cpu().numpy(), v[:40].cpu().numpy())
    place, _ = P.places()
    for raw, pool in zip(kv.download(0, 0, 40), P.raw):
        blocks = torch.from_numpy(raw).view(40, 4, 4, 34)
        codes, scales = (x.cpu() for x in parts(pool, 128))
        pg, sl = torch.tensor([p for p, _ in place[:40]]), torch.tensor([s for _, s in place[:40]])
        assert torch.equal(blocks[..., 2:].contiguous().view(torch.int8).flatten(2), codes[pg, :, sl])
        assert torch.equal(blocks[..., :2].contiguous().view(torch.float16)[..., 0], scales[pg, :, :, sl])
    kv.free()


def test_two_contexts_on_two_streams(torch_gpu):
    torch = torch_gpu
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [vva.Context(0, s) for s in streams]
    sets = [Q8Pages(torch, [(1, 3000), (200, 500)], *H7, vva.F16, 16, seed=i) for i in range(2)]
    outs = [torch.empty_like(P.q) for P in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, P, o in zip(ctxs, sets, outs):
            c.paged_attn(P.q, P.k, P.v, P.batch(), 0.09, o)
    torch.cuda.synchronize()
    for P, o in zip(sets, outs):
        ref, tol = attention(P, 0.09)
        check_rows(o, ref, tol)
    for c in ctxs:
        c.close()


@pytest.mark.parametrize("lens", [[(1, 5000), (1, 70), (3, 900)], [(300, 2500), (1, 900)]])
def test_repeated_calls_give_the_same_bits(ctx, torch_gpu, lens):
    torch = torch_gpu
    P = Q8Pages(torch, lens, *H7, vva.BF16, 16, seed=30)
    outs = []
    for _ in range(6):
        o = torch.empty_like(P.q)
        ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.09, o)
        outs.append(o)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_calls_refuse_tensors_elsewhere(ctx, torch_gpu):
    torch = torch_gpu
    P = Q8Pages(torch, [(1, 20)], *H05, vva.F16, 16, seed=1)
    host = vva.q8_pages(torch.zeros(P.raw[0].shape, dtype=torch.uint8), 64)
    for call in (lambda: ctx.paged_attn(P.q, host, P.v, P.batch(), 0.1, torch.empty_like(P.q)),
                 lambda: ctx.paged_read(P.batch(), P.k, host, k=torch.empty(1, 2, 64, device="cuda")),
                 lambda: ctx.paged_read(P.batch(), P.k, P.v, k=torch.empty(1, 2, 64))):
        with pytest.raises(ValueError):
            call()
