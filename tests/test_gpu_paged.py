"""Packed tokens over a cache in pages (vva_paged_rope_append, vva_paged_attn) against plain 64-bit results, at the lengths
and layouts where they can go wrong: no tokens, no keys, one key, tiles and pages that end inside each other, shared prefixes,
stale and NaN slots, strided pages, long caches, captured steps that grow."""
import numpy as np
import pytest

import vva
from paged_util import HALF, Pages, attention, check_rows, dtype

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


SETS = {
    "one_key": [(1, 1)],
    "one_token": [(1, 130)],
    "singles": [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 31), (1, 32), (1, 33), (1, 64), (1, 65), (1, 1000), (1, 257)],
    "no_tokens_and_no_keys": [(0, 40), (1, 0), (3, 0), (0, 0), (2, 90), (5, 2), (0, 7)],
    "few": [(2, 70), (3, 3), (4, 333), (4, 4), (1, 500), (2, 129)],
    "prompts": [(1, 1), (63, 63), (64, 64), (65, 65), (2, 2), (129, 129), (37, 37)],
    "chunks": [(40, 700), (256, 300), (5, 1111)],
    "mixed": [(100, 400), (1, 900), (1, 33), (0, 0), (70, 70), (1, 1), (4, 257)],
}


@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("heads,t,page", [(H7, vva.F16, 16), (H05, vva.BF16, 32), (H15, vva.BF16, 64), (H05, vva.F16, 128)])
def test_attention_of_packed_sequences(ctx, torch_gpu, name, heads, t, page):
    print(name, heads, t, page, flush=True)
    P = Pages(torch_gpu, SETS[name], *heads, t, page, seed=len(name) + page, extra_rows=3)
    run_attn(ctx, P)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (8, 1), (32, 1), (33, 1), (40, 2), (3, 3)])
@pytest.mark.parametrize("lens", [[(1, 77), (1, 300)], [(3, 200), (60, 90)]])
def test_attention_head_layouts(ctx, torch_gpu, Hq, Hkv, lens):
    print(Hq, Hkv, lens, flush=True)
    P = Pages(torch_gpu, lens, Hq, Hkv, 64, vva.F16, 16, seed=Hq, extra_rows=1)
    run_attn(ctx, P)


@pytest.mark.parametrize("lens,heads,t,page", [
    ([(1, 20011)], H7, vva.F16, 16),
    ([(1, 9000), (1, 40), (2, 6001)], H7, vva.BF16, 1024),
    ([(512, 5000)], H7, vva.F16, 64),
    ([(100, 3000), (1, 12000)], H05, vva.BF16, 16),
])
def test_attention_over_long_caches(ctx, torch_gpu, lens, heads, t, page):
    print(lens, heads, t, page, flush=True)
    run_attn(ctx, Pages(torch_gpu, lens, *heads, t, page, seed=5))


def test_attention_of_the_most_sequences(ctx, torch_gpu):
    rng = np.random.default_rng(3)
    lens = [(int(rng.integers(0, 3)), int(rng.integers(3, 50))) for _ in range(1024)]
    run_attn(ctx, Pages(torch_gpu, lens, 4, 2, 64, vva.F16, 16, seed=4))


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("lens", [[(1, 100), (2, 40)], [(50, 130), (1, 10)]])
def test_attention_strided_pages_and_rows(ctx, torch_gpu, t, lens):
    """[page][slot][head][dim] pools, q inside wider rows, out rows of a wider buffer."""
    torch = torch_gpu
    P = Pages(torch, lens, *H7, t, 32, seed=9, slot_major=True, extra_rows=2)
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
    """Scores from all but equal to ones that leave a single key."""
    run_attn(ctx, Pages(torch_gpu, lens, *H05, t, 16, seed=11), scale=scale)


@pytest.mark.parametrize("lens", [[(1, 200)], [(2, 70), (33, 100)], [(64, 64)]])
def test_rising_scores(ctx, torch_gpu, lens):
    """Each key's score well above all before it: the running maximum moves with every tile."""
    torch = torch_gpu
    P = Pages(torch, lens, *H05, vva.F16, 16, seed=2)
    for s, (n, L) in enumerate(lens):
        for j in range(L):
            P.k[int(P.table_host[s, j // 16]), :, j % 16] = 0.02 * (j + 1)
    P.q.fill_(1.0)
    run_attn(ctx, P, scale=0.5)


def test_infinite_value_stays_with_the_rows_that_see_it(ctx, torch_gpu):
    """V of the newest tokens infinite or NaN: the tokens before them do not see it."""
    torch = torch_gpu
    for lens in ([(4, 70)], [(60, 200)], [(300, 300)]):
        for bad in (float("inf"), float("nan"), -float("inf")):
            P = Pages(torch, lens, *H05, vva.F16, 16, seed=6)
            n, L = lens[0]
            hit = [L - 1, L - 3]                           # tokens n - 1 and n - 3
            for j in hit:
                P.v[int(P.table_host[0, j // 16]), :, j % 16, 5] = bad
            out = torch.empty_like(P.q)
            ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.125, out)
            torch.cuda.synchronize()
            seen = out[:, :, 5].float()
            assert bool(torch.isfinite(out[:n - 3]).all()), (lens, bad)
            assert not bool(torch.isfinite(seen[n - 3:]).any()), (lens, bad)
            rest = torch.cat([out[:, :, :5], out[:, :, 6:]], -1)
            assert bool(torch.isfinite(rest).all()), (lens, bad)
            for j in hit:
                P.v[int(P.table_host[0, j // 16]), :, j % 16, 5] = 0.0
            ref, tol = attention(P, 0.125)
            check_rows(out[:n - 3], ref[:n - 3], tol[:n - 3])
            keep = [i for i in range(64) if i != 5]
            check_rows(out[:, :, keep], ref[:, :, keep], tol[:, :, keep])


def test_shared_prefix_pages(ctx, torch_gpu):
    """Two sequences over the same first pages."""
    torch = torch_gpu
    P = Pages(torch, [(1, 100), (3, 90)], *H15, vva.BF16, 16, seed=8)
    P.table_host[1, :4] = P.table_host[0, :4]
    P.table = torch.from_numpy(P.table_host).cuda()
    run_attn(ctx, P)


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
@pytest.mark.parametrize("lens", [[(1, 100), (1, 90), (1, 70)], [(40, 100), (50, 90), (2, 70)]])
def test_page_id_outside_the_pool_gives_nan(ctx, torch_gpu, bad, lens):
    """The sequence that names it answers NaN, the others are as ever."""
    torch = torch_gpu
    P = Pages(torch, lens, *H05, vva.F16, 16, seed=13)
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


def test_batches_that_point_outside_are_cut(ctx, torch_gpu):
    """Starts past the rows, falling starts, lengths past the table: no row beyond the tensors is touched."""
    torch = torch_gpu
    P = Pages(torch, [(2, 40), (3, 50)], *H05, vva.F16, 16, seed=14)
    ref, tol = attention(P, 0.125)
    for starts, lens, good in [([0, 2, 99], [40, 50], slice(0, 2)), ([0, 2, -5], [40, 50], slice(0, 2)),
                               ([-7, 2, 5], [40, 50], slice(0, 5)), ([0, 2, 5], [40, 2 ** 30], slice(0, 2)),
                               ([0, 2, 5], [-3, 50], slice(2, 5))]:
        P.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        P.kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        out = torch.full((9, 14, 64), 5.0, dtype=P.q.dtype, device="cuda")
        ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.125, out[:5])
        torch.cuda.synchronize()
        check_rows(out[good], ref[good], tol[good], f"{starts} {lens}")
        assert bool((out[5:] == 5.0).all())
    # max_new below what a sequence brings: its later rows are left
    P = Pages(torch, [(2, 40), (50, 60)], *H05, vva.F16, 16, seed=15)
    for m in (1, 2, 40):
        out = torch.full_like(P.q, 5.0)
        ctx.paged_attn(P.q, P.k, P.v, P.batch(m), 0.125, out)
        torch.cuda.synchronize()
        ref, tol = attention(P, 0.125)
        check_rows(out[:min(m, 2)], ref[:min(m, 2)], tol[:min(m, 2)])
        check_rows(out[2:2 + m], ref[2:2 + m], tol[2:2 + m])
        assert bool((out[2 + m:] == 5.0).all())


@pytest.mark.parametrize("lens,max_new,pad", [([(1, 100), (40, 300)], 40, 39), ([(0, 0), (3, 70), (64, 64)], 64, 125),
                                              ([(2, 33), (0, 9), (1, 1)], 2, 3), ([(4, 900)], 80, 76)])
@pytest.mark.parametrize("heads", [H7, H05])
def test_batch_padded_to_its_rows(ctx, torch_gpu, lens, max_new, pad, heads):
    """n_seq * max_new rows, of which the sequences fill some: short ones are computed, the rows behind them kept."""
    P = Pages(torch_gpu, lens, *heads, vva.F16, 16, seed=6, extra_rows=pad)
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
    P = Pages(torch_gpu, lens, *heads, vva.BF16, 16, seed=len(lens), extra_rows=1)
    out = run_attn(ctx, P, max_new=max_new)
    again = torch_gpu.full_like(P.q, 77.0)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(max_new), P.d ** -0.5, again)
    torch_gpu.cuda.synchronize()
    assert torch_gpu.equal(out, again)


def test_one_captured_call_for_every_kind_of_batch(ctx, torch_gpu):
    """128 token rows for 8 sequences, captured once: prompts, single tokens, both, nothing, whatever the batch says."""
    torch = torch_gpu
    P = Pages(torch, [(0, 1200)] * 8, *H7, vva.F16, 16, seed=12, extra_rows=128)
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


@pytest.mark.parametrize("heads,t", [(H7, vva.F16), (H05, vva.BF16)])
def test_parts_of_one_projections_rows(ctx, torch_gpu, heads, t):
    """q, k and v as the parts of packed rows, q rotated in place; K and V pages by turns in one pool."""
    torch = torch_gpu
    Hq, Hkv, d = heads
    lens = [(1, 40), (50, 90), (2, 7)]
    P, R = [Pages(torch, lens, *heads, t, 16, seed=8) for _ in range(2)]
    both = torch.stack([P.k, P.v], 1)
    P.k, P.v = both[:, 0], both[:, 1]
    y = torch.randn(P.rows, Hq + 2 * Hkv, d, generator=P.gen, device="cuda").to(dtype(torch, t))
    q, k, v = y.split([Hq, Hkv, Hkv], 1)
    rope = rope_table(ctx, torch, 100, d)
    plain = torch.empty(P.rows, Hq, d, dtype=y.dtype, device="cuda")
    ctx.paged_rope_append(q.contiguous(), k.contiguous(), v.contiguous(), rope, R.batch(), R.k, R.v, plain)
    keep = y[:, Hq:].clone()
    ctx.paged_rope_append(q, k, v, rope, P.batch(), P.k, P.v, q)
    torch.cuda.synchronize()
    assert torch.equal(q, plain) and torch.equal(y[:, Hq:], keep)
    for a, b in ((P.k, R.k), (P.v, R.v)):
        assert bool(((a == b) | (a.isnan() & b.isnan())).all())
    wide = torch.full((P.rows, 2 * Hq, d), 77.0, dtype=y.dtype, device="cuda")
    wide[:, :Hq] = q
    P.q = wide[:, :Hq]
    run_attn(ctx, P, out=wide[:, Hq:])


def test_pool_beyond_32_bit_offsets(ctx, torch_gpu):
    """Pools of 5 GiB: the pages at their far end."""
    torch = torch_gpu
    for lens in ([(1, 50), (2, 33)], [(70, 120)]):
        P = Pages(torch, lens, 4, 2, 128, vva.F16, 16, seed=1, n_pages=5 * 2 ** 30 // (2 * 16 * 128 * 2))
        assert int(P.table_host[0, 0]) * 2 * 16 * 128 * 2 > 2 ** 32
        run_attn(ctx, P)
        append(ctx, P, vva.F32)
        del P
        torch.cuda.empty_cache()


# ------------------------------------------------------------------ append

def rope_table(ctx, torch, n, d, base=1.0e6):
    """The angles of vva_rope_append: vva_rope_ext of rows of d / 2 ones, then zeros."""
    x = torch.zeros(1, n, 1, d, device="cuda")
    x[..., :d // 2] = 1.0
    ctx.rope_ext(x, torch.arange(n, dtype=torch.int32, device="cuda"), base)
    return x.view(n, d)


def append(ctx, P, io, q_type=None, pos=None, n_pos=None):
    """The call on random rows, checked against the 64-bit rotation; every other slot has to stay as it was."""
    torch, d = P.torch, P.d
    q_type = P.type if q_type is None else q_type
    rng = np.random.default_rng(P.rows)
    mk = lambda H: torch.from_numpy(rng.standard_normal((P.rows, H, d)).astype(np.float32)).cuda().to(dtype(torch, io))  # noqa: E731
    q, k, v = mk(P.Hq), mk(P.Hkv), mk(P.Hkv)
    n_pos = n_pos or max([1] + [L for _, L in P.lens])
    table = rope_table(ctx, torch, n_pos, d)
    q_out = torch.full((P.rows, P.Hq, d), 77.0, dtype=dtype(torch, q_type), device="cuda")
    place, index, row = [], [], []
    for s, (n, L) in enumerate(P.lens):
        for t in range(n):
            j = L - n + t
            index.append(j)
            row.append(int(P.starts[s]) + t)
            place.append((int(P.table_host[s, j // P.page]), j % P.page) if j >= 0 else None)
    own = [p for p in place if p is not None]
    pg, sl = torch.tensor([p for p, _ in own]).cuda(), torch.tensor([x for _, x in own]).cuda()
    small = P.k.numel() < 1 << 26
    before = [P.k.clone(), P.v.clone()] if small else None
    ctx.paged_rope_append(q, k, v, table, P.batch(), P.k, P.v, q_out, pos=pos)
    torch.cuda.synchronize()
    at = torch.tensor(index).cuda() if pos is None else pos.long()[:P.n_tok]
    inside = (at >= 0) & (at < n_pos)
    cs = table[at.clamp(0, n_pos - 1)].double()
    c, sn = cs[:, None, :d // 2], cs[:, None, d // 2:]

    def turned(x):
        a, b = x[:P.n_tok].double().split(d // 2, -1)
        # the two products of each half: a c and b s, then a s and b c
        mag = torch.cat([a.abs() * c.abs() + b.abs() * sn.abs(), a.abs() * sn.abs() + b.abs() * c.abs()], -1)
        return torch.cat([a * c - b * sn, a * sn + b * c], -1), mag

    def close(got, ref, mag, t):
        # one rounding to the type, two F32 products and their sum
        check_rows(got, ref, HALF[t] * ref.abs() * 1.001 + 2.0 ** -23 * mag + 2.0 ** -25, "append")

    qr, qm = turned(q)
    close(q_out[:P.n_tok][inside], qr[inside], qm[inside], q_type)
    assert bool(torch.isnan(q_out[:P.n_tok][~inside]).all())
    assert bool((q_out[P.n_tok:] == 77.0).all())
    kr, km = turned(k)
    live = torch.tensor([p is not None for p in place]).cuda()
    ok = inside[live]
    close(P.k[pg, :, sl][ok], kr[live][ok], km[live][ok], P.type)
    assert bool((P.v[pg, :, sl] == v[:P.n_tok][live].to(P.v.dtype)).all())
    if small:
        for pool, b in zip((P.k, P.v), before):
            b[pg, :, sl] = pool[pg, :, sl]
            assert bool(((pool == b) | (pool.isnan() & b.isnan())).all()), "a slot of no new token was written"
    return q, k, v, q_out


@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("heads,t,page,io", [(H7, vva.F16, 16, vva.F32), (H05, vva.BF16, 32, vva.BF16), (H15, vva.F16, 64, vva.F16),
                                             (H05, vva.F16, 1024, vva.F32)])
def test_append_of_packed_sequences(ctx, torch_gpu, name, heads, t, page, io):
    print(name, heads, t, page, io, flush=True)
    append(ctx, Pages(torch_gpu, SETS[name], *heads, t, page, seed=3, extra_rows=2), io)


def test_append_positions_and_q_types(ctx, torch_gpu):
    torch = torch_gpu
    for q_type in (vva.F32, vva.BF16, vva.F16):
        P = Pages(torch, [(5, 20), (1, 3)], *H05, vva.F16, 16, seed=3, extra_rows=1)
        pos = torch.tensor([7, 0, 99, 100, -1, 2 ** 31 - 1, 5], dtype=torch.int32, device="cuda")
        append(ctx, P, vva.F32, q_type=q_type, pos=pos, n_pos=100)


def test_append_equals_the_resident_cache(ctx, torch_gpu):
    """The rows and the rotated q of vva_rope_append, bit for bit, for each type of input."""
    torch = torch_gpu
    for io in (vva.F32, vva.F16, vva.BF16):
        P = Pages(torch, [(40, 40)], *H7, vva.F16, 16, seed=3)
        q, k, v, q_out = append(ctx, P, io)
        kv = vva.KVCache(ctx, 1, 4, 128, 64, 1, vva.F16)
        qr = torch.empty(1, 40, 28, 128, dtype=torch.float16, device="cuda")
        ctx.rope_append(kv, 0, q[None], k[None], v[None], torch.arange(40, dtype=torch.int32, device="cuda"), qr)
        torch.cuda.synchronize()
        for raw, pool in zip(kv.download(0, 0, 40), (P.k, P.v)):
            rows = torch.from_numpy(raw.view(np.float16).reshape(40, 4, 128)).cuda()
            got = torch.cat([pool[int(i)] for i in P.table_host[0, :3]], 1)[:, :40].transpose(0, 1)
            assert torch.equal(rows, got)
        assert torch.equal(qr[0], q_out)
        kv.free()


def test_append_drops_tokens_without_a_page(ctx, torch_gpu):
    torch = torch_gpu
    P = Pages(torch, [(3, 20), (2, 35)], *H05, vva.BF16, 16, seed=3, stale=1.5)
    for bad in (-1, 10 ** 6):
        table = P.table_host.copy()
        table[1, 2] = bad                                   # keys 32 .. of the second sequence: both its new tokens
        P.table = torch.from_numpy(table).cuda()
        kb, vb = P.k.clone(), P.v.clone()
        rows = [torch.randn(5, h, 64, device="cuda") for h in (14, 2, 2)]
        q_out = torch.empty(5, 14, 64, device="cuda")
        ctx.paged_rope_append(*rows, rope_table(ctx, torch, 40, 64), P.batch(), P.k, P.v, q_out)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(q_out).all())
        for a, b in ((P.k, kb), (P.v, vb)):
            rows_changed = (a != b).any(-1).any(1).nonzero().tolist()
            assert all(p == int(table[0, j // 16]) and s == j % 16 for (p, s), j in zip(sorted(rows_changed), range(17, 20))), rows_changed


# --------------------------------------------------------- streams and graphs

def test_captured_step_grows_with_its_batch(ctx, torch_gpu):
    """Append + attention captured once, replayed while every sequence grows by a token; eager work between the replays."""
    torch = torch_gpu
    lens = [(1, 60), (1, 400), (1, 5), (2, 130)]
    P = Pages(torch, lens, *H7, vva.F16, 16, seed=21, stale=0.25, width=40)
    rng = np.random.default_rng(0)
    table = P.table_host.copy()
    n0, more = P.k.shape[0], torch.zeros(4, 4, 16, 128, dtype=P.k.dtype, device="cuda")
    for s in range(4):                                      # a page to grow into
        table[s, -(-lens[s][1] // 16)] = n0 + s
    P.k, P.v = torch.cat([P.k, more]), torch.cat([P.v, more])
    P.table_host, P.table = table, torch.from_numpy(table).cuda()
    rows = [torch.from_numpy(rng.standard_normal((5, h, 128)).astype(np.float32)).cuda() for h in (28, 4, 4)]
    rope = rope_table(ctx, torch, 700, 128)
    q_out = torch.empty(5, 28, 128, dtype=torch.float16, device="cuda")
    out = torch.empty_like(q_out)
    batch = P.batch()

    def step():
        ctx.paged_rope_append(*rows, rope, batch, P.k, P.v, q_out)
        ctx.paged_attn(q_out, P.k, P.v, batch, 128 ** -0.5, out)

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
        for x, seed in zip(rows, (1, 2, 3)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * r + seed)))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        P.lens = [(n, L + r) for n, L in lens]
        ref, tol = attention(P, 128 ** -0.5, q=q_out)
        check_rows(out, ref, tol, f"replay {r}")
        eager = torch.empty_like(out)
        ctx.paged_attn(q_out, P.k, P.v, batch, 128 ** -0.5, eager)
        torch.cuda.synchronize()
        assert torch.equal(eager, out), r
        P.kv_len += 1                                       # the captured pointers stay


def test_two_contexts_on_two_streams(torch_gpu):
    torch = torch_gpu
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [vva.Context(0, s) for s in streams]
    sets = [Pages(torch, [(1, 3000), (200, 500)], *H7, vva.F16, 16, seed=i) for i in range(2)]
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
    P = Pages(torch, lens, *H7, vva.BF16, 16, seed=30)
    outs = []
    for _ in range(6):
        o = torch.empty_like(P.q)
        ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.09, o)
        outs.append(o)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])
