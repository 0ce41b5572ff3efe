"""The packed-batch operators together, as a decoder layer uses them: vva_add_rms_norm to Q8_0 rows, vva_qkv_proj,
vva_paged_rope_append, vva_paged_attn, vva_out_proj_residual; and the projections over Q8_0 rows.

Every stage is checked against 64 bits from the values the stage before it left, so each tolerance is one operator's own."""
import numpy as np
import pytest

import vva
import vvo
from paged_util import Pages, attention, check_rows

pytestmark = pytest.mark.gpu


def rope_table(ctx, torch, n, d, base=1.0e6):
    x = torch.zeros(1, n, 1, d, device="cuda")
    x[..., :d // 2] = 1.0
    ctx.rope_ext(x, torch.arange(n, dtype=torch.int32, device="cuda"), base)
    return x.view(n, d)


def weight(torch, rng, M, K, w_type):
    """(64-bit values as the weight's type holds them, Weight)"""
    w = (rng.standard_normal((M, K)) * K ** -0.5).astype(np.float32)
    raw = vvo.from_f32(w, w_type)
    if w_type == vva.F16:
        vals = torch.from_numpy(np.ascontiguousarray(raw).view(np.float16).reshape(M, K).copy()).cuda().double()
    else:
        vals = q8_values(torch, torch.from_numpy(raw).cuda().view(M, K // 32, 34)).flatten(1)
    return vals, vva.Weight(torch.from_numpy(raw).cuda(), w_type, K, M)


def q8_values(torch, raw):
    """Scale times code of uint8 blocks [..., 34], in 64 bits (exact in F32 too)."""
    d = raw[..., :2].contiguous().view(torch.float16).double()
    return d * raw[..., 2:].contiguous().view(torch.int8).double()


class Layer:
    def __init__(self, torch, rng, hidden, Hq, Hkv, d, width, pages):
        self.w = torch.from_numpy(rng.standard_normal(hidden).astype(np.float32)).cuda()
        rows = [Hq * d, Hkv * d, Hkv * d]
        made = [weight(torch, rng, m, hidden, vva.Q8_0) for m in rows]
        self.wv, self.weights = torch.cat([v for v, _ in made]), [w for _, w in made]
        self.b = [torch.from_numpy(rng.standard_normal(m).astype(np.float32) * 0.5).cuda() for m in rows]
        self.wo, self.w_o = weight(torch, rng, hidden, Hq * d, vva.F16)
        self.k, self.v = [torch.full((pages, Hkv, 16, d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]
        new = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
        self.raw, self.y = new(1, width, hidden // 32, 34, dt=torch.uint8), new(1, width, sum(rows))
        self.q, self.o = new(width, Hq, d, dt=torch.float16), new(width, Hq, d, dt=torch.float16)
        self.h = new(1, width, hidden)


def test_steps_of_a_growing_batch_captured_once(ctx, torch_gpu):
    """Two layers over 8 token rows, captured once: replays bring prompts in chunks, single tokens and no tokens, padded rows
    behind the last sequence; lengths move on the device only."""
    torch = torch_gpu
    rng = np.random.default_rng(5)
    hidden, Hq, Hkv, d, width, n_seq = 896, 14, 2, 64, 8, 3
    layers = [Layer(torch, rng, hidden, Hq, Hkv, d, width, 9) for _ in range(2)]
    P = Pages(torch, [(1, 16 * 3)] * n_seq, Hq, Hkv, d, vva.F16, 16, seed=1)
    P.table_host = np.asarray(rng.permutation(9).reshape(3, 3), np.int32)
    table = torch.from_numpy(P.table_host).cuda()
    q_start, kv_len = torch.zeros(n_seq + 1, dtype=torch.int32, device="cuda"), torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    batch = vva.Batch(q_start, kv_len, table, width)
    rope = rope_table(ctx, torch, 48, d)
    x = torch.zeros(1, width, hidden, device="cuda")
    last = torch.zeros_like(x)
    ends = np.cumsum([Hq, Hkv, Hkv])

    def step():
        src = x
        for L in layers:
            ctx.add_rms_norm(src, L.w, vva.q8_view(L.raw))
            ctx.qkv_proj(vva.q8_view(L.raw), *L.weights, L.y, *L.b)
            heads = L.y.view(width, -1, d)
            ctx.paged_rope_append(heads[:, :ends[0]], heads[:, ends[0]:ends[1]], heads[:, ends[1]:], rope, batch, L.k, L.v, L.q)
            ctx.paged_attn(L.q, L.k, L.v, batch, d ** -0.5, L.o)
            ctx.out_proj_residual(L.o.view(1, width, -1), L.w_o, src, L.h)
            src = L.h
        ctx.add_rms_norm(src, layers[0].w, last)

    step()                                                  # no tokens yet; the workspace grows
    torch.cuda.synchronize()
    for L in layers:
        assert bool(L.k.isnan().all()) and bool((L.o == 0).all())
    g = torch.cuda.CUDAGraph()
    default = torch.cuda.current_stream()
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream())
            step()
    finally:
        ctx.set_stream(default)

    lens = np.zeros(n_seq, np.int64)
    for r, new in enumerate([(5, 2, 1), (0, 4, 3), (8, 0, 0), (1, 1, 1), (0, 0, 0), (0, 1, 2), (1, 1, 1), (2, 5, 1)]):
        lens += new
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        n = int(starts[-1])
        q_start.copy_(torch.from_numpy(starts))
        kv_len.copy_(torch.from_numpy(lens.astype(np.int32)))
        x.copy_(torch.from_numpy(rng.standard_normal((1, width, hidden)).astype(np.float32)))
        pools = [(L.k.clone(), L.v.clone()) for L in layers]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()

        index = [int(lens[s]) - new[s] + t for s in range(n_seq) for t in range(new[s])]
        seq = [s for s in range(n_seq) for _ in range(new[s])]
        pg = torch.tensor([int(P.table_host[s, j // 16]) for s, j in zip(seq, index)], dtype=torch.long, device="cuda")
        sl = torch.tensor([j % 16 for j in index], dtype=torch.long, device="cuda")
        cs = rope[torch.tensor(index, dtype=torch.long, device="cuda")].double()[:, None]
        c, sn = cs.split(d // 2, -1)

        def turned(rows):
            a, b = rows.double().split(d // 2, -1)
            return (torch.cat([a * c - b * sn, a * sn + b * c], -1),
                    torch.cat([a.abs() * c.abs() + b.abs() * sn.abs(), a.abs() * sn.abs() + b.abs() * c.abs()], -1))

        src = x
        for i, L in enumerate(layers):
            what = f"step {r} layer {i}"
            xd = src.double()
            ref = xd / (xd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * L.w.double()
            blk = ref.unflatten(-1, (-1, 32))
            amax = blk.abs().amax(-1, keepdim=True)
            # half a step, the scale's F16 rounding on every code, and the F32 value's own error
            rows = q8_values(torch, L.raw)
            check_rows(rows, blk, amax / 254 + (blk.abs() + amax / 254) * 2.0 ** -11 * 1.01 + 2.0 ** -25 * 127 + (amax + blk.abs()) * (hidden + 20) * 2.0 ** -24, what + " norm")
            # integer sums of 32 codes are exact; a block's two scales, the blocks' sum and the bias round in F32
            rows = rows.flatten(2)
            prod = rows @ L.wv.t().contiguous() + torch.cat(L.b).double()
            mag = rows.abs() @ L.wv.abs().t().contiguous() + torch.cat(L.b).abs().double()
            check_rows(L.y, prod, mag * (hidden // 32 + 6) * 2.0 ** -24, what + " projection")
            heads = L.y.view(width, -1, d)[:n]
            kr, km = turned(heads[:, ends[0]:ends[1]])
            qr, qm = turned(heads[:, :ends[0]])
            for got, rr, m in ((L.k[pg, :, sl], kr, km), (L.q[:n], qr, qm)):
                check_rows(got, rr, 2.0 ** -11 * 1.001 * rr.abs() + 2.0 ** -23 * m + 2.0 ** -25, what + " rope")
            assert torch.equal(L.v[pg, :, sl], heads[:, ends[1]:].half()), what
            for pool, before in zip((L.k, L.v), pools[i]):  # the other slots
                before[pg, :, sl] = pool[pg, :, sl]
                assert bool(((pool == before) | (pool.isnan() & before.isnan())).all()), what
            P.k, P.v, P.lens, P.starts, P.rows = L.k, L.v, [(m, int(ll)) for m, ll in zip(new, lens)], starts, width
            ref, tol = attention(P, d ** -0.5, q=L.q)
            check_rows(L.o[:n], ref[:n], tol[:n], what + " attention")
            # o is F16 already: exact products, an F32 sum of Hq d of them and the residual
            o = L.o.view(1, width, -1).double()
            ref = o @ L.wo.t().contiguous() + xd
            mag = o.abs() @ L.wo.abs().t().contiguous() + xd.abs()
            check_rows(L.h, ref, mag * (Hq * d + 2) * 2.0 ** -24, what + " output")
            src = L.h
        xd = src.double()
        ref = xd / (xd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * layers[0].w.double()
        check_rows(last, ref, ref.abs() * (hidden / 2 + 8) * 2.0 ** -24 + 1e-38, f"step {r} last norm")
        kept = [(L.h.clone(), L.k.clone(), L.v.clone()) for L in layers]
        step()                                              # the same step again, not captured: the same bits
        torch.cuda.synchronize()
        for L, (h, k, v) in zip(layers, kept):
            assert torch.equal(L.h, h), r
            for a, b in ((L.k, k), (L.v, v)):
                assert bool(((a == b) | (a.isnan() & b.isnan())).all()), r


# ------------------------------------------------- projections over Q8_0 rows

def q8_rows(ctx, torch, B, T, K, gap=0):
    """(blocks a norm wrote, rows `gap` blocks apart, their F32 values)"""
    x = torch.randn(B, T, K, generator=torch.Generator(device="cuda").manual_seed(K + T), device="cuda")
    x[..., :32] = 0.0                                       # a block of zeros
    raw = torch.zeros((B, T, K // 32 + gap, 34), dtype=torch.uint8, device="cuda")[:, :, :K // 32]
    ctx.add_rms_norm(x, torch.ones(K, device="cuda"), vva.q8_view(raw))
    torch.cuda.synchronize()
    return raw, q8_values(torch, raw).float().flatten(2)


@pytest.mark.parametrize("K,rows,B,T,gap", [(896, (896, 128, 128), 2, 1, 0), (896, (896, 128, 128), 1, 8, 3),
                                            (3584, (3584, 512, 512), 1, 2, 1), (64, (64, 64, 64), 1, 1, 0)])
def test_few_rows_in_blocks(ctx, torch_gpu, K, rows, B, T, gap):
    """The bits of the F32 rows of the same values: quantizing them gives the same scales and codes again."""
    torch = torch_gpu
    rng = np.random.default_rng(K)
    ws = [weight(torch, rng, m, K, vva.Q8_0)[1] for m in rows]
    raw, vals = q8_rows(ctx, torch, B, T, K, gap)
    ys = [torch.full((B, T, sum(rows)), float("nan"), device="cuda") for _ in range(2)]
    for x, y in zip((vva.q8_view(raw), vals), ys):
        ctx.qkv_proj(x, *ws, y)
    torch.cuda.synchronize()
    assert torch.equal(*ys)


@pytest.mark.parametrize("hidden,Hq,Hkv,d,ct,B,T,gap", [
    (896, 14, 2, 64, vva.F16, 2, 1, 1),                     # few rows
    (896, 14, 2, 64, vva.Q8_0, 1, 5, 0),                    # few rows, into a Q8_0 cache
    (896, 14, 2, 64, vva.BF16, 1, 9, 0),
    (3584, 28, 4, 128, vva.Q8_0, 2, 129, 3),
    (1536, 12, 2, 128, vva.F16, 1, 1100, 0),                # weights dequantized ahead
    (4480, 14, 2, 64, vva.F16, 1, 3, 0),                    # wider than the few-row kernel takes
])
def test_appending_projection_of_blocks(ctx, torch_gpu, hidden, Hq, Hkv, d, ct, B, T, gap):
    torch = torch_gpu
    rng = np.random.default_rng(hidden)
    ws = [weight(torch, rng, m * d, hidden, vva.Q8_0)[1] for m in (Hq, Hkv, Hkv)]
    raw, vals = q8_rows(ctx, torch, B, T, hidden, gap)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    got = []
    for x in (vva.q8_view(raw), vals):
        kv = vva.KVCache(ctx, 1, Hkv, d, T, B, ct)
        q = torch.empty(B, T, Hq, d, device="cuda")
        ctx.qkv_rope_append(kv, 0, x, *ws, pos, q)
        torch.cuda.synchronize()
        got.append([q.cpu().numpy()] + [np.asarray(t).copy() for s in range(B) for t in kv.download(0, s, T)])
        kv.free()
    for a, b in zip(*got):
        assert a.tobytes() == b.tobytes()


def test_blocks_captured(ctx, torch_gpu):
    torch = torch_gpu
    rng = np.random.default_rng(9)
    ws = [weight(torch, rng, m, 896, vva.Q8_0)[1] for m in (896, 128, 128)]
    raw, vals = q8_rows(ctx, torch, 1, 4, 896)
    y, ref = [torch.zeros(1, 4, 1152, device="cuda") for _ in range(2)]
    ctx.qkv_proj(vva.q8_view(raw), *ws, y)
    g = torch.cuda.CUDAGraph()
    default = torch.cuda.current_stream()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream())
            ctx.qkv_proj(vva.q8_view(raw), *ws, y)
    finally:
        ctx.set_stream(default)
    for r in range(3):
        raw[..., 2:] = torch.randint(0, 256, raw[..., 2:].shape, device="cuda", dtype=torch.uint8).clamp(max=127)
        raw[..., 2] = 127
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        ctx.qkv_proj(q8_values(torch, raw).float().flatten(2), *ws, ref)
        torch.cuda.synchronize()
        assert torch.equal(y, ref), r
