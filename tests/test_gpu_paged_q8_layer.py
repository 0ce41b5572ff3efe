"""A decoder layer's operators over Q8_0 pages together: vva_add_rms_norm, vva_qkv_proj, vva_paged_rope_append,
vva_paged_attn, vva_out_proj_residual, captured once over a batch that grows; then the sequences read back whole."""
import numpy as np
import pytest

import vva
from paged_q8_util import Q8Pages, attention, parts, quantise, values
from paged_util import HALF, check_rows
from test_gpu_layer_run import rope_table, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden,Hq,Hkv,d", [(896, 14, 2, 64), (1536, 12, 2, 128)])
def test_layers_of_a_growing_batch_captured_once(ctx, torch_gpu, hidden, Hq, Hkv, d):
    """Two layers over 8 token rows: prompts in chunks, single tokens and no tokens; lengths move on the device only."""
    torch = torch_gpu
    rng = np.random.default_rng(6)
    width, n_seq, scale = 8, 3, d ** -0.5
    rows = [Hq * d, Hkv * d, Hkv * d]
    ends = np.cumsum([Hq, Hkv, Hkv])
    new = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731

    class Layer:
        def __init__(self):
            self.w = torch.from_numpy(rng.standard_normal(hidden).astype(np.float32)).cuda()
            self.weights = [weight(torch, rng, m, hidden, vva.Q8_0)[1] for m in rows]
            self.wo, self.w_o = weight(torch, rng, hidden, Hq * d, vva.F16)
            self.P = Q8Pages(torch, [(1, 48)] * n_seq, Hq, Hkv, d, vva.F16, 16, seed=int(rng.integers(99)))
            for r in self.P.raw:                                # nothing in the pages yet
                parts(r, d)[1].fill_(float("nan"))
            self.xn, self.y, self.h = new(1, width, hidden), new(1, width, sum(rows)), new(1, width, hidden)
            self.q, self.o = new(width, Hq, d, dt=torch.float16), new(width, Hq, d, dt=torch.float16)
            self.back = new(2, width, Hkv, d)

    layers = [Layer() for _ in range(2)]
    P0 = layers[0].P
    for L in layers:                                            # one table for all layers
        L.P.table_host, L.P.table = P0.table_host, P0.table
    q_start, kv_len = new(n_seq + 1, dt=torch.int32), new(n_seq, dt=torch.int32)
    batch = vva.Batch(q_start, kv_len, P0.table, width)
    rope = rope_table(ctx, torch, 48, d)
    x = new(1, width, hidden)

    def step():
        src = x
        for L in layers:
            ctx.add_rms_norm(src, L.w, L.xn)
            ctx.qkv_proj(L.xn, *L.weights, L.y)
            heads = L.y.view(width, -1, d)
            ctx.paged_rope_append(heads[:, :ends[0]], heads[:, ends[0]:ends[1]], heads[:, ends[1]:], rope, batch, L.P.k, L.P.v, L.q)
            ctx.paged_attn(L.q, L.P.k, L.P.v, batch, scale, L.o)
            ctx.paged_read(batch, L.P.k, L.P.v, k=L.back[0], v=L.back[1])
            ctx.out_proj_residual(L.o.view(1, width, -1), L.w_o, src, L.h)
            src = L.h

    step()                                                      # no tokens yet; the workspace grows
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    default = torch.cuda.current_stream()
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream())
            step()
    finally:
        ctx.set_stream(default)
    lens = np.zeros(n_seq, np.int64)
    for r, fresh in enumerate([(5, 2, 1), (0, 4, 3), (8, 0, 0), (1, 1, 1), (0, 0, 0), (0, 1, 2), (1, 1, 1), (2, 5, 1)]):
        lens += fresh
        starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
        n = int(starts[-1])
        q_start.copy_(torch.from_numpy(starts))
        kv_len.copy_(torch.from_numpy(lens.astype(np.int32)))
        x.copy_(torch.from_numpy(rng.standard_normal((1, width, hidden)).astype(np.float32)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        src = x
        for i, L in enumerate(layers):
            what = f"step {r} layer {i}"
            L.P.lens, L.P.starts, L.P.rows, L.P.n_tok = [(m, int(ll)) for m, ll in zip(fresh, lens)], starts, width, n
            place, index = L.P.places()
            heads = L.y.view(width, -1, d)[:n]
            if n:
                cs = rope[torch.tensor(index, device="cuda")].double()[:, None]
                c, sn = cs.split(d // 2, -1)
                a, b = heads[:, ends[0]:ends[1]].double().split(d // 2, -1)
                kr = torch.cat([a * c - b * sn, a * sn + b * c], -1)
                big = kr.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
                # half a code, the F16 scale's rounding on every code, the F32 steps of the rotation (two products and a
                # sum) and the quotients
                tol = (big / 254 + (kr.unflatten(-1, (-1, 32)).abs() + big / 254) * HALF[vva.F16] * 1.01 + 127 * 2.0 ** -25 + big * 2.0 ** -20).flatten(-2)
                check_rows(L.back[0, :n], kr, tol, what + " k")
                codes, scales = quantise(heads[:, ends[1]:].cpu().numpy())
                want = codes.astype(np.float64) * np.repeat(scales.astype(np.float64), 32, -1)
                assert np.array_equal(L.back[1, :n].double().cpu().numpy(), want), what
                ref, tol = attention(L.P, scale, q=L.q)
                check_rows(L.o[:n], ref[:n], tol[:n], what + " attention")
            o = L.o.view(1, width, -1).double()
            ref = o @ L.wo.t().contiguous() + src.double()
            mag = o.abs() @ L.wo.abs().t().contiguous() + src.double().abs()
            check_rows(L.h, ref, mag * (Hq * d + 2) * 2.0 ** -24, what + " output")
            src = L.h
        kept = [[t.clone() for t in (L.h, *L.P.raw)] for L in layers]
        step()                                                  # the same step again, not captured: the same bits
        torch.cuda.synchronize()
        for L, k in zip(layers, kept):
            assert all(torch.equal(a, b) for a, b in zip((L.h, *L.P.raw), k)), r
    # every key of every sequence, in one call
    total = int(lens.sum())
    whole = vva.Batch(torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda(), kv_len, P0.table, 1)
    for L in layers:
        k, v = new(total, Hkv, d), new(total, Hkv, d)
        ctx.paged_read(whole, L.P.k, L.P.v, k=k, v=v)
        torch.cuda.synchronize()
        at = [(int(P0.table_host[s, j // 16]), j % 16) for s in range(n_seq) for j in range(int(lens[s]))]
        for rows_back, raw in ((k, L.P.raw[0]), (v, L.P.raw[1])):
            vals = values(raw, d)
            assert torch.equal(rows_back.double(), torch.stack([vals[p, :, s] for p, s in at]))
