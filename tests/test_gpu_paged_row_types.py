"""Rows of unlike types and of one buffer, appended and read back: what a type by itself gives, bit for bit."""
import itertools

import pytest

import vva
from paged_q8_util import Q8Pages
from paged_util import Pages, dtype
from test_gpu_paged import rope_table

pytestmark = pytest.mark.gpu

TYPES = [vva.F32, vva.F16, vva.BF16]
LENS = [(3, 20), (40, 40), (1, 1), (2, 35)]


def pools(torch, pages, heads, seed):
    """A batch over pools of a page type, their tensors or views, and the bytes that they are."""
    if pages == vva.Q8_0:
        P = Q8Pages(torch, LENS, *heads, vva.F16, 16, seed=seed)
        return P, (P.k, P.v), lambda: [r.clone() for r in P.raw]
    P = Pages(torch, LENS, *heads, pages, 16, seed=seed)
    return P, (P.k, P.v), lambda: [x.view(torch.int16).clone() for x in (P.k, P.v)]


@pytest.mark.parametrize("pages", [vva.F16, vva.BF16, vva.Q8_0])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (3, 3, 64)])
def test_append_of_rows_of_unlike_types(ctx, torch_gpu, pages, heads):
    torch = torch_gpu
    Hq, Hkv, d = heads
    gen = torch.Generator(device="cuda").manual_seed(d)
    rope = rope_table(ctx, torch, 64, d)
    for types in itertools.product(TYPES, repeat=3):
        print(pages, heads, types, flush=True)
        got = []
        rows = [torch.randn(46, h, d, generator=gen, device="cuda").to(dtype(torch, t)) for h, t in zip((Hq, Hkv, Hkv), types)]
        for r in (rows, [x.float() for x in rows]):
            P, (kp, vp), kept = pools(torch, pages, heads, seed=5)
            q_out = torch.empty(46, Hq, d, device="cuda")
            ctx.paged_rope_append(*r, rope, P.batch(), kp, vp, q_out)
            torch.cuda.synchronize()
            got.append([q_out] + kept())
        assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("pages", [vva.F16, vva.BF16, vva.Q8_0])
@pytest.mark.parametrize("io", TYPES)
def test_rows_of_one_projection_in_place(ctx, torch_gpu, pages, io):
    """q, k and v as parts of one buffer's rows, q rotated where it is; k and v read back into such a buffer."""
    torch = torch_gpu
    Hq, Hkv, d = heads = 14, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(46, Hq + 2 * Hkv, d, generator=gen, device="cuda").to(dtype(torch, io))
    q, k, v = wide[:, :Hq], wide[:, Hq:Hq + Hkv], wide[:, Hq + Hkv:]
    rope = rope_table(ctx, torch, 64, d)
    P, (kp, vp), kept = pools(torch, pages, heads, seed=5)
    q_out = torch.empty(46, Hq, d, dtype=wide.dtype, device="cuda")
    ctx.paged_rope_append(q.contiguous(), k.contiguous(), v.contiguous(), rope, P.batch(), kp, vp, q_out)
    torch.cuda.synchronize()
    want = kept()
    P, (kp, vp), kept = pools(torch, pages, heads, seed=5)
    before = wide.clone()
    ctx.paged_rope_append(q, k, v, rope, P.batch(), kp, vp, q)
    torch.cuda.synchronize()
    assert torch.equal(q, q_out) and torch.equal(wide[:, Hq:], before[:, Hq:])
    assert all(torch.equal(a, b) for a, b in zip(kept(), want))
    apart = [torch.empty(46, Hkv, d, dtype=wide.dtype, device="cuda") for _ in range(2)]
    ctx.paged_read(P.batch(), kp, vp, k=apart[0], v=apart[1])
    ctx.paged_read(P.batch(max_new=1), kp, vp, k=k, v=v)           # all tokens, whatever max_new is
    torch.cuda.synchronize()
    assert torch.equal(k, apart[0]) and torch.equal(v, apart[1]) and torch.equal(q, q_out)
    assert not bool(k.isnan().any())
