"""Rows read back out of pages go into pages again, bit for bit: vva_paged_rope_append with one row of the rope table, of
ones, then zeros, for every token (a rotation by nothing)."""
import pytest

import vva
from paged_q8_util import Q8Pages, parts
from paged_util import Pages
from test_gpu_paged_q8 import append

pytestmark = pytest.mark.gpu

H7, H05 = (28, 4, 128), (14, 2, 64)


def restore(ctx, torch, P, k, v):
    """The pages of another batch of these sequences that k and v are appended to; q is scratch."""
    N = P.n_tok
    to = Q8Pages(torch, P.lens, P.Hkv, P.Hkv, P.d, vva.F16, 32, seed=99)
    rope = torch.zeros(1, P.d, device="cuda")
    rope[:, :P.d // 2] = 1.0
    scratch = torch.empty(N, P.Hkv, P.d, dtype=k.dtype, device="cuda")
    ctx.paged_rope_append(k, k, v, rope, to.batch(), to.k, to.v, scratch, pos=torch.zeros(N, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    return to


def rows(P, which):
    """Codes [N, Hkv, d] and scales' bits [N, Hkv, d / 32] of the batch's tokens."""
    torch = P.torch
    place, _ = P.places()
    pg, sl = (torch.tensor(x, dtype=torch.long).cuda() for x in zip(*place))
    codes, scales = parts(P.raw[which], P.d)
    return codes[pg, :, sl], scales[pg, :, :, sl].contiguous().view(torch.int16)


@pytest.mark.parametrize("heads", [H7, H05])
@pytest.mark.parametrize("scale", [1.0, 1e-4, 3e3])
def test_a_parked_request_comes_back(ctx, torch_gpu, heads, scale):
    """The scales are F16's normal numbers, its smallest ones, large ones."""
    torch = torch_gpu
    P = Q8Pages(torch, [(40, 40), (1, 1), (77, 77)], *heads, vva.F16, 16, seed=3)
    append(ctx, P, vva.F32, q_type=vva.F32, scale=scale)
    k, v = (torch.empty(P.n_tok, P.Hkv, P.d, device="cuda") for _ in range(2))
    ctx.paged_read(P.batch(), P.k, P.v, k=k, v=v)
    to = restore(ctx, torch, P, k, v)
    for which in (0, 1):
        for x, y in zip(rows(P, which), rows(to, which)):
            assert torch.equal(x, y)


def test_blocks_of_zeros_and_of_nan_come_back(ctx, torch_gpu):
    """The blocks that the append writes for zeros (codes and scale 0) and for what is not finite (a NaN scale, codes of 1); of
    values below F16's smallest scale zeros are left, and of values above its largest NaN."""
    torch = torch_gpu
    P = Q8Pages(torch, [(5, 5)], *H05, vva.F16, 16, seed=3)
    k, v = (torch.randn(5, 2, 64, generator=P.gen, device="cuda") for _ in range(2))
    v[0, :, :32] = 0.0
    v[1, :, 40] = float("inf")
    v[2, :, 3] = float("nan")
    v[3, :, 32:] *= 1e-7
    v[4, :, :32] *= 1e9
    q = torch.zeros(5, 14, 64, device="cuda")
    rope = torch.zeros(5, 64, device="cuda")
    rope[:, :32] = 1.0
    ctx.paged_rope_append(q, k, v, rope, P.batch(), P.k, P.v, torch.empty_like(q))
    back = [torch.empty(5, 2, 64, device="cuda") for _ in range(2)]
    ctx.paged_read(P.batch(), P.k, P.v, k=back[0], v=back[1])
    to = restore(ctx, torch, P, *back)
    assert all(torch.equal(x, y) for x, y in zip(rows(P, 0), rows(to, 0)))
    (codes, scales), (codes2, scales2) = rows(P, 1), rows(to, 1)
    codes, codes2 = codes.unflatten(-1, (2, 32)), codes2.unflatten(-1, (2, 32))
    same = torch.ones(5, 2, 2, dtype=torch.bool, device="cuda")
    same[3, :, 1] = same[4, :, 0] = False
    assert torch.equal(codes[same], codes2[same]) and torch.equal(scales[same], scales2[same])
    assert bool((scales[3, :, 1] == 0).all()) and bool((codes[3, :, 1] != 0).any())
    assert not bool(codes2[3, :, 1].any()) and not bool(scales2[3, :, 1].any())
    assert bool((scales[4, :, 0] == 0x7c00).all()) and bool((scales2[4, :, 0] == 0x7e00).all()) and bool((codes2[4, :, 0] == 1).all())


def test_16_bit_rows_round_the_values_once_more(ctx, torch_gpu):
    """Rows read as F16 are off by 2^-11, and so is the largest of a block: its scale may round to the next one, and a code's
    quotient is off by 127 * 2^-10 at most, less than a half: the codes stay."""
    torch = torch_gpu
    P = Q8Pages(torch, [(60, 60)], *H05, vva.F16, 16, seed=3)
    append(ctx, P, vva.F32)
    k, v = (torch.empty(60, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.paged_read(P.batch(), P.k, P.v, k=k, v=v)
    to = restore(ctx, torch, P, k, v)
    for which in (0, 1):
        (c, s), (c2, s2) = rows(P, which), rows(to, which)
        assert torch.equal(c, c2) and int((s.int() - s2.int()).abs().max()) <= 1


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
def test_16_bit_pages_come_back(ctx, torch_gpu, t):
    torch = torch_gpu
    lens = [(40, 40), (1, 1), (77, 77)]
    P, to = Pages(torch, lens, *H05, t, 16, seed=3), Pages(torch, lens, 2, 2, 64, t, 32, seed=4)
    k, v = (torch.empty(P.n_tok, 2, 64, dtype=P.q.dtype, device="cuda") for _ in range(2))
    ctx.paged_read(P.batch(), P.k, P.v, k=k, v=v)
    rope = torch.zeros(1, 64, device="cuda")
    rope[:, :32] = 1.0
    pos = torch.zeros(P.n_tok, dtype=torch.int32, device="cuda")
    ctx.paged_rope_append(k, k, v, rope, to.batch(), to.k, to.v, torch.empty_like(k), pos=pos)
    torch.cuda.synchronize()
    for s in range(3):
        for kvh in range(2):
            assert torch.equal(P.keys(s, P.k, kvh), to.keys(s, to.k, kvh)) and torch.equal(P.keys(s, P.v, kvh), to.keys(s, to.v, kvh))
