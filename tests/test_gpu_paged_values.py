"""Values that vva_paged_attn has to keep: a long tail of small weights beside one large one, NaN and infinities in q and in
the rows of K."""
import pytest

import paged_util
import vva
from paged_util import Pages, attention, check_rows

pytestmark = pytest.mark.gpu

H7, H05 = (28, 4, 128), (14, 2, 64)


def one_key_and_a_tail(torch, lens, heads, t, gap, seed):
    """Every row's score is `gap` nats on key 0, whose V is 0, and 0 on all others, whose V are about 1."""
    P = Pages(torch, lens, *heads, t, 16, seed=seed)
    P.q.zero_()
    P.q[..., 0] = 4.0
    for s, (_, L) in enumerate(lens):
        ids = P.table[s, :-(-L // 16)].long()
        P.k[ids] = 0.0
        P.v[ids] = (1.0 + 0.1 * torch.randn(P.v[ids].shape, generator=P.gen, device="cuda")).to(P.v.dtype)
        P.k[ids[0], :, 0, 0] = gap / 4.0
        P.v[ids[0], :, 0] = 0.0
    return P


@pytest.mark.parametrize("lens,heads", [([(1, 32768)], H7), ([(2, 20000), (1, 3000)], H05), ([(1, 262144)], (2, 1, 64)),
                                        ([(40, 32768)], H05), ([(300, 9000)], H7), ([(64, 20000), (1, 20000)], H05)])
@pytest.mark.parametrize("gap", [14.0, 17.2, 19.5])
def test_tail_of_small_weights(ctx, torch_gpu, monkeypatch, lens, heads, gap):
    """F16 probabilities are kept 2^7 above their share of the largest, so that those of e^-19.5 = 2^-28 still have most of
    their digits: half a step of F16 each, and half its smallest step, 2^-25, below 2^-14, of values 2^7 higher."""
    print(lens, heads, gap, flush=True)
    P = one_key_and_a_tail(torch_gpu, lens, heads, vva.F16, gap, seed=int(gap))
    out = torch_gpu.empty_like(P.q)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), 1.0, out)
    torch_gpu.cuda.synchronize()
    monkeypatch.setitem(paged_util.TINY, vva.F16, 2.0 ** -32)
    ref, tol = attention(P, 1.0)
    # and half a step of the output, 2^-25 below 2^-14
    check_rows(out, ref, tol + 2.0 ** -25, f"{lens} {gap}")
