"""A few proposed tokens of each of many sequences over Q8_0 pages: 17 to 32 rows of a sequence and kv head, more sequences
than the workgroups that run at once are cut evenly into."""
import pytest

import vva
from paged_q8_util import Q8Pages
from test_gpu_paged_q8 import run_attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("heads,n", [((14, 2, 64), 4), ((8, 4, 64), 16), ((28, 4, 128), 4)])
def test_proposed_tokens_of_many_sequences(ctx, torch_gpu, heads, n, t):
    print(heads, n, t, flush=True)
    torch = torch_gpu
    P = Q8Pages(torch, [(n, n + (97 * i) % 1301) for i in range(140)], *heads, t, 16, seed=n)
    out = run_attn(ctx, P)
    again = torch.full_like(P.q, 77.0)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), P.d ** -0.5, again)
    torch.cuda.synchronize()
    assert torch.equal(out, again)
