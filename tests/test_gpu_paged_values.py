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


def call(ctx, P, out=None):
    out = P.torch.full_like(P.q, 77.0) if out is None else out
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), P.d ** -0.5, out)
    P.torch.cuda.synchronize()
    return out


# few rows in one piece and in many (two levels of sums too), many rows in one share and in many, both kinds in a launch
NAN_SETS = [([(4, 40)], H7), ([(4, 3000), (3, 700)], H7), ([(2, 40000)], H05), ([(3, 65)] * 70, H05), ([(90, 90)], H05),
            ([(300, 2500)], H7), ([(256, 9000)], H7), ([(4, 2000), (70, 1500), (1, 900)], H05), ([(2, 9), (33, 64)], H7)]


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("lens,heads", NAN_SETS)
def test_nan_in_a_query_row(ctx, torch_gpu, lens, heads, t):
    """One head of some tokens with a NaN in its q answers NaN; every other row keeps its bits."""
    torch = torch_gpu
    print(lens[:3], heads, t, flush=True)
    P = Pages(torch, lens, *heads, t, 16, seed=3)
    ref = call(ctx, P)
    own = torch.zeros(ref.shape[:2], dtype=torch.bool, device="cuda")
    for n, h in [(int(P.starts[0]), heads[0] - 1), (int(P.starts[0]) + lens[0][0] // 2, 0), (P.n_tok - 1, 3)]:
        P.q[n, h, 7] = float("nan")
        own[n, h] = True
    out = call(ctx, P)
    assert bool(out[own].isnan().all())
    assert torch.equal(out[~own], ref[~own])


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("lens,heads", NAN_SETS)
@pytest.mark.parametrize("back", [1, 2])
def test_nan_in_a_row_of_k(ctx, torch_gpu, lens, heads, t, back):
    """A NaN in the K of a sequence's newest key, or of the one before, for one kv head: that head's rows that see it answer
    NaN, every other row keeps its bits."""
    torch = torch_gpu
    print(lens[:3], heads, t, back, flush=True)
    P = Pages(torch, lens, *heads, t, 16, seed=4)
    ref = call(ctx, P)
    n, L = lens[0]
    j, kvh, G = L - back, heads[1] - 1, heads[0] // heads[1]
    P.k[int(P.table_host[0, j // 16]), kvh, j % 16, 5] = float("nan")
    out = call(ctx, P)
    sees = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
    sees[max(0, n - back):n, kvh * G:] = True
    assert bool(out[sees].isnan().all())
    assert torch.equal(out[~sees], ref[~sees])


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("lens,heads", NAN_SETS)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_infinity_in_a_query_row(ctx, torch_gpu, lens, heads, t, bad):
    """Scores of one sign's infinity by K's: the softmax of such a row is NaN where one is +inf, and where all are -inf, as a
    prompt's first token's only one may be.  Rows whose scores are -inf in part are not made here (no K is 0)."""
    torch = torch_gpu
    print(lens[:3], heads, t, bad, flush=True)
    P = Pages(torch, lens, *heads, t, 16, seed=3)
    ref = call(ctx, P)
    own = torch.zeros(ref.shape[:2], dtype=torch.bool, device="cuda")
    for n, h in [(int(P.starts[0]), heads[0] - 1), (P.n_tok - 1, 3)]:
        P.q[n, h, 7] = bad
        own[n, h] = True
    out = call(ctx, P)
    assert bool(out[own].isnan().all())
    assert torch.equal(out[~own], ref[~own])


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("lens,heads", [([(1, 1)], H7), ([(4, 30)], H7), ([(2, 5000)], H05), ([(60, 90)], H05), ([(300, 2500)], H7),
                                        ([(3, 2), (70, 1500), (1, 900)], H05)])
def test_rows_whose_scores_are_all_minus_infinity(ctx, torch_gpu, lens, heads, t):
    """K of -inf times a q above 0 for every key: NaN, but zeros still where a token sees no key."""
    torch = torch_gpu
    print(lens, heads, t, flush=True)
    P = Pages(torch, lens, *heads, t, 16, seed=5)
    P.q[:, :, 9] = 0.5
    n, L = lens[0]
    for j in range(L):
        P.k[int(P.table_host[0, j // 16]), :, j % 16, 9] = -float("inf")
    out = call(ctx, P)
    none = max(0, n - L)                                    # tokens before key 0
    assert bool((out[:none] == 0).all()) and bool(out[none:n].isnan().all())
    ref, tol = attention(P, P.d ** -0.5)
    check_rows(out[n:P.n_tok], ref[n:P.n_tok], tol[n:P.n_tok])


@pytest.mark.parametrize("lens,heads", [([(4, 3000), (1, 9)], H7), ([(70, 300)], H05)])
def test_keys_of_minus_infinity_are_left_out(ctx, torch_gpu, lens, heads):
    """Some keys' scores -inf, whole tiles of them and the first ones among them: the others' softmax."""
    torch = torch_gpu
    P = Pages(torch, lens, *heads, vva.BF16, 16, seed=5)
    P.q[:, :, 9] = 0.5
    n, L = lens[0]
    gone = list(range(0, 70)) + list(range(128, 192)) + [200, 201]
    for j in gone:
        P.k[int(P.table_host[0, j // 16]), :, j % 16, 9] = -float("inf")
    out = call(ctx, P)
    G, scale = heads[0] // heads[1], P.d ** -0.5
    for h in range(heads[0]):
        k, v = P.keys(0, P.k, h // G), P.keys(0, P.v, h // G)
        q = P.q[:n, h].double()
        sc = (q @ k.t().contiguous()) * scale
        seen = torch.arange(L, device="cuda")[None] <= (L - n + torch.arange(n, device="cuda"))[:, None]
        w = torch.softmax(sc.masked_fill(~seen, -float("inf")), -1)
        mag = (q.abs() @ k.abs().nan_to_num(posinf=0.0).t().contiguous()) * scale
        # as in attention(): half a step of each weight, its score's error, twice for the row sum, and the output's half step
        e = w * (2.0 ** -8 + 2.0 ** -23 * (8 + (P.d + 2) * mag + (sc - sc.amax(-1, keepdim=True)).abs().nan_to_num(posinf=0.0)))
        ref = w @ v
        tol = 1.01 * (e @ v.abs() + e.sum(-1, keepdim=True) * ref.abs()) + 2.0 ** -8 * ref.abs()
        check_rows(out[:n, h], ref, tol)


@pytest.mark.parametrize("lens,heads,scale", [([(1, 130), (2, 40)], H7, 1.0), ([(4, 3001)], H7, 0.5), ([(1, 20000), (3, 77)], H05, 0.2),
                                              ([(2, 700), (90, 200)], H05, 0.3), ([(1, 5)] * 80, H05, 1.0)])
def test_few_rows_keep_the_digits_of_bf16_probabilities(ctx, torch_gpu, monkeypatch, lens, heads, scale):
    """Sequences of at most 32 rows of a kv group: probabilities p in two BF16 parts.  The first is p cut to 8 digits, which
    leaves less than 2^-7 p (and 2^-23 p that is added); the second is that, rounded by 2^-8 of it: together 2^-15 p."""
    torch = torch_gpu
    print(lens[:3], heads, scale, flush=True)
    P = Pages(torch, lens, *heads, vva.BF16, 16, seed=17)
    out = torch.empty_like(P.q)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), scale, out)
    torch.cuda.synchronize()
    last = paged_util.HALF[vva.BF16]
    monkeypatch.setitem(paged_util.HALF, vva.BF16, 2.0 ** -15 * (1 + 2.0 ** -6))
    ref, tol = attention(P, scale)
    for s, (n, _) in enumerate(lens):
        if n * (heads[0] // heads[1]) <= 32:
            r = slice(int(P.starts[s]), int(P.starts[s]) + n)
            # and the output's one rounding
            check_rows(out[r], ref[r], tol[r] + last * (ref[r].abs() + tol[r]), f"sequence {s}")


@pytest.mark.parametrize("t", [vva.F16, vva.BF16])
@pytest.mark.parametrize("lens,heads", NAN_SETS)
def test_infinite_value_gives_its_infinity(ctx, torch_gpu, lens, heads, t):
    """V infinite at a key that every token sees, +inf in some dims and -inf in others: those dims answer with its sign, the
    others keep their bits."""
    torch = torch_gpu
    print(lens[:3], heads, t, flush=True)
    P = Pages(torch, lens, *heads, t, 16, seed=6, scale=0.3)
    ref = call(ctx, P)
    n, L = lens[0]
    for j in {0, (L - n) // 2, max(0, L - n - 1)}:
        row = P.v[int(P.table_host[0, j // 16]), :, j % 16]
        row[:, 3], row[:, 40] = float("inf"), -float("inf")
    out = call(ctx, P)
    assert bool((out[:n, :, 3] == float("inf")).all()) and bool((out[:n, :, 40] == -float("inf")).all())
    keep = [i for i in range(P.d) if i not in (3, 40)]
    assert torch.equal(out[:n][..., keep], ref[:n][..., keep]) and torch.equal(out[n:], ref[n:])
