"""Batches of more than 64 sequences (the kernels look 64 of them up at a time), and tokens beyond
max_new."""
import numpy as np
import pytest

import vva
from paged_util import Pages, attention, check_rows
from test_gpu_paged import append, run_attn

pytestmark = pytest.mark.gpu

H7, H05 = (28, 4, 128), (14, 2, 64)


def ragged(n, new, most, seed):
    """n sequences of 0 to `new` tokens behind up to `most` keys, some of no tokens and some of no keys but their own."""
    rng = np.random.default_rng(seed)
    lens = []
    for s in range(n):
        t = int(rng.integers(0, new + 1))
        lens.append((t, t + (0 if s % 7 == 3 else int(rng.integers(0, most)))))
    return lens


@pytest.mark.parametrize("n", [64, 65, 128, 130, 1024])
@pytest.mark.parametrize("heads,t,io", [(H05, vva.F16, vva.F32), (H7, vva.BF16, vva.BF16)])
def test_append_of_many_sequences(ctx, torch_gpu, n, heads, t, io):
    print(n, heads, flush=True)
    lens = ragged(n, 3, 60, n)
    append(ctx, Pages(torch_gpu, lens, *heads, t, 16, seed=n, extra_rows=2), io)
    lens = [(0, 9)] * (n - 1) + [(5, 30)]                   # the last one alone brings tokens
    append(ctx, Pages(torch_gpu, lens, *heads, t, 16, seed=n, extra_rows=1), io)


@pytest.mark.parametrize("n,long", [(65, 6), (130, 5), (200, 9)])
@pytest.mark.parametrize("heads,t", [(H7, vva.BF16), (H05, vva.F16)])
def test_single_tokens_of_many_sequences(ctx, torch_gpu, n, long, heads, t):
    """Some of thousands of keys, in pieces, on both sides of the 64th; max_new = 1."""
    torch = torch_gpu
    print(n, heads, flush=True)
    rng = np.random.default_rng(n)
    lens = [(1, int(rng.integers(1, 130))) for _ in range(n)]
    for s in list(range(0, n, n // long)) + [63, 64, n - 1]:
        lens[s] = (1, int(rng.integers(3000, 9000)))
    lens[2], lens[n - 2] = (1, 0), (0, 40)
    P = Pages(torch, lens, *heads, t, 128, seed=n, extra_rows=2)
    out = run_attn(ctx, P)
    again = torch.full_like(P.q, 77.0)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), P.d ** -0.5, again)
    torch.cuda.synchronize()
    assert torch.equal(out, again)


@pytest.mark.parametrize("n,new,heads", [(70, 5, H7), (130, 9, H05), (200, 40, (4, 4, 64)), (65, 300, (2, 2, 128))])
def test_as_many_tokens_of_each_of_many_sequences(ctx, torch_gpu, n, new, heads):
    """n_seq * max_new rows: one kernel for all of them, also where the batch then fills fewer."""
    torch = torch_gpu
    print(n, new, heads, flush=True)
    rng = np.random.default_rng(n)
    lens = [(new, new + int(rng.integers(0, 400))) for _ in range(n)]
    lens[66 % n] = (new, new + 3000)
    P = Pages(torch, lens, *heads, vva.BF16, 128, seed=n)
    assert P.rows == n * new
    run_attn(ctx, P)
    lens = [(int(rng.integers(0, new + 1)), L) for _, L in lens]
    lens[0] = (new, lens[0][1])
    filled = sum(t for t, _ in lens)
    run_attn(ctx, Pages(torch, lens, *heads, vva.BF16, 128, seed=n, extra_rows=n * new - filled), max_new=new)


def test_few_beside_many_of_many_sequences(ctx, torch_gpu):
    lens = ragged(150, 1, 900, 5)
    for s in (3, 63, 64, 100, 149):
        lens[s] = (40 + s, 900 + s)
    run_attn(ctx, Pages(torch_gpu, lens, *H7, vva.F16, 64, seed=5, extra_rows=3))


@pytest.mark.parametrize("max_new", [1, 2, 40])
def test_tokens_beyond_max_new(ctx, torch_gpu, max_new):
    """The attention computes a sequence's first max_new tokens; the append takes all of them."""
    torch = torch_gpu
    P = Pages(torch, [(2, 40), (50, 60)], *H05, vva.F16, 16, seed=15, extra_rows=1)
    P.max_new = max_new
    append(ctx, P, vva.F16)
    out = torch.full_like(P.q, 5.0)
    ctx.paged_attn(P.q, P.k, P.v, P.batch(), 0.125, out)
    torch.cuda.synchronize()
    ref, tol = attention(P, 0.125)
    a, b = min(max_new, 2), 2 + max_new
    check_rows(out[:a], ref[:a], tol[:a])
    check_rows(out[2:b], ref[2:b], tol[2:b])
    assert bool((out[a:2] == 5.0).all()) and bool((out[b:] == 5.0).all())
