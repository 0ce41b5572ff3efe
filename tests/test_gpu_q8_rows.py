"""Q8_0 rows between the norm and the projections: values that are not finite, blocks whose largest code is not 127."""
import numpy as np
import pytest

import vva
import vvo

pytestmark = pytest.mark.gpu


def values(torch, raw):
    """Scale times code of uint8 blocks [..., 34], [..., 32] in 32 bits (exact)."""
    return raw[..., :2].contiguous().view(torch.float16).float() * raw[..., 2:].contiguous().view(torch.int8).float()


def norm(ctx, torch, x, w, add=None, eps=1e-6):
    raw = torch.full((*x.shape[:-1], x.shape[-1] // 32, 34), 201, dtype=torch.uint8, device="cuda")
    ctx.add_rms_norm(x, w, vva.q8_view(raw), add=add, eps=eps)
    torch.cuda.synchronize()
    return raw


@pytest.mark.parametrize("K", [32, 512, 3584])
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_norm_blocks_that_are_not_finite(ctx, torch_gpu, K, dt):
    """What the F32 output gives as NaN or infinity the blocks give as NaN, 32 values at a time, and the others as ever."""
    torch = torch_gpu
    x = torch.randn(1, 7, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(K)).to(getattr(torch, dt))
    w = torch.ones(K, device="cuda")
    clean = norm(ctx, torch, x, w)
    x[0, 1, K // 2], x[0, 3, 5], x[0, 4, K - 1] = float("nan"), float("inf"), -float("inf")
    w2 = w.clone()
    raw = norm(ctx, torch, x, w)
    y = torch.empty(1, 7, K, device="cuda")
    ctx.add_rms_norm(x, w, y)
    torch.cuda.synchronize()
    bad = ~torch.isfinite(y.unflatten(-1, (-1, 32))).all(-1)
    assert bool(bad[0, 1].all()) and int(bad[0, 3].sum()) == int(bad[0, 4].sum()) == 1      # inf: 0 times the others
    got = values(torch, raw)
    assert bool(got[bad].isnan().all()) and bool(torch.isfinite(got[~bad]).all())
    assert bool((raw[..., 2:][bad] == 1).all())
    assert torch.equal(raw[0, [0, 2, 5, 6]], clean[0, [0, 2, 5, 6]])
    # a weight that is not finite: its block alone
    w2[K - 1] = float("inf")
    raw = norm(ctx, torch, torch.ones(1, 2, K, device="cuda"), w2)
    got = values(torch, raw)
    assert bool(got[:, :, -1].isnan().all()) and bool(torch.isfinite(got[:, :, :-1]).all())


def test_norm_blocks_of_a_zero_row_without_eps(ctx, torch_gpu):
    """0 / 0: NaN, as in the other types."""
    torch = torch_gpu
    x = torch.zeros(1, 2, 96, device="cuda")
    x[0, 1] = 1.0
    got = values(torch, norm(ctx, torch, x, torch.ones(96, device="cuda"), eps=0.0))
    assert bool(got[0, 0].isnan().all()) and bool((got[0, 1] - 1.0).abs().max() <= 2.0 ** -11)
    got = values(torch, norm(ctx, torch, x, torch.ones(96, device="cuda"), eps=1e-6))
    assert bool((got[0, 0] == 0).all())


def weights(torch, rng, K, rows):
    return [vva.Weight(torch.from_numpy(vvo.from_f32((rng.standard_normal((m, K)) * K ** -0.5).astype(np.float32), vva.Q8_0)).cuda(),
                       vva.Q8_0, K, m) for m in rows]


def project(ctx, torch, x, ws, T, Hq, Hkv, d, ct):
    """q and the cache rows of vva_qkv_rope_append, as arrays."""
    kv = vva.KVCache(ctx, 1, Hkv, d, T, 1, ct)
    q = torch.empty(1, T, Hq, d, device="cuda")
    ctx.qkv_rope_append(kv, 0, x, *ws, torch.arange(T, dtype=torch.int32, device="cuda"), q)
    torch.cuda.synchronize()
    got = [q[0].cpu().numpy()] + [np.asarray(r).reshape(T, -1).copy() for r in kv.download(0, 0, T)]
    kv.free()
    return got


@pytest.mark.parametrize("hidden", [896, 4480])
@pytest.mark.parametrize("T", [1, 3, 8, 9, 40, 1100])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_projections_of_blocks_that_are_not_finite(ctx, torch_gpu, hidden, T, bad):
    """A NaN in a row of the hidden state: the row's q, k and v are NaN, the other rows' the bits they were."""
    torch = torch_gpu
    Hq, Hkv, d = 14, 2, 64
    ws = weights(torch, np.random.default_rng(hidden), hidden, (Hq * d, Hkv * d, Hkv * d))
    x = torch.randn(1, T, hidden, device="cuda", generator=torch.Generator(device="cuda").manual_seed(T))
    w = torch.ones(hidden, device="cuda")
    ref = project(ctx, torch, vva.q8_view(norm(ctx, torch, x, w)), ws, T, Hq, Hkv, d, vva.F32)
    x[0, T // 2, 77] = float(bad)
    raw = norm(ctx, torch, x, w)
    got = project(ctx, torch, vva.q8_view(raw), ws, T, Hq, Hkv, d, vva.F32)
    keep = [t for t in range(T) if t != T // 2]
    for a, b in zip(got, ref):
        a, b = (v.view(np.float32).reshape(T, -1) for v in (a, b))
        assert np.isnan(a[T // 2]).all()
        assert (a[keep].view(np.uint32) == b[keep].view(np.uint32)).all()
    if hidden <= 4096 and T <= 8:
        y = torch.empty(1, T, (Hq + 2 * Hkv) * d, device="cuda")
        ctx.qkv_proj(vva.q8_view(raw), *ws, y)
        torch.cuda.synchronize()
        assert bool(y[0, T // 2].isnan().all()) and bool(torch.isfinite(y[0, keep]).all())


@pytest.mark.parametrize("hidden,T", [(896, 1), (896, 8), (896, 9), (896, 130), (896, 1100), (4480, 3), (3584, 60)])
@pytest.mark.parametrize("kind", ["small", "-128", "random", "tiny"])
def test_projections_of_blocks_no_rounding_made(ctx, torch_gpu, hidden, T, kind):
    """Blocks whose largest code is below 127 or is -128: the bits of F32 rows of their values, at every count of rows."""
    torch = torch_gpu
    Hq, Hkv, d = 14, 2, 64
    rng = np.random.default_rng(T)
    ws = weights(torch, rng, hidden, (Hq * d, Hkv * d, Hkv * d))
    lo, hi = {"small": (-77, 78), "-128": (-128, -127), "random": (-128, 128), "tiny": (-1, 2)}[kind]
    codes = rng.integers(lo, hi, (1, T, hidden // 32, 32)).astype(np.int8)
    if kind == "-128":
        codes[..., 3:9], codes[..., 9] = 50, 100
    scales = (rng.random((1, T, hidden // 32, 1)) * 0.05 + 1e-4).astype(np.float16)
    scales[0, 0, 0] = 0.0
    raw = torch.from_numpy(np.concatenate([scales.view(np.uint8), codes.view(np.uint8)], -1)).cuda()
    rows = values(torch, raw).flatten(2)
    a, b = (project(ctx, torch, x, ws, T, Hq, Hkv, d, vva.F32) for x in (vva.q8_view(raw), rows))
    for x, y in zip(a, b):
        assert (x.view(np.uint8) == y.view(np.uint8)).all()
    if hidden <= 4096 and T <= 8:
        ys = [torch.empty(1, T, (Hq + 2 * Hkv) * d, device="cuda") for _ in range(2)]
        for x, y in zip((vva.q8_view(raw), rows), ys):
            ctx.qkv_proj(x, *ws, y)
        torch.cuda.synchronize()
        assert torch.equal(*ys)
