"""vva_add_rms_norm against its definition in 64 bits: every type, odd widths and strides, Q8_0 blocks, aliases."""
import numpy as np
import pytest

import vva
from paged_util import HALF, check_rows, dtype

pytestmark = pytest.mark.gpu


def reference(x, add, w, eps):
    h = x.double() + (0.0 if add is None else add.double())
    return h, h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def close(got, h, y, K, t, what):
    """y: the F32 sum of K squares is within K 2^-24 of itself at most (half of that in its root), five more roundings, one
    rounding to the type; F16 also half its smallest step."""
    tol = y.abs() * (HALF[t] * 1.001 + (K / 2 + 8) * 2.0 ** -24) + (2.0 ** -25 if t == vva.F16 else 1e-38)
    check_rows(got, y, tol, what)


def run(ctx, torch, x, add, w, y_type, eps=1e-6, keep=True):
    y = torch.full(x.shape, 7.0, dtype=dtype(torch, y_type), device="cuda")
    total = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda") if keep else None
    ctx.add_rms_norm(x, w, y, add=add, total=total, eps=eps)
    torch.cuda.synchronize()
    h, ref = reference(x, add, w, eps)
    close(y, h, ref, x.shape[-1], y_type, f"{tuple(x.shape)}")
    if keep:
        t = {torch.float32: vva.F32, torch.float16: vva.F16, torch.bfloat16: vva.BF16}[x.dtype]
        check_rows(total, h, h.abs() * HALF[t] * 1.001 + 2.0 ** -25, "sum")
    return y


@pytest.mark.parametrize("K", [1, 2, 7, 32, 63, 64, 896, 1000, 1023, 1536, 3584, 8192, 8200, 16384])
@pytest.mark.parametrize("xt,at,yt", [(vva.F32, vva.F32, vva.F32), (vva.F32, None, vva.F16), (vva.BF16, vva.BF16, vva.BF16),
                                      (vva.F16, vva.F32, vva.BF16), (vva.F32, vva.BF16, vva.F16)])
def test_norm_types_and_widths(ctx, torch_gpu, K, xt, at, yt):
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(K)
    mk = lambda t: (torch.randn(2, 3, K, generator=gen, device="cuda") * 2).to(dtype(torch, t))  # noqa: E731
    run(ctx, torch, mk(xt), None if at is None else mk(at), torch.randn(K, generator=gen, device="cuda"), yt)


def test_norm_rows_of_many_shapes(ctx, torch_gpu):
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(96, generator=gen, device="cuda")
    for B, T in [(1, 1), (1, 1000), (5, 1), (16, 33), (1, 70000)]:
        run(ctx, torch, torch.randn(B, T, 96, generator=gen, device="cuda"), None, w, vva.F16)


def test_norm_strided_and_unaligned_rows(ctx, torch_gpu):
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(2)
    for dt in (torch.float32, torch.float16):
        for off, K in [(0, 96), (1, 96), (3, 61), (4, 64)]:
            base = torch.randn(2, 5, 200, generator=gen, device="cuda").to(dt)
            x, add = base[:, :, off:off + K], base[:, 1:2, 90 + off:90 + off + K].expand(2, 5, K)
            y = torch.full((2, 5, 201), 7.0, device="cuda")
            w = torch.randn(K + off, generator=gen, device="cuda")[off:]
            ctx.add_rms_norm(x, w, y[:, :, off:off + K], add=add, eps=1e-5)
            torch.cuda.synchronize()
            h, ref = reference(x, add, w, 1e-5)
            close(y[:, :, off:off + K], h, ref, K, vva.F32, f"{off} {K}")
            assert bool((y[:, :, :off] == 7.0).all()) and bool((y[:, :, off + K:] == 7.0).all())


def test_norm_in_place(ctx, torch_gpu):
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, a = (torch.randn(1, 40, 896, generator=gen, device="cuda") for _ in range(2))
    w = torch.randn(896, generator=gen, device="cuda")
    h, ref = reference(x, a, w, 1e-6)
    x1, a1 = x.clone(), a.clone()
    ctx.add_rms_norm(x1, w, a1, add=a1, total=x1)           # the sum over x, the norm over the addend
    torch.cuda.synchronize()
    close(a1, h, ref, 896, vva.F32, "in place")
    check_rows(x1, h, h.abs() * 2.0 ** -24)


@pytest.mark.parametrize("eps", [0.0, 1e-6, 1.0])
def test_norm_small_rows_and_eps(ctx, torch_gpu, eps):
    """Rows of tiny values (eps decides), and rows of zeros: zeros, or NaN where eps is 0, as the definition gives."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randn(256, generator=gen, device="cuda")
    x = torch.randn(1, 4, 256, generator=gen, device="cuda") * 1e-4
    run(ctx, torch, x, None, w, vva.F32, eps=eps)
    y = torch.empty(1, 1, 256, device="cuda")
    ctx.add_rms_norm(torch.zeros(1, 1, 256, device="cuda"), w, y, eps=eps)
    torch.cuda.synchronize()
    assert bool((y == 0).all()) if eps > 0 else bool(y.isnan().all())


def test_norm_not_finite_rows(ctx, torch_gpu):
    """A NaN or an infinity stays in its row."""
    torch = torch_gpu
    x = torch.randn(1, 3, 512, device="cuda")
    x[0, 1, 77] = float("nan")
    w = torch.ones(512, device="cuda")
    y = torch.empty_like(x)
    ctx.add_rms_norm(x, w, y)
    torch.cuda.synchronize()
    assert bool(y[0, 1].isnan().all()) and bool(torch.isfinite(y[0, [0, 2]]).all())
    x[0, 1, 77] = float("inf")
    ctx.add_rms_norm(x, w, y)
    torch.cuda.synchronize()
    assert bool(y[0, 1, 77].isnan()) and bool(torch.isfinite(y[0, [0, 2]]).all())


@pytest.mark.parametrize("K", [32, 96, 896, 3584, 8224])
@pytest.mark.parametrize("xt", [vva.F32, vva.BF16])
def test_norm_to_q8_blocks(ctx, torch_gpu, K, xt):
    """Scales amax / 127 in F16, codes within half a step of the value (and the F32 value's own error)."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(2, 9, K, generator=gen, device="cuda").to(dtype(torch, xt))
    add, w = torch.randn(2, 9, K, generator=gen, device="cuda"), torch.randn(K, generator=gen, device="cuda")
    w[:32] = 0.0                                            # a block of zeros
    raw = torch.full((2, 9, K // 32, 34), 201, dtype=torch.uint8, device="cuda")
    ctx.add_rms_norm(x, w, vva.q8_view(raw), add=add)
    torch.cuda.synchronize()
    _, ref = reference(x, add, w, 1e-6)
    b = ref.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    d = raw[..., :2].contiguous().view(torch.float16).double()
    codes = raw[..., 2:].contiguous().view(torch.int8).double()
    err = (K / 2 + 10) * 2.0 ** -24
    check_rows(d, amax / 127, amax / 127 * (2.0 ** -11 + err) + 2.0 ** -25, "scales")
    step = amax / 127
    check_rows(codes * step, b, step * 0.5 + (amax + b.abs()) * 2 * err, "codes")
    assert bool((codes[..., 0, :] == 0).all())
    assert int(codes.abs().max()) <= 127


def test_norm_q8_strided_rows(ctx, torch_gpu):
    torch = torch_gpu
    raw = torch.full((1, 6, 5, 34), 201, dtype=torch.uint8, device="cuda")
    x, w = torch.randn(1, 6, 96, device="cuda"), torch.ones(96, device="cuda")
    ctx.add_rms_norm(x, w, vva.q8_view(raw[:, :, 1:4]))
    torch.cuda.synchronize()
    assert bool((raw[:, :, [0, 4]] == 201).all())
    dense = torch.empty((1, 6, 3, 34), dtype=torch.uint8, device="cuda")
    ctx.add_rms_norm(x, w, vva.q8_view(dense))
    torch.cuda.synchronize()
    assert torch.equal(raw[:, :, 1:4], dense)


def test_norm_captured(ctx, torch_gpu):
    torch = torch_gpu
    x, a, w = torch.randn(1, 20, 896, device="cuda"), torch.randn(1, 20, 896, device="cuda"), torch.randn(896, device="cuda")
    y = torch.empty(1, 20, 896, dtype=torch.float16, device="cuda")
    ctx.add_rms_norm(x, w, y, add=a)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    default = torch.cuda.current_stream()
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream())
            ctx.add_rms_norm(x, w, y, add=a)
    finally:
        ctx.set_stream(default)
    for r in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(r)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        h, ref = reference(x, a, w, 1e-6)
        close(y, h, ref, 896, vva.F16, f"replay {r}")
