"""vva.q8_view and the calls bound over it, on the CPU."""
import gc
import weakref
from types import SimpleNamespace

import pytest
import torch

import vva


def blocks(*shape):
    return torch.zeros(*shape, 34, dtype=torch.uint8)


def test_q8_view_keeps_its_blocks():
    """A view, and a bound call that holds nothing else of them, keep the memory that the call will write."""
    raw = blocks(2, 3, 4)
    seen = weakref.ref(raw)
    v = vva.q8_view(raw)
    del raw
    gc.collect()
    assert seen() is not None and v.data == seen().data_ptr()
    call = vva.Context._bound(None, None, (v,), v, 1.0)
    del v
    gc.collect()
    assert seen() is not None
    del call
    gc.collect()
    assert seen() is None


def test_q8_view_shape():
    raw = blocks(2, 3, 7)[:, :, 1:5]
    v = vva.q8_view(raw)
    assert list(v.ne) == [128, 3, 2, 1] and list(v.nb)[:3] == [34, 7 * 34, 3 * 7 * 34]
    assert v.type == vva.Q8_0 and v.data == raw.data_ptr()


@pytest.mark.parametrize("raw", [blocks(2, 3, 4)[:, :, ::2], blocks(2, 3, 4).transpose(2, 3).contiguous().transpose(2, 3),
                                 blocks(2, 3, 4)[..., :33], blocks(3, 4), blocks(2, 3, 4).view(torch.int8),
                                 torch.zeros(2, 3, 4, 17, dtype=torch.float16), blocks(2, 3, 4).expand(2, 3, 4, 34).flip(3)[..., :32]])
def test_q8_view_refuses_other_layouts(raw):
    """Blocks that do not lie one after the other in a row, or are no blocks."""
    with pytest.raises(ValueError):
        vva.q8_view(raw)


def test_bound_calls_refuse_tensors_of_another_device():
    """A tensor in host memory, a batch's among them, is refused by name before the library sees its address."""
    ctx = object.__new__(vva.Context)
    ctx.h, ctx.device = None, 0
    ctx.lib = SimpleNamespace(vva_paged_attn=None, vva_paged_rope_append=None, vva_add_rms_norm=None)
    ints = torch.zeros(4, dtype=torch.int32)
    batch = vva.Batch(ints, ints[:3], torch.zeros(3, 2, dtype=torch.int32), 1)
    q, kv, pool, out = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(2, 2, 16, 64), torch.zeros(3, 4, 64)
    x, w = torch.zeros(1, 3, 64), torch.zeros(64)
    for bind in (lambda: ctx.bind_paged_attn(q, pool, pool, batch, 0.1, out),
                 lambda: ctx.bind_paged_rope_append(q, kv, kv, w.view(1, 64), batch, pool, pool, out),
                 lambda: ctx.bind_add_rms_norm(x, w, x), lambda: ctx.bind_add_rms_norm(x, w, vva.q8_view(blocks(1, 3, 2)))):
        with pytest.raises(ValueError, match="cpu"):
            bind()

    class Here:                                             # a tensor of the device, as far as the check looks
        device = SimpleNamespace(type="cuda", index=0)

    there = SimpleNamespace(device=SimpleNamespace(type="cuda", index=1))
    ctx._here(Here(), None, Here())
    for bad in ((Here(), there), (batch,), (vva.q8_view(blocks(1, 1, 1)),)):
        with pytest.raises(ValueError):
            ctx._here(*bad)
