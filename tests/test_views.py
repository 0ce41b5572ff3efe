"""vva.q8_view and the calls bound over it, on the CPU."""
import gc
import weakref

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
