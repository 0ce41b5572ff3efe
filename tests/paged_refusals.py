"""Layouts that the paged-cache and norm entry points refuse or take, on the CPU (a child program of test_paged_refusals.py, not
a test module), over the stand-in of the HIP runtime that host_routes.py loads.  `python paged_refusals.py NAME` runs one."""
import sys

from host_routes import FAKE, LIB, NO_LIMIT, ref, vva
from paged_routes import INV, Call, change


def layout(c, name, data, strides):
    """Tensor `name` at `data` with these strides of [slot, head, page] or [head, token] in bytes."""
    change(c, name, data=data, nb={i + 1: x for i, x in enumerate(strides)})


def pages_that_meet():
    """K and V pages of one pool: by turns in every order that keeps them apart, and all those that do not."""
    d, ps, H, n, e = 64, 16, 2, 40, 2
    row = d * e
    apart = {
        "page by page": ([row, ps * row, 2 * H * ps * row], H * ps * row),
        "head by head": ([row, 2 * ps * row, 2 * H * ps * row], ps * row),
        "slot by slot": ([2 * row, 2 * ps * row, 2 * H * ps * row], row),
        "heads of a slot": ([2 * H * row, row, 2 * H * ps * row], H * row),
        "heads of a slot by turns": ([2 * H * row, 2 * row, 2 * H * ps * row], row),
        "the pool of V first": ([row, ps * row, H * ps * row], -n * H * ps * row),
        "halves of a page, slots by turns": ([2 * row, 2 * ps * row, 2 * H * ps * row], row),
    }
    for what, (nb, off) in apart.items():
        c = Call()
        at = c.a["k_pages"].data + (1 << 30)
        layout(c, "k_pages", at, nb)
        layout(c, "v_pages", at + off, nb)
        assert c.append() == vva.OK, (what, LIB.vva_last_error(c.c.h))
        for more in (16, row) if off < 0 else (16, -16, row, -row) if off > row else (16, -16):   # further down is free
            layout(c, "v_pages", at + off + more, nb)
            c.refused(c.append, INV, (what, more))
    nb = [row, ps * row, H * ps * row]
    for off in (0, 16, row, 5 * row, ps * row, H * ps * row, (n - 1) * H * ps * row, n * H * ps * row - 16, -row):
        c = Call()
        at = c.a["k_pages"].data + (1 << 30)
        layout(c, "k_pages", at, nb)
        layout(c, "v_pages", at + off, nb)
        c.refused(c.append, INV, off)
        assert c.attn() == vva.OK, (off, LIB.vva_last_error(c.c.h))     # reads them only


SCENARIOS = [pages_that_meet]

if __name__ == "__main__":
    FAKE.fake_set(0, NO_LIMIT)
    {f.__name__: f for f in SCENARIOS}[sys.argv[1]]()
