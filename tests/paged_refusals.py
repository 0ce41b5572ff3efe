"""Layouts that the paged-cache and norm entry points refuse or take, on the CPU (a child program of test_paged_refusals.py, not
a test module), over the stand-in of the HIP runtime that host_routes.py loads.  `python paged_refusals.py NAME` runs one."""
import sys

from host_routes import FAKE, LIB, NO_LIMIT, Host, ref, vva
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


def rows_that_meet_their_own():
    """Outputs whose rows share memory: refused; inputs may (broadcast)."""
    for name, fn in (("q_out", "append"), ("out", "attn")):
        row = 64 * 2
        for nb in ([0, 14 * row], [row, 0], [row, 13 * row], [row - 16, 14 * row], [4 * row, row], [row, row]):
            c = Call()
            layout(c, name, c.a[name].data, nb)
            c.refused(getattr(c, fn), INV, (name, nb))
        for nb in ([row, 14 * row], [row + 16, 16 * row], [5 * row, row]):        # the last: the tokens of a head together
            c = Call()
            layout(c, name, c.a[name].data, nb)
            assert getattr(c, fn)() == vva.OK, (name, nb, LIB.vva_last_error(c.c.h))
    for name in ("k_pages", "v_pages"):
        row, page = 128, 16 * 128
        for nb in ([0, page, 2 * page], [row, 0, 2 * page], [row, page, 0], [row, page, page], [row - 16, page, 2 * page]):
            c = Call()
            layout(c, name, c.a[name].data, nb)
            c.refused(c.append, INV, (name, nb))
            assert c.attn() == vva.OK, (name, nb, LIB.vva_last_error(c.c.h))
    c = Call(N=1, n_seq=1, n_pages=1)                      # strides of dims of one element do not count
    layout(c, "q_out", c.a["q_out"].data, [128, 0])
    layout(c, "k_pages", c.a["k_pages"].data, [128, 16 * 128, 0])
    assert c.append() == vva.OK, LIB.vva_last_error(c.c.h)
    for name in ("q", "k", "v", "rope"):                   # the same rows for every token, or every position
        c = Call()
        change(c, name, nb={1 if name == "rope" else 2: 0})
        assert c.append() == vva.OK, (name, LIB.vva_last_error(c.c.h))


def norm_rows_that_meet_their_own():
    h = Host()
    T = h.tensor

    def norm(x, y, add=None, total=None):
        return LIB.vva_add_rms_norm(h.h, ref(x), ref(add) if add else None, ref(w), 1e-6, ref(total) if total else None, ref(y))

    w = T(vva.F32, [64])
    dense = [T(vva.F32, [64, 5, 2]) for _ in range(3)]
    once = [T(vva.F32, [64, 5, 2], nb=[4, 0, 0, 0]), T(vva.F32, [64, 5, 2], nb=[4, 256, 0, 0]), T(vva.F32, [64, 5, 2], nb=[4, 0, 256, 0]),
            T(vva.F32, [64, 5, 2], nb=[4, 252, 1280, 2560]), T(vva.F32, [64, 5, 2], nb=[4, 256, 1024, 2048])]
    for o in once:
        FAKE.fake_take_log()
        for x, y, add, total in ((dense[0], o, None, None), (dense[0], dense[1], dense[2], o), (dense[0], dense[1], o, o), (o, o, None, None)):
            assert norm(x, y, add, total) == INV, list(o.nb)
        assert not FAKE.fake_take_log()
        assert norm(o, dense[1], dense[0]) == vva.OK and norm(dense[0], dense[1], o, dense[2]) == vva.OK
    q8 = T(vva.Q8_0, [64, 5, 2], nb=[34, 34, 340, 680])
    assert norm(dense[0], q8) == INV
    assert norm(dense[0], T(vva.Q8_0, [64, 5, 2])) == vva.OK
    # rows of the batches by turns
    assert norm(dense[0], T(vva.F32, [64, 5, 2], nb=[4, 512, 256, 4096])) == vva.OK


SCENARIOS = [pages_that_meet, rows_that_meet_their_own, norm_rows_that_meet_their_own]

if __name__ == "__main__":
    FAKE.fake_set(0, NO_LIMIT)
    {f.__name__: f for f in SCENARIOS}[sys.argv[1]]()
