"""Refusals and launches of the entry points over Q8_0 pages, and of reading pages back, on the CPU (a child program of
test_paged_q8_routes.py, not a test module), over the stand-in of the HIP runtime that host_routes.py loads.
`python paged_q8_routes.py NAME` runs one."""
import sys

from host_routes import FAKE, LIB, NO_LIMIT, ref, vva
from paged_routes import INV, NOT, Call, change, log

ROW = 64 // 32 * 34                        # bytes of a row of 64 dims
RUN = 16 * ROW                             # of a page of a head


class Q8Call(Call):
    """A correct call over Q8_0 pages (t: of q_out, q and out); read() too."""

    def __init__(self, N=5, Hkv=2, d=64, page=16, n_pages=40, t=vva.F16, rows=vva.F32, pages=vva.Q8_0, **kw):
        super().__init__(N=N, Hkv=Hkv, d=d, page=page, n_pages=n_pages, t=t, **kw)
        for n in ("k_pages", "v_pages"):
            self.a[n] = self.make(pages, [d, page, Hkv, n_pages])
        self.a["k_rows"], self.a["v_rows"] = (self.make(rows, [d, Hkv, N]) for _ in range(2))

    def read(self, batch=True):
        r = self._ref
        return LIB.vva_paged_read(self.c.h, ref(self.batch()) if batch else None, r("k_pages"), r("v_pages"), r("k_rows"),
                                  r("v_rows"))


CALLS = ("append", "attn", "read")
PAGES = [
    (dict(type=vva.F16), NOT), (dict(type=vva.F32), NOT), (dict(data=None), INV), (dict(nb={0: 2}), INV), (dict(nb={0: 68}), INV),
    (dict(nb={1: ROW + 2}), INV), (dict(nb={1: 64}), INV), (dict(nb={2: RUN + 8}), INV), (dict(nb={3: 2 * RUN + 4}), INV),
    (dict(shift=8), INV), (dict(shift=2), INV), (dict(ne={3: 0}), INV), (dict(ne={1: 32}), INV), (dict(ne={0: 128}), INV),
]
BATCH = [
    ("kv_len", dict(ne={0: 0}), INV), ("kv_len", dict(ne={0: 1025}), INV), ("kv_len", dict(type=vva.F32), INV),
    ("kv_len", dict(data=None), INV), ("q_start", dict(ne={0: 3}), INV), ("q_start", dict(data=None), INV),
    ("table", dict(ne={1: 4}), INV), ("table", dict(type=vva.F16), INV), ("table", dict(nb={1: 30}), INV),
    ("table", dict(ne={0: 1 << 27}), NOT),
]
ROWS = [
    (dict(type=vva.I32), INV), (dict(type=vva.Q8_0), INV), (dict(ne={0: 32}), INV), (dict(ne={1: 3}), INV), (dict(ne={2: 4}), INV),
    (dict(ne={3: 2}), INV), (dict(nb={0: 8}), INV), (dict(nb={1: 264}), INV), (dict(nb={2: 520}), INV), (dict(shift=4), INV),
    (dict(nb={1: 0}), INV), (dict(nb={2: 256}), INV), (dict(data=None), INV),
]


def refusals():
    for name in CALLS:
        for pages in ("k_pages", "v_pages"):
            for kw, status in PAGES:
                c = Q8Call()
                change(c, pages, **kw)
                c.refused(getattr(c, name), status, (name, pages, kw))
        for tensor, kw, status in BATCH:
            c = Q8Call()
            change(c, tensor, **kw)
            c.refused(getattr(c, name), status, (name, tensor, kw))
        for d, page in ((32, 16), (96, 16), (256, 16), (64, 8), (64, 24), (64, 2048)):
            c = Q8Call(d=d, page=page)
            c.refused(getattr(c, name), NOT, (name, d, page))
        for d in (48, 8):                                  # no whole blocks
            c = Q8Call(d=d)
            c.refused(getattr(c, name), INV, (name, d))
        c = Q8Call()
        c.refused(lambda: getattr(c, name)(batch=False), INV, "no batch")
        c = Q8Call()
        c.a["max_new"] = 0
        c.refused(getattr(c, name), INV, (name, "max_new"))
    for t in (vva.F32, vva.Q8_0):                          # what the attention takes and gives
        c = Q8Call(t=t)
        c.refused(c.attn, INV, t)
    for name, t in (("qa", vva.BF16), ("out", vva.BF16), ("out", vva.F32)):
        c = Q8Call()
        change(c, name, type=t)
        c.refused(c.attn, INV, (name, t))
    for rows in ("k_rows", "v_rows"):
        for kw, status in ROWS:
            c = Q8Call()
            change(c, rows, **kw)
            c.refused(c.read, status, (rows, kw))
    c = Q8Call()
    c.a["k_rows"] = c.a["v_rows"] = None
    c.refused(c.read, INV, "nothing to read")
    assert LIB.vva_paged_read(None, None, None, None, None, None) == INV


def accepted():
    for kw in (dict(), dict(N=1, n_seq=1, n_pages=1, max_pages=1), dict(t=vva.BF16, io=vva.F16, Hq=28, Hkv=4, d=128, page=1024),
               dict(N=3, n_seq=1024), dict(N=70000, n_seq=2), dict(Hq=33, Hkv=1), dict(rows=vva.BF16), dict(pages=vva.F16),
               dict(pages=vva.BF16, t=vva.BF16, rows=vva.F16)):
        for name in CALLS:
            c = Q8Call(**kw)
            log()
            assert getattr(c, name)() == vva.OK, (name, kw, LIB.vva_last_error(c.c.h))
            lines = [x for x in log() if x.startswith("kernel")]
            assert len(lines) == 1 and lines[0].startswith("kernel paged"), lines
    for keep in ("k_rows", "v_rows"):
        c = Q8Call()
        c.a["v_rows" if keep == "k_rows" else "k_rows"] = None
        assert c.read() == vva.OK
    c = Q8Call()                                           # k and v of two types
    c.a["v_rows"] = c.make(vva.BF16, [64, 2, 5])
    assert c.read() == vva.OK


def layouts():
    """Runs of K and V by turns and further apart; runs, and rows read back, that share memory."""
    n = 40
    for what, (nb, off) in {"page by page": ([RUN, 4 * RUN], 2 * RUN), "head by head": ([2 * RUN, 4 * RUN], RUN),
                            "page by page of a head": ([n * RUN, RUN], 2 * n * RUN), "wide": ([RUN + 32, 2 * RUN + 256], 1 << 28)}.items():
        c = Q8Call()
        change(c, "k_pages", nb={2: nb[0], 3: nb[1]})
        change(c, "v_pages", data=c.a["k_pages"].data + off, nb={2: nb[0], 3: nb[1]})
        for name in CALLS:
            assert getattr(c, name)() == vva.OK, (what, name, LIB.vva_last_error(c.c.h))
        if off < 1 << 28:
            for more in (-16,) if off == 2 * n * RUN else (16, -16):   # a pool further up is free
                change(c, "v_pages", data=c.a["k_pages"].data + off + more)
                c.refused(c.append, INV, (what, more))
                assert c.attn() == vva.OK and c.read() == vva.OK   # read them only
    for nb in ({2: 0}, {3: 0}, {3: RUN}, {2: RUN - 16}):
        c = Q8Call()
        change(c, "v_pages", nb=nb)
        c.refused(c.append, INV, nb)
        assert c.attn() == vva.OK and c.read() == vva.OK
    for a in ("k_rows", "v_rows"):
        for b in ("k_pages", "v_pages", "q_start", "kv_len", "table"):
            c = Q8Call()
            change(c, a, data=c.a[b].data - c.a[b].data % 16)
            c.refused(c.read, INV, (a, b))
    c = Q8Call()
    change(c, "v_rows", data=c.a["k_rows"].data + 256)
    c.refused(c.read, INV, "k over v")
    change(c, "k_rows", nb={1: 512, 2: 1024})              # heads by turns
    change(c, "v_rows", nb={1: 512, 2: 1024})
    assert c.read() == vva.OK, LIB.vva_last_error(c.c.h)
    for name in ("out", "q_out"):
        c = Q8Call()
        change(c, name, data=c.a["k_pages"].data)
        c.refused(c.attn if name == "out" else c.append, INV, name)


def limits():
    for kw, ok in ((dict(Hq=256, Hkv=1, N=1), True), (dict(Hq=257, Hkv=1, N=1), False), (dict(Hq=1, Hkv=1, N=1 << 22), True),
                   (dict(Hq=1, Hkv=1, N=(1 << 22) + 1), False), (dict(Hq=63, Hkv=63, N=1, n_seq=1024), True),
                   (dict(Hq=64, Hkv=64, N=1, n_seq=1024), False), (dict(n_seq=1, max_pages=(1 << 30) // 16 + 1), False)):
        for name in CALLS:
            if name == "read" and kw.get("Hq") in (256, 257):
                continue
            c = Q8Call(**kw)
            if ok:
                assert getattr(c, name)() == vva.OK, (name, kw, LIB.vva_last_error(c.c.h))
            else:
                c.refused(getattr(c, name), NOT, (name, kw))
    c = Q8Call(max_pages=500)                              # keys enough for partial sums
    log()
    FAKE.fake_set(1, NO_LIMIT)                             # under capture, before the workspace has grown
    c.refused(c.attn, INV, "capture")
    assert c.append() == vva.OK and c.read() == vva.OK
    FAKE.fake_set(0, 0)                                    # on a full device
    c.refused(c.attn, -5, "no memory")
    FAKE.fake_set(0, NO_LIMIT)
    assert c.attn() == vva.OK


def views():
    """q8_pages: what it takes, and that it keeps the pages alive."""
    import torch
    raw = torch.zeros(3, 2, 16 * 68, dtype=torch.uint8)
    v = vva.q8_pages(raw, 64)
    assert list(v.ne) == [64, 16, 2, 3] and list(v.nb) == [34, 68, 1088, 2176] and v.raw is raw and v.data == raw.data_ptr()
    v = vva.q8_pages(torch.zeros(4, 5, 2 * 16 * 136, dtype=torch.uint8)[:, 1:4, :16 * 136], 128)
    assert list(v.ne) == [128, 16, 3, 4] and list(v.nb) == [34, 136, 4352, 21760]
    for bad, d in ((raw.to(torch.int8), 64), (raw[0], 64), (raw, 128 + 16), (raw, 0), (raw[..., :100], 64), (raw[..., ::2], 64)):
        try:
            vva.q8_pages(bad, d)
        except ValueError:
            continue
        raise AssertionError((bad.shape, d))


SCENARIOS = [refusals, accepted, layouts, limits, views]

if __name__ == "__main__":
    FAKE.fake_set(0, NO_LIMIT)
    {f.__name__: f for f in SCENARIOS}[sys.argv[1]]()
