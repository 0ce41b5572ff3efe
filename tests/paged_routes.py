"""Refusals and launches of the paged-cache and norm entry points on the CPU (a child program of test_paged_routes.py, not a
test module), over the stand-in of the HIP runtime that host_routes.py loads.  `python paged_routes.py NAME` runs one."""
import ctypes
import sys

from host_routes import LIB, NO_LIMIT, FAKE, Host, ref, vva

INT = vva.I32


def log():
    return FAKE.fake_take_log().decode().splitlines()


class Call:
    """A correct call's arguments by name; changes() alters one."""

    def __init__(self, N=5, n_seq=3, Hq=14, Hkv=2, d=64, page=16, n_pages=40, max_pages=7, t=vva.F16, io=vva.F32):
        self.c = Host()
        T = self.c.tensor
        self.a = {
            "q": T(io, [d, Hq, N]), "k": T(io, [d, Hkv, N]), "v": T(io, [d, Hkv, N]), "rope": T(vva.F32, [d, 200]),
            "pos": None, "q_out": T(t, [d, Hq, N]), "qa": T(t, [d, Hq, N]), "out": T(t, [d, Hq, N]),
            "k_pages": T(t, [d, page, Hkv, n_pages]), "v_pages": T(t, [d, page, Hkv, n_pages]), "scale": 0.125,
            "q_start": T(INT, [n_seq + 1]), "kv_len": T(INT, [n_seq]), "table": T(INT, [max_pages, n_seq]), "max_new": 4}
        self.make = T

    def batch(self):
        b = vva.BatchDesc()
        for n in ("q_start", "kv_len", "table"):
            ctypes.memmove(ref(getattr(b, n)), ref(self.a[n]), ctypes.sizeof(vva.Tensor))
        b.max_new = self.a["max_new"]
        return b

    def _ref(self, n):
        return None if self.a[n] is None else ref(self.a[n])

    def append(self, batch=True):
        r = self._ref
        return LIB.vva_paged_rope_append(self.c.h, r("q"), r("k"), r("v"), r("rope"), r("pos"),
                                         ref(self.batch()) if batch else None, r("k_pages"), r("v_pages"), r("q_out"))

    def attn(self, batch=True):
        r = self._ref
        return LIB.vva_paged_attn(self.c.h, r("qa"), r("k_pages"), r("v_pages"), ref(self.batch()) if batch else None,
                                  self.a["scale"], r("out"))

    def refused(self, fn, status, what):
        log()
        got = fn()
        lines = log()
        msg = LIB.vva_last_error(self.c.h).decode()
        assert got == status and msg, (what, got, msg)
        assert not any(x.startswith("kernel") for x in lines), (what, lines)


def change(call, name, **kw):
    """A copy of tensor `name` with fields changed: ne=, nb= as {index: value}, type=, data=, shift= (bytes)."""
    t = vva.Tensor()
    ctypes.memmove(ref(t), ref(call.a[name]), ctypes.sizeof(vva.Tensor))
    for k, v in kw.items():
        if k == "shift":
            t.data += v
        elif k in ("ne", "nb"):
            for i, x in v.items():
                getattr(t, k)[i] = x
        else:
            setattr(t, k, v)
    call.a[name] = t


INV, NOT = vva.ERR_INVALID_ARG, vva.ERR_NOT_IMPLEMENTED
# (tensor, change, status): of both calls, of the append, of the attention
BOTH = [
    ("k_pages", dict(type=vva.Q8_0), NOT), ("k_pages", dict(type=vva.F32), NOT), ("v_pages", dict(type=vva.BF16), NOT),
    ("k_pages", dict(data=None), INV), ("v_pages", dict(ne={3: 0}), INV), ("v_pages", dict(ne={1: 32}), INV),
    ("v_pages", dict(ne={3: 41}), INV), ("k_pages", dict(nb={0: 4}), INV), ("k_pages", dict(nb={1: 136}), INV),
    ("v_pages", dict(nb={2: 2056}), INV), ("v_pages", dict(shift=8), INV),
    ("kv_len", dict(ne={0: 0}), INV), ("kv_len", dict(ne={0: 1025}), INV), ("kv_len", dict(type=vva.F32), INV),
    ("kv_len", dict(nb={0: 8}), INV), ("kv_len", dict(data=None), INV), ("kv_len", dict(shift=2), INV),
    ("kv_len", dict(ne={1: 2}), INV), ("q_start", dict(ne={0: 3}), INV), ("q_start", dict(type=vva.F32), INV),
    ("q_start", dict(data=None), INV), ("table", dict(ne={1: 4}), INV), ("table", dict(ne={0: 0}), INV),
    ("table", dict(type=vva.F16), INV), ("table", dict(nb={0: 8}), INV), ("table", dict(nb={1: 30}), INV),
    ("table", dict(data=None), INV), ("table", dict(ne={0: 1 << 27}), NOT),
]
APPEND = [
    ("q", dict(data=None), INV), ("q", dict(ne={1: 13}), INV), ("q", dict(ne={0: 128}), INV), ("q", dict(type=vva.Q8_0), INV),
    ("q", dict(shift=4), INV), ("q", dict(nb={0: 8}), INV), ("q", dict(ne={3: 2}), INV), ("k", dict(ne={2: 4}), INV),
    ("k", dict(ne={1: 1}), INV), ("k", dict(shift=8), INV), ("v", dict(ne={1: 14}), INV), ("v", dict(data=None), INV),
    ("q_out", dict(type=vva.I32), INV), ("q_out", dict(nb={1: 130}), INV), ("q_out", dict(ne={2: 6}), INV),
    ("rope", dict(type=vva.F16), INV), ("rope", dict(ne={0: 32}), INV), ("rope", dict(nb={1: 260}), INV),
    ("rope", dict(data=None), INV), ("rope", dict(ne={1: 0}), INV),
]
ATTN = [
    ("qa", dict(data=None), INV), ("qa", dict(type=vva.F32), INV), ("qa", dict(type=vva.BF16), INV),
    ("qa", dict(ne={1: 15}), INV), ("qa", dict(shift=2), INV), ("qa", dict(ne={2: 0}), INV), ("out", dict(type=vva.F32), INV),
    ("out", dict(ne={2: 6}), INV), ("out", dict(nb={2: 14 * 128 + 8}), INV), ("out", dict(data=None), INV),
]


def refusals():
    for name, kw, status in BOTH + APPEND:
        c = Call()
        change(c, name, **kw)
        c.refused(c.append, status, ("append", name, kw))
    for name, kw, status in BOTH + ATTN:
        c = Call()
        change(c, name, **kw)
        c.refused(c.attn, status, ("attn", name, kw))
    for d, page in ((32, 16), (96, 16), (256, 16), (64, 8), (64, 24), (64, 2048)):
        c = Call(d=d, page=page)
        c.refused(c.attn, NOT, (d, page))
        c.refused(c.append, NOT, (d, page))
    c = Call()
    c.refused(lambda: c.attn(batch=False), INV, "no batch")
    c.refused(lambda: c.append(batch=False), INV, "no batch")
    for s in (0.0, -1.0, float("nan"), float("inf")):
        c = Call()
        c.a["scale"] = s
        c.refused(c.attn, INV, s)
    for m in (0, -3):
        c = Call()
        c.a["max_new"] = m
        c.refused(c.attn, INV, m)
        c.refused(c.append, INV, m)
    c = Call()
    c.a["pos"] = c.make(INT, [4])
    c.refused(c.append, INV, "pos too short")
    c.a["pos"] = c.make(vva.F32, [5])
    c.refused(c.append, INV, "pos type")
    assert LIB.vva_paged_attn(None, None, None, None, None, 1.0, None) == INV
    assert LIB.vva_paged_rope_append(None, None, None, None, None, None, None, None, None, None) == INV
    assert LIB.vva_add_rms_norm(None, None, None, None, 1.0, None, None) == INV


def overlaps():
    for a, b in (("out", "qa"), ("out", "k_pages"), ("out", "v_pages")):
        c = Call()
        change(c, a, data=c.a[b].data)
        c.refused(c.attn, INV, (a, b))
        change(c, a, data=c.a[b].data + 64 * 2)
        c.refused(c.attn, INV, (a, b))
    for b in ("k", "v", "k_pages", "v_pages", "rope"):
        c = Call()
        change(c, "q_out", data=c.a[b].data)
        c.refused(c.append, INV, b)
    c = Call(io=vva.F16)                                   # q in place, but not over a shifted or differently typed q
    change(c, "q_out", data=c.a["q"].data)
    assert c.append() == vva.OK
    change(c, "q_out", data=c.a["q"].data + 128)
    c.refused(c.append, INV, "shifted")
    c = Call(io=vva.F32)
    change(c, "q_out", data=c.a["q"].data)
    c.refused(c.append, INV, "type")


def accepted():
    for kw in (dict(), dict(N=1, n_seq=1, n_pages=1, max_pages=1), dict(t=vva.BF16, io=vva.F16, Hq=28, Hkv=4, d=128, page=1024),
               dict(N=3, n_seq=1024), dict(N=70000, n_seq=2), dict(Hq=33, Hkv=1)):
        c = Call(**kw)
        log()
        assert c.append() == vva.OK, LIB.vva_last_error(c.c.h)
        assert any(x.startswith("kernel paged_append") for x in log())
        assert c.attn() == vva.OK, LIB.vva_last_error(c.c.h)
        assert any(x.startswith("kernel paged") for x in log())


def norm():
    def call(x, w, y, add=None, total=None, eps=1e-6):
        return LIB.vva_add_rms_norm(h.h, ref(x) if x else None, ref(add) if add else None, ref(w) if w else None, eps,
                                    ref(total) if total else None, ref(y) if y else None)

    h = Host()
    T = h.tensor

    def refused(status, *a, **kw):
        log()
        got = call(*a, **kw)
        assert got == status and LIB.vva_last_error(h.h).decode(), (got, a, kw)
        assert not log()

    x, w, y, a, s = T(vva.F32, [64, 5, 2]), T(vva.F32, [64]), T(vva.F16, [64, 5, 2]), T(vva.BF16, [64, 5, 2]), T(vva.F16, [64, 5, 2])
    assert call(x, w, y, a, s) == vva.OK and call(x, w, y) == vva.OK
    assert call(x, w, x) == vva.OK and call(x, w, y, a, x) == vva.OK and call(x, w, x, a, a) == vva.OK
    assert call(x, w, T(vva.Q8_0, [64, 5, 2])) == vva.OK
    refused(INV, None, w, y)
    refused(INV, x, None, y)
    refused(INV, x, w, None)
    refused(INV, x, T(vva.F32, [63]), y)
    refused(INV, x, T(vva.F16, [64]), y)
    refused(INV, T(vva.I32, [64, 5, 2]), w, y)
    refused(INV, T(vva.F32, [64, 5, 2, 2]), w, y)
    refused(INV, x, w, T(vva.F16, [64, 5, 1]))
    refused(INV, x, w, T(vva.I32, [64, 5, 2]))
    refused(INV, x, w, y, T(vva.F32, [64, 4, 2]))
    refused(INV, x, w, y, a, T(vva.F32, [32, 5, 2]))
    refused(INV, x, w, y, a, T(vva.Q8_0, [64, 5, 2]))
    refused(INV, T(vva.F32, [48, 5, 2]), T(vva.F32, [48]), T(vva.Q8_0, [64, 5, 2]))
    q8 = T(vva.Q8_0, [64, 5, 2])
    q8.ne[0] = 48
    refused(INV, T(vva.F32, [48, 5, 2]), T(vva.F32, [48]), q8)
    refused(INV, x, w, T(vva.Q8_0, [64, 5, 2], off=1))
    refused(INV, x, w, T(vva.F32, [64, 5, 2], nb=[8, 512, 2560, 5120]))
    for eps in (-1.0, float("nan"), float("inf")):
        refused(INV, x, w, y, eps=eps)
    refused(NOT, T(vva.F32, [16385, 1, 1]), T(vva.F32, [16385]), T(vva.F32, [16385, 1, 1]))
    # overlaps other than an input itself
    refused(INV, x, w, T(vva.F32, [64, 5, 2], data=x.data + 256))
    refused(INV, x, w, T(vva.F16, [64, 5, 2], data=x.data))
    refused(INV, x, w, y, a, T(vva.F16, [64, 5, 2], data=y.data))
    refused(INV, x, w, T(vva.F32, [64, 1, 1], data=w.data))
    refused(INV, x, w, y, a, T(vva.F32, [64, 5, 2], data=x.data + 4))


def limits():
    """The largest calls, and those past them."""
    for kw, ok in ((dict(Hq=256, Hkv=1, N=1), True), (dict(Hq=257, Hkv=1, N=1), False), (dict(Hq=512, Hkv=2, N=1), True),
                   (dict(Hq=1, Hkv=1, N=1 << 22), True), (dict(Hq=1, Hkv=1, N=(1 << 22) + 1), False),
                   (dict(Hq=63, Hkv=63, N=1, n_seq=1024), True), (dict(Hq=64, Hkv=64, N=1, n_seq=1024), False),
                   (dict(n_seq=16, max_pages=(1 << 30) // 16), True), (dict(n_seq=17, max_pages=(1 << 30) // 16), False),
                   (dict(n_seq=1, max_pages=(1 << 30) // 16 + 1), False)):
        for name in ("append", "attn"):
            c = Call(**kw)
            if ok:
                assert getattr(c, name)() == vva.OK, (name, kw, LIB.vva_last_error(c.c.h))
            else:
                c.refused(getattr(c, name), NOT, (name, kw))
    c = Call()
    change(c, "k_pages", nb={1: 1 << 27})
    c.refused(c.attn, NOT, "a page of 2 GiB")
    for i in (1, 2):                                        # rows of q 4 MiB apart
        c = Call()
        change(c, "qa", nb={i: 1 << 22, 2: 1 << 26} if i == 1 else {2: 1 << 22})
        c.refused(c.attn, NOT, i)
    c = Call(max_pages=500)                                 # keys enough for partial sums
    log()
    FAKE.fake_set(1, NO_LIMIT)                              # under capture, before the workspace has grown
    c.refused(c.attn, INV, "capture")
    assert c.append() == vva.OK
    FAKE.fake_set(0, 0)                                     # on a full device
    c.refused(c.attn, -5, "no memory")
    FAKE.fake_set(0, NO_LIMIT)
    assert c.attn() == vva.OK


def interleaved_rows():
    """The parts of one projection's rows, q in place or out beside it; pages of K and V by turns."""
    for io in (vva.F32, vva.F16):
        c = Call(io=io, t=vva.F16)
        es, whole = (4 if io == vva.F32 else 2), 14 + 4
        y = c.make(io, [64, whole, 5])
        for name, h, at in (("q", 14, 0), ("k", 2, 14), ("v", 2, 16)):
            change(c, name, data=y.data + at * 64 * es, ne={1: h}, nb={2: 64 * es * whole, 3: 64 * es * whole * 5})
        c.a["q_out"] = c.a["q"]
        assert c.append() == vva.OK, LIB.vva_last_error(c.c.h)
        change(c, "q_out", shift=64 * es)
        c.refused(c.append, INV, "a head further: k's first")
    c = Call()                                             # out between q's rows
    change(c, "qa", nb={2: 2 * 14 * 128, 3: 2 * 14 * 128 * 5})
    change(c, "out", data=c.a["qa"].data + 14 * 128, nb={2: 2 * 14 * 128, 3: 2 * 14 * 128 * 5})
    assert c.attn() == vva.OK, LIB.vva_last_error(c.c.h)
    change(c, "out", shift=-16)
    c.refused(c.attn, INV, "16 bytes of each row")
    change(c, "out", shift=16, nb={2: 3 * 14 * 128, 3: 3 * 14 * 128 * 5})
    c.refused(c.attn, INV, "rows of another pitch")
    c = Call()
    p = c.a["k_pages"]
    two = {3: 2 * p.nb[3]}
    change(c, "v_pages", data=p.data + p.nb[3], nb=two)
    change(c, "k_pages", nb=two)
    assert c.append() == vva.OK and c.attn() == vva.OK, LIB.vva_last_error(c.c.h)
    change(c, "v_pages", data=c.a["k_pages"].data)
    c.refused(c.append, INV, "K and V in the same rows")
    for name in ("q", "k", "v", "rope", "pos", "q_start", "kv_len", "table"):
        c = Call()
        c.a["pos"] = c.make(INT, [5])
        change(c, name, data=c.a["v_pages"].data + 4096)
        c.refused(c.append, INV, name)
    for name in ("q_start", "kv_len", "table"):
        c = Call()
        change(c, "out", data=c.a[name].data - c.a[name].data % 16)
        c.refused(c.attn, INV, name)


def blocks_to_projections():
    """Q8_0 rows as x of the projections, beside Q8_0 weights."""
    h = Host()
    T = h.tensor
    w = lambda t, K=896: [T(t, [K, m]) for m in (896, 128, 128)]  # noqa: E731

    def proj(x, ws, N, expect, kernels=None, **kw):
        y = T(vva.F32, [1152, N])
        st, names, _ = h.call("vva_qkv_proj", ref(x), *map(ref, ws), None, None, None, ref(y), **kw)
        assert st == expect, (st, h.err())
        assert [n.split("<")[0] for n in names] == (kernels or []), names

    def fused(x, ws, N, expect, **kw):
        kv = h.kv(2, 64, 64, 1, vva.F16, [0])
        q, pos = T(vva.F32, [64, 14, N]), T(INT, [N])
        st, names, _ = h.call("vva_qkv_rope_append", kv, 0, ref(x), *map(ref, ws), None, None, None, ref(pos), None, 1e6, ref(q), **kw)
        assert st == expect, (st, h.err())
        return [n.split("<")[0] for n in names]

    wq8, wf16 = w(vva.Q8_0), w(vva.F16)
    x = T(vva.Q8_0, [896, 3])
    proj(x, wq8, 3, INV, capturing=True)                   # the F32 rows' workspace is not there yet
    proj(x, wq8, 3, vva.OK, ["proj_rows_from_q8_kernel", "proj_gemv_q8_kernel"])
    proj(x, wq8, 3, vva.OK, ["proj_rows_from_q8_kernel", "proj_gemv_q8_kernel"], capturing=True)
    proj(T(vva.F32, [896, 3]), wq8, 3, vva.OK, ["proj_gemv_q8_kernel"])
    assert fused(x, wq8, 3, vva.OK)[0] == "proj_rows_from_q8_kernel"
    assert "proj_rows_from_q8_kernel" not in fused(T(vva.Q8_0, [896, 40]), wq8, 40, vva.OK)
    bad = [(x, wf16, INV), (T(vva.Q8_0, [896, 3], off=1), wq8, INV), (T(vva.Q8_0, [896, 3], nb=[34, 953, 2859, 2859]), wq8, INV),
           (T(vva.Q8_0, [896, 3], nb=[68, 1904, 5712, 5712]), wq8, INV), (T(vva.Q8_0, [896, 3, 1, 2]), wq8, INV),
           (T(vva.Q8_0, [832, 3]), wq8, INV)]
    for b, ws, st in bad:
        proj(b, ws, 3, st)
        assert fused(b, ws, 3, st) == []
    proj(T(vva.Q8_0, [896, 9]), wq8, 9, NOT)


SCENARIOS = [refusals, overlaps, accepted, norm, limits, interleaved_rows, blocks_to_projections]

if __name__ == "__main__":
    FAKE.fake_set(0, NO_LIMIT)
    {f.__name__: f for f in SCENARIOS}[sys.argv[1]]()
