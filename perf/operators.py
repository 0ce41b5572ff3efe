"""Timed cases of the operators that serve many requests at once.

  attn    vva_paged_attn: causal grouped attention of packed new tokens over a cache in pages
  append  vva_paged_rope_append: RoPE of packed q and k rows, k and v into the pages
  norm    vva_add_rms_norm: residual addition and root-mean-square norm, in 16 / 32 bits or in Q8_0 blocks

A batch of requests is `n_seq` sequences, each with its own number of new tokens and of keys; the tokens of all of them are
packed one after the other.  The pages of a sequence lie anywhere in the pool, as they do after some hours of serving.

listed() gives the fixed cases, draw() others of the same ranges, prepare() what a program holds before the call, run()
one pass, work() the bytes and operations of a pass, exact() the result in 64 bits.
"""
import math
import random
import sys

import torch

own = False

THETA = 1.0e6
EPS = 1.0e-6
# hidden size, query heads, kv heads, head dim of the language models
MODELS = {"0.5b": (896, 14, 2, 64), "1.5b": (1536, 12, 2, 128), "7b": (3584, 28, 4, 128)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _batch(op, model, dtype, n_seq, new, past, page, mix, spread, io="f32"):
    """spread: "even" (every sequence `new` tokens behind `past`), "ragged" (both drawn below those bounds), "mixed" (the
    first sequence brings `new` tokens, the others one)."""
    return {"op": op, "model": model, "type": dtype, "n_seq": n_seq, "new": new, "past": past, "page": page, "mix": mix,
            "spread": spread, "io": io}


def _norm(rows, hidden, x, add, out):
    return {"op": "norm", "rows": rows, "hidden": hidden, "x": x, "add": add, "out": out}


def listed():
    cases = [
        # One guidance step of the realtime TTS on paged caches: two streams of the 0.5B model, about 1k keys each.
        ("attn_step_0p5b_2seq", _batch("attn", "0.5b", "f16", 2, 1, 1040, 16, 1, "even")),
        # A transcript decode of one hour-long recording: one stream, 30k keys.
        ("attn_step_7b_long", _batch("attn", "7b", "f16", 1, 1, 30011, 64, 2, "even")),
        # The decode step of a server: 48 requests of very different lengths.
        ("attn_step_7b_48seq", _batch("attn", "7b", "bf16", 48, 1, 8000, 16, 3, "ragged")),
        # The same server while it takes in a new request: one 256-token chunk beside 23 decoding requests.
        ("attn_mixed_7b_24seq", _batch("attn", "7b", "bf16", 24, 256, 4096, 32, 4, "mixed")),
        # A batch of voice prompts and texts of different lengths, none of them in the cache yet.
        ("attn_prompts_1p5b_8seq", _batch("attn", "1.5b", "bf16", 8, 1500, 0, 16, 5, "ragged")),
        # One of the 512-token chunks that long-form ASR prefills in, half-way through an hour.
        ("attn_chunk_7b_512", _batch("attn", "7b", "f16", 1, 512, 15872, 64, 6, "even")),
        # A wide chunk of the same prefill.  The largest case.
        ("attn_chunk_7b_2048", _batch("attn", "7b", "f16", 1, 2048, 28672, 128, 7, "even")),
        # The new rows of a 48-request decode step.
        ("append_step_7b_48seq", _batch("append", "7b", "bf16", 48, 1, 8000, 16, 8, "ragged")),
        # The new rows of packed prompts, about 4k tokens, from F32 projections.
        ("append_prompts_7b", _batch("append", "7b", "f16", 8, 1000, 300, 16, 9, "ragged")),
        # The norm before the projections of a decode step: two rows, quantized for the Q8_0 weights.
        ("norm_step_7b_q8", _norm(2, 3584, "f32", "f32", "q8_0")),
        # The same of an ASR chunk.
        ("norm_chunk_7b_q8", _norm(512, 3584, "f32", "f16", "q8_0")),
        # The norm of a wide prefill in 16 bits.
        ("norm_prompts_7b_bf16", _norm(8192, 3584, "bf16", "bf16", "bf16")),
    ]
    return [dict(name=n, **c) for n, c in cases]


def draw(rng):
    """Another case of these ranges: sizes spread over their logarithm, odd ones among them."""
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attn", "attn", "attn", "append", "norm"])
    if op == "norm":
        out = rng.choice(["q8_0", "f16", "bf16", "f32"])
        hidden = size(2, 256) * 32 if out == "q8_0" else size(64, 8192)
        return _norm(size(1, min(8192, 2 ** 25 // hidden)), hidden, rng.choice(["f32", "f32", "bf16", "f16"]),
                     rng.choice(["none", "f32", "f16", "bf16"]), out)
    model, dtype = rng.choice(list(MODELS)), rng.choice(["f16", "bf16"])
    page, mix = rng.choice([16, 16, 32, 64, 128]), rng.randrange(1 << 20)
    if op == "append":
        new = rng.choice([1, size(2, 2048)])
        return _batch(op, model, dtype, size(1, max(1, min(64, 8192 // new))), new, size(1, 4096), page, mix,
                      rng.choice(["even", "ragged", "mixed"]), io=rng.choice(["f32", "f32", "f16", "bf16"]))
    kind = rng.choice(["step", "step", "chunk", "mixed", "prompts"])
    if kind == "step":                     # single tokens, and the few that a draft model proposes
        n_seq = size(1, 64)
        return _batch(op, model, dtype, n_seq, rng.choice([1, 1, 1, 4]), size(16, min(32768, 2 ** 18 // n_seq)), page, mix,
                      rng.choice(["even", "ragged"]))
    if kind == "chunk":
        new = size(5, 1024)
        return _batch(op, model, dtype, rng.choice([1, 1, 2]), new, size(16, 16384), page, mix,
                      rng.choice(["even", "ragged"]))
    if kind == "mixed":
        return _batch(op, model, dtype, size(2, 24), size(16, 256), size(16, 4096), page, mix, "mixed")
    return _batch(op, model, dtype, size(1, 8), size(2, 1500), 0, page, mix, "ragged")


def _lens(c):
    """(new tokens, keys after the call) of each sequence."""
    rng = random.Random(c["mix"])

    def below(n):                          # 1 .. n, over the logarithm, the top two octaves the likeliest
        return max(1, min(n, int(round(n * 2.0 ** -(4.0 * rng.random() ** 2)))))

    got = []
    for s in range(c["n_seq"]):
        new, past = c["new"], c["past"]
        if c["spread"] == "ragged" and c["n_seq"] > 1:
            new, past = below(new), below(past) if past else 0
        if c["spread"] == "mixed" and s > 0:
            new, past = 1, below(past) if past else 0
        got.append((new, past + new))
    return got


# ------------------------------------------------------------------ inputs

def _rope_table(n, d):
    """[n, d]: the cosines of a position's d / 2 angles, then the sines.  The angles are the library's: position times
    theta^(-2/d), once per pair, each product in 32 bits."""
    ts = torch.tensor(THETA ** (-2.0 / d), dtype=torch.float32, device="cuda")
    th = torch.arange(n, device="cuda", dtype=torch.float32)
    ang = [th]
    while len(ang) < d // 2:
        ang.append(ang[-1] * ts)
    ang = torch.stack(ang, -1).double()
    return torch.cat([torch.cos(ang), torch.sin(ang)], -1).float()


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    if c["op"] == "norm":
        n, h = c["rows"], c["hidden"]
        s = {"x": normal(1, n, h, dtype=TYPES[c["x"]]), "w": 1.0 + normal(h, scale=0.2)}
        s["add"] = None if c["add"] == "none" else normal(1, n, h, dtype=TYPES[c["add"]])
        return s
    hidden, hq, hkv, d = MODELS[c["model"]]
    dt, page = TYPES[c["type"]], c["page"]
    lens = _lens(c)
    used = [-(-L // page) for _, L in lens]
    # the pages of a sequence in the order a pool hands them out after a while, some pages of other requests between;
    # every slot that is not (yet) a sequence's holds what earlier requests left there
    pages = torch.randperm(sum(used) + 7, generator=torch.Generator().manual_seed(int(seed))).to(torch.int32)
    table = torch.full((len(lens), max(used)), -1, dtype=torch.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = pages[at:at + u]
        at += u
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    s = {"table": table.cuda(), "q_start": torch.tensor(starts, dtype=torch.int32).cuda(),
         "kv_len": torch.tensor([L for _, L in lens], dtype=torch.int32).cuda(),
         "max_new": max(n for n, _ in lens), "max_kv": max(L for _, L in lens)}
    n_tok, n_pages = starts[-1], len(pages)
    s["k_pages"] = normal(n_pages, hkv, page, d, dtype=dt)
    s["v_pages"] = normal(n_pages, hkv, page, d, dtype=dt)
    if c["op"] == "attn":
        s["q"] = normal(n_tok, hq, d, dtype=dt)
        s["scale"] = d ** -0.5
    else:
        io = TYPES[c["io"]]
        s["q"], s["k"], s["v"] = (normal(n_tok, h, d, dtype=io) for h in (hq, hkv, hkv))
        s["rope"] = _rope_table(s["max_kv"], d)
    return s


def _library():
    if "vibevoice.cpp_amd" not in sys.path:
        sys.path.insert(0, "vibevoice.cpp_amd")
    import vva
    return vva


def _bind(c, s):
    """The context, the output buffers and the call with its tensor descriptors, which a program makes once and passes
    with every step."""
    vva = _library()
    ctx = vva.Context(0)
    if c["op"] == "norm":
        n, h = c["rows"], c["hidden"]
        total = torch.empty_like(s["x"]) if s["add"] is not None else None
        if c["out"] == "q8_0":
            raw = torch.empty((1, n, h // 32, 34), dtype=torch.uint8, device="cuda")
            y, values = vva.q8_view(raw), (raw[..., 2:].view(torch.int8), raw[..., :2].view(torch.float16))
        else:
            y = values = torch.empty((1, n, h), dtype=TYPES[c["out"]], device="cuda")
        return {"call": ctx.bind_add_rms_norm(s["x"], s["w"], y, add=s["add"], total=total, eps=EPS), "y": values,
                "sum": total}
    batch = vva.Batch(s["q_start"], s["kv_len"], s["table"], s["max_new"])
    out = torch.empty(s["q"].shape, dtype=TYPES[c["type"]], device="cuda")
    if c["op"] == "attn":
        return {"call": ctx.bind_paged_attn(s["q"], s["k_pages"], s["v_pages"], batch, s["scale"], out), "out": out}
    return {"call": ctx.bind_paged_rope_append(s["q"], s["k"], s["v"], s["rope"], batch, s["k_pages"], s["v_pages"], out),
            "out": out}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:                                # the library's handle: a plain program has none
        s["own"] = _bind(case, s)
    return s


# ---------------------------------------------------------------- plain forms

def _where(s):
    """Of each packed token: its sequence, its index among the sequence's new tokens, its index in the sequence."""
    n = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), n, right=True) - 1
    t = n - s["q_start"].long()[seq]
    return seq, t, (s["kv_len"] - s["q_start"].diff()).long()[seq] + t


def _plain_attn(s):
    q, table, start, length = s["q"], s["table"].long(), s["q_start"].long(), s["kv_len"].long()
    n_tok, hq, d = q.shape
    n_seq, hkv, page = len(length), s["k_pages"].shape[1], s["k_pages"].shape[2]
    g, T, L = hq // hkv, s["max_new"], table.shape[1] * page

    def gather(pages):                     # [n_seq, hkv, L, d]
        return pages[table.clamp(min=0)].float().transpose(1, 2).reshape(n_seq, hkv, L, d)

    t = torch.arange(T, device="cuda")
    rows = q[(start[:-1, None] + t).clamp(max=n_tok - 1)].float()                 # [n_seq, T, hq, d]
    rows = rows.view(n_seq, T, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(n_seq, hkv, T * g, d)
    sc = torch.matmul(rows, gather(s["k_pages"]).transpose(-1, -2).contiguous()).mul_(s["scale"])
    last = (length - start.diff())[:, None] + t                                   # [n_seq, T]: the last key a token sees
    hidden = torch.arange(L, device="cuda") > last[..., None]
    sc.view(n_seq, hkv, T, g, L).masked_fill_(hidden[:, None, :, None], -math.inf)
    p = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    den = p.sum(-1, keepdim=True)
    out = torch.matmul(p, gather(s["v_pages"])).div_(den)
    seq, t, _ = _where(s)
    return out.view(n_seq, hkv, T, g, d)[seq, :, t].reshape(n_tok, hq, d).to(q.dtype)


def _rotate(x, table, half):
    a, b = x[..., :half], x[..., half:]
    c, s = table[:, None, :half], table[:, None, half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _slots(s):
    seq, _, i = _where(s)
    page = s["k_pages"].shape[2]
    return s["table"].long()[seq, i // page], i % page, i


def _plain_append(s):
    dt, d = s["k_pages"].dtype, s["q"].shape[-1]
    page, slot, i = _slots(s)
    rope = s["rope"][i]
    s["k_pages"][page, :, slot] = _rotate(s["k"].float(), rope, d // 2).to(dt)
    s["v_pages"][page, :, slot] = s["v"].to(dt)
    return {"q": _rotate(s["q"].float(), rope, d // 2).to(dt), "k": s["k_pages"], "v": s["v_pages"]}


def _plain_norm(c, s):
    h = s["x"].float() if s["add"] is None else s["x"].float() + s["add"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"]
    got = {} if s["add"] is None else {"sum": h.to(s["x"].dtype)}
    if c["out"] == "q8_0":
        b = y.unflatten(-1, (-1, 32))
        d = b.abs().amax(-1, keepdim=True) / 127.0
        z = b * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
        got["y"] = (torch.sign(z) * torch.floor(z.abs() + 0.5)).to(torch.int8) * d.half()
    else:
        got["y"] = y.to(TYPES[c["out"]])
    return got


def run(state):
    """One pass.  The lengths stay where they are, so a pass appends the same rows again."""
    c = state["case"]
    if own:
        b = state["own"]
        b["call"]()
        if c["op"] == "attn":
            return b["out"]
        if c["op"] == "append":
            return {"q": b["out"], "k": state["k_pages"], "v": state["v_pages"]}
        got = {} if b["sum"] is None else {"sum": b["sum"]}
        # Q8_0 blocks are returned as the values they stand for: codes times their block's scale
        got["y"] = b["y"][0] * b["y"][1] if c["out"] == "q8_0" else b["y"]
        return got
    if c["op"] == "attn":
        return _plain_attn(state)
    return _plain_append(state) if c["op"] == "append" else _plain_norm(c, state)


# --------------------------------------------------------------------- work

def work(case):
    c = case
    if c["op"] == "norm":
        size = {"f32": 4, "f16": 2, "bf16": 2, "none": 0, "q8_0": 34 / 32}
        total = size[c["x"]] if c["add"] != "none" else 0
        n = c["rows"] * c["hidden"]
        return {"bytes": n * (size[c["x"]] + size[c["add"]] + total + size[c["out"]]) + 4.0 * c["hidden"], "flops": 5.0 * n}
    hidden, hq, hkv, d = MODELS[c["model"]]
    lens = _lens(c)
    n_tok = sum(n for n, _ in lens)
    if c["op"] == "append":
        io = 4 if c["io"] == "f32" else 2
        return {"bytes": float(n_tok * (hq + 2 * hkv) * d * (io + 2) + n_tok * d * 4),
                "flops": 3.0 * n_tok * (hq + hkv) * d}
    pairs = sum(n * (L - n) + n * (n + 1) // 2 for n, L in lens)
    return {"bytes": 2.0 * (2 * n_tok * hq * d + 2 * sum(L for _, L in lens) * hkv * d), "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------------ 64-bit results

def _exact_attn(c, s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    hq, d = s["q"].shape[1:]
    hkv, page = s["k_pages"].shape[1:3]
    at = 0
    for i, (n, L) in enumerate(_lens(c)):
        ids = s["table"][i, :-(-L // page)].long()
        j = torch.arange(L, device="cuda")
        seen = j[None, :] <= (L - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(hq):
            kv = h // (hq // hkv)
            k, v = (p[ids, kv].reshape(-1, d)[:L].double() for p in (s["k_pages"], s["v_pages"]))
            w = torch.mm(s["q"][at:at + n, h].double(), k.t().contiguous()) * s["scale"]
            w = torch.where(seen, w, torch.full_like(w, -math.inf)).softmax(-1)
            out[at:at + n, h] = torch.mm(w, v)
        at += n
    return out


def _exact_append(c, s):
    d = s["q"].shape[-1]
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    length, table = s["kv_len"].tolist(), s["table"].tolist()
    page = s["k_pages"].shape[2]
    place, at = [], []
    for i, (n, L) in enumerate(_lens(c)):
        for j in range(length[i] - n, length[i]):
            place.append(table[i][j // page] * page + j % page)
            at.append(j)
    place, at = (torch.tensor(v, device="cuda") for v in (place, at))
    cos, sin = (x[:, None] for x in s["rope"].double()[at].split(d // 2, -1))

    def turned(x):
        a, b = x.double().split(d // 2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    for pages, rows in ((k_pages, turned(s["k"])), (v_pages, s["v"].double())):
        pages[place // page, :, place % page] = rows
    return {"q": turned(s["q"]), "k": k_pages, "v": v_pages}


def _exact_norm(c, s):
    h = s["x"].double() + (0.0 if s["add"] is None else s["add"].double())
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"].double()
    if c["out"] == "q8_0":
        b = y.unflatten(-1, (-1, 32))
        d = b.abs().amax(-1, keepdim=True) / 127
        codes = torch.where(d > 0, b / d.clamp(min=1e-300), 0 * b)
        y = torch.trunc(codes + torch.where(codes < 0, -0.5, 0.5)) * d.float().half().double()
    return {"y": y} if s["add"] is None else {"sum": h, "y": y}


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = _inputs(case, seed)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    return _exact_append(case, s) if case["op"] == "append" else _exact_norm(case, s)
