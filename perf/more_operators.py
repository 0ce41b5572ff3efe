"""Timed cases of the operators over a cache in pages of 8 bits.

  attn    vva_paged_attn: causal grouped attention of packed new tokens over Q8_0 pages
  append  vva_paged_rope_append: RoPE of packed q and k rows, k and v quantised into the pages
  read    vva_paged_read: keys and values of the batch's tokens read back out of the pages

A page of a kv head is `page` rows of d codes of 8 bits, then d / 32 rows of `page` F16 scales, one for 32 dims of a slot.  The
batches are those of a server: sequences of new tokens packed one after the other, their pages anywhere in the pool.

listed() gives the fixed cases, draw() others of the same ranges, prepare() what a program holds before the call, run()
one pass, work() the bytes and operations of a pass, exact() the result in 64 bits.
"""
import math
import random
import sys

import torch

own = False

THETA = 1.0e6
# query heads, kv heads, head dim of the language models
MODELS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _batch(op, model, dtype, n_seq, new, past, page, mix, spread, io="f32"):
    """spread: "even" (every sequence `new` tokens behind `past`), "ragged" (both drawn below those bounds), "mixed" (the
    first sequence brings `new` tokens, the others one).  type: of q and the output; of what is read back."""
    return {"op": op, "model": model, "type": dtype, "n_seq": n_seq, "new": new, "past": past, "page": page, "mix": mix,
            "spread": spread, "io": io}


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
        ("append_step_7b_48seq", _batch("append", "7b", "bf16", 48, 1, 70, 16, 8, "ragged")),
        # The new rows of packed prompts, about 4k tokens, from F32 projections.
        ("append_prompts_7b", _batch("append", "7b", "f16", 8, 1000, 300, 16, 9, "ragged")),
        # The cache of a voice prompt of one stream, read back to be kept with the voice.
        ("read_voice_0p5b", _batch("read", "0.5b", "f32", 1, 333, 0, 16, 10, "even")),
        # Requests that are parked on the host while others run.
        ("read_parked_7b_6seq", _batch("read", "7b", "bf16", 6, 8000, 0, 32, 11, "ragged")),
    ]
    return [dict(name=n, **c) for n, c in cases]


def draw(rng):
    """Another case of these ranges: sizes spread over their logarithm, odd ones among them."""
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attn", "attn", "attn", "append", "read"])
    model, dtype = rng.choice(list(MODELS)), rng.choice(["f16", "bf16"])
    page, mix = rng.choice([16, 16, 32, 64, 128]), rng.randrange(1 << 20)
    if op == "append":
        new = rng.choice([1, size(2, 2048)])
        return _batch(op, model, dtype, size(1, max(1, min(64, 8192 // new))), new, size(1, 128), page, mix,
                      rng.choice(["even", "ragged", "mixed"]), io=rng.choice(["f32", "f32", "f16", "bf16"]))
    if op == "read":
        new = rng.choice([1, size(2, 16384)])
        return _batch(op, model, rng.choice(["f32", "f16", "bf16"]), size(1, max(1, min(64, 32768 // new))), new,
                      rng.choice([0, size(1, 4096)]), page, mix, rng.choice(["even", "ragged", "mixed"]))
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
    ang = [torch.arange(n, device="cuda", dtype=torch.float32)]
    while len(ang) < d // 2:
        ang.append(ang[-1] * ts)
    ang = torch.stack(ang, -1).double()
    return torch.cat([torch.cos(ang), torch.sin(ang)], -1).float()


def _codes(raw, d):
    """The codes [n_pages, Hkv, page, d] and the scales [n_pages, Hkv, d / 32, page] of pages, as views of their bytes."""
    n, h, size = raw.shape
    page = size * 16 // (17 * d)
    return (raw[..., :page * d].view(torch.int8).view(n, h, page, d),
            raw[..., page * d:].view(torch.float16).view(n, h, d // 32, page))


def _quantise(y):
    """Codes and scales of rows [..., d] in 32 bits: d / 127 of a block's largest magnitude, each step in 32 bits, as the
    codes next to a border go by it."""
    b = y.unflatten(-1, (-1, 32))
    big = b.abs().amax(-1, keepdim=True)
    step = big / torch.full_like(big, 127.0)
    z = b * torch.where(step > 0, torch.ones_like(step) / step, torch.zeros_like(step))
    low = z.abs().floor()
    codes = torch.sign(z) * (low + (z.abs() - low >= 0.5))
    return codes.to(torch.int8).flatten(-2), step.squeeze(-1).half()


def _pool(n, hkv, page, d, normal):
    raw = torch.empty(n, hkv, page * (d + d // 16), dtype=torch.uint8, device="cuda")
    codes, scales = _codes(raw, d)
    for i in range(0, n, 4096):            # in parts: the rows take four times the pages' memory
        c, s = _quantise(normal(min(4096, n - i), hkv, page, d))
        codes[i:i + 4096], scales[i:i + 4096] = c, s.transpose(-1, -2)
    return raw


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    hq, hkv, d = MODELS[c["model"]]
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
    n_tok = starts[-1]
    s = {"table": table.cuda(), "q_start": torch.tensor(starts, dtype=torch.int32).cuda(),
         "kv_len": torch.tensor([L for _, L in lens], dtype=torch.int32).cuda(),
         "max_new": max(n for n, _ in lens), "max_kv": max(L for _, L in lens), "n_tok": n_tok, "d": d}
    s["k_pages"], s["v_pages"] = (_pool(len(pages), hkv, page, d, normal) for _ in range(2))
    if c["op"] == "attn":
        s["q"] = normal(n_tok, hq, d, dtype=dt)
        s["scale"] = d ** -0.5
    elif c["op"] == "append":
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
    dt, d = TYPES[c["type"]], s["d"]
    batch = vva.Batch(s["q_start"], s["kv_len"], s["table"], s["max_new"])
    k_pages, v_pages = (vva.q8_pages(s[n], d) for n in ("k_pages", "v_pages"))
    if c["op"] == "read":
        k, v = (torch.empty(s["n_tok"], s["k_pages"].shape[1], d, dtype=dt, device="cuda") for _ in range(2))
        return {"call": ctx.bind_paged_read(batch, k_pages, v_pages, k, v), "k": k, "v": v}
    out = torch.empty(s["q"].shape, dtype=dt, device="cuda")
    if c["op"] == "attn":
        return {"call": ctx.bind_paged_attn(s["q"], k_pages, v_pages, batch, s["scale"], out), "out": out}
    return {"call": ctx.bind_paged_rope_append(s["q"], s["k"], s["v"], s["rope"], batch, k_pages, v_pages, out), "out": out}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:                                # the library's handle: a plain program has none
        s["own"] = _bind(case, s)
    return s


# ---------------------------------------------------------------- plain forms

def _values(raw, d):
    """[..., page, d] in 32 bits, of pages [..., bytes]."""
    codes, scales = _codes(raw, d)
    return codes.float() * scales.transpose(-1, -2).float().repeat_interleave(32, -1)


def _stored(raw, d):
    """What the pages stand for, in the type of their scales."""
    codes, scales = _codes(raw, d)
    return codes.unflatten(-1, (-1, 32)) * scales.transpose(-1, -2)[..., None]


def _where(s):
    """Of each packed token: its sequence, its index among the sequence's new tokens, its index in the sequence."""
    n = torch.arange(s["n_tok"], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), n, right=True) - 1
    t = n - s["q_start"].long()[seq]
    return seq, t, (s["kv_len"] - s["q_start"].diff()).long()[seq] + t


def _slots(s):
    seq, _, i = _where(s)
    page = s["k_pages"].shape[2] * 16 // (17 * s["d"])
    return s["table"].long()[seq, i // page], i % page, i


def _plain_attn(s):
    q, table, start, length, d = s["q"], s["table"].long(), s["q_start"].long(), s["kv_len"].long(), s["d"]
    n_tok, hq, _ = q.shape
    n_seq, hkv, page = len(length), s["k_pages"].shape[1], s["k_pages"].shape[2] * 16 // (17 * d)
    g, T, L = hq // hkv, s["max_new"], table.shape[1] * page

    def gather(raw):                       # [n_seq, hkv, L, d]
        rows = _values(raw[table.clamp(min=0).flatten()], d)
        return rows.view(n_seq, -1, hkv, page, d).transpose(1, 2).reshape(n_seq, hkv, L, d)

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
    """x0 c - x1 s and x0 s + x1 c in 32 bits, the second product rounded, the first not: 64 bits hold it."""
    a, b = x[..., :half].double(), x[..., half:]
    c, s = table[:, None, :half], table[:, None, half:]
    return torch.cat([a * c.double() - (b * s).double(), a * s.double() + (b * c).double()], -1).float()


def _plain_append(s, dt):
    d = s["d"]
    page, slot, i = _slots(s)
    rope = s["rope"][i]
    for raw, rows in ((s["k_pages"], _rotate(s["k"].float(), rope, d // 2)), (s["v_pages"], s["v"].float())):
        codes, scales = _codes(raw, d)
        codes[page, :, slot], scales[page, :, :, slot] = _quantise(rows)
    return _rotate(s["q"].float(), rope, d // 2).to(dt)


def _plain_read(s, dt):
    page, slot, _ = _slots(s)
    got = {}
    for n in ("k", "v"):
        codes, scales = _codes(s[n + "_pages"], s["d"])
        got[n] = (codes[page, :, slot].float() * scales[page, :, :, slot].float().repeat_interleave(32, -1)).to(dt)
    return got


def run(state):
    """One pass.  The lengths stay where they are, so a pass appends the same rows again."""
    c = state["case"]
    dt, d = TYPES[c["type"]], state["d"]
    if own:
        b = state["own"]
        b["call"]()
        if c["op"] == "read":
            return {"k": b["k"], "v": b["v"]}
        out = b["out"]
    elif c["op"] == "read":
        return _plain_read(state, dt)
    else:
        out = _plain_attn(state) if c["op"] == "attn" else _plain_append(state, dt)
    if c["op"] == "attn":
        return out
    # the pages are returned as the values they stand for: codes times their block's scale
    return {"q": out, "k": _stored(state["k_pages"], d), "v": _stored(state["v_pages"], d)}


# --------------------------------------------------------------------- work

def work(case):
    c = case
    hq, hkv, d = MODELS[c["model"]]
    lens = _lens(c)
    n_tok = sum(n for n, _ in lens)
    row = 2 * hkv * d * 34.0 / 32          # a token's K and V in the pages
    size = 4 if c["type"] == "f32" else 2
    if c["op"] == "read":
        return {"bytes": n_tok * (row + 2 * hkv * d * size), "flops": 2.0 * n_tok * hkv * d}
    if c["op"] == "append":
        io = 4 if c["io"] == "f32" else 2
        return {"bytes": n_tok * ((hq + 2 * hkv) * d * io + hq * d * size + row + d * 4.0),
                "flops": 3.0 * n_tok * (hq + hkv) * d + 4.0 * n_tok * hkv * d}
    pairs = sum(n * (L - n) + n * (n + 1) // 2 for n, L in lens)
    return {"bytes": 2.0 * n_tok * hq * d * size + sum(L for _, L in lens) * row, "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------------ 64-bit results

def _blocks(raw, d):
    """The pages' values [n_pages, Hkv, page, d] in 64 bits."""
    n, h, size = raw.shape
    page = size * 16 // (17 * d)
    codes, scales = raw.split([page * d, page * d // 16], -1)
    scales = scales.contiguous().view(torch.float16).double().view(n, h, d // 32, page, 1)
    codes = codes.contiguous().view(torch.int8).double().view(n, h, page, d // 32, 32)
    return (codes * scales.transpose(2, 3)).view(n, h, page, d)


def _exact_attn(c, s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    hq, d = s["q"].shape[1:]
    hkv = s["k_pages"].shape[1]
    at = 0
    for i, (n, L) in enumerate(_lens(c)):
        ids = s["table"][i, :-(-L // c["page"])].long()
        j = torch.arange(L, device="cuda")
        seen = j[None, :] <= (L - n + torch.arange(n, device="cuda"))[:, None]
        for kv in range(hkv):
            k, v = (_blocks(p[ids, kv:kv + 1], d).reshape(-1, d)[:L] for p in (s["k_pages"], s["v_pages"]))
            for h in range(kv * (hq // hkv), (kv + 1) * (hq // hkv)):
                w = torch.mm(s["q"][at:at + n, h].double(), k.t().contiguous()) * s["scale"]
                w = torch.where(seen, w, torch.full_like(w, -math.inf)).softmax(-1)
                out[at:at + n, h] = torch.mm(w, v)
        at += n
    return out


def _places(c, s):
    """Page and slot of every token of the batch, and its index in its sequence."""
    length, table, page = s["kv_len"].tolist(), s["table"].tolist(), c["page"]
    got = [(table[i][j // page], j % page, j) for i, (n, _) in enumerate(_lens(c)) for j in range(length[i] - n, length[i])]
    return torch.tensor(got, device="cuda").unbind(-1)


def _exact_append(c, s):
    d = s["d"]
    page, slot, at = _places(c, s)
    cos, sin = (x[:, None] for x in s["rope"].double()[at].split(d // 2, -1))

    def turned(x):
        a, b = x.double().split(d // 2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    def rounded(x):
        b = x.unflatten(-1, (-1, 32))
        step = b.abs().amax(-1, keepdim=True) / 127
        z = torch.where(step > 0, b / step.clamp(min=1e-300), 0 * b)
        return (torch.trunc(z + torch.where(z < 0, -0.5, 0.5)) * step.float().half().double()).flatten(-2)

    got = {"q": turned(s["q"])}
    for n, rows in (("k", turned(s["k"])), ("v", s["v"].double())):
        got[n] = _blocks(s[n + "_pages"], d)
        got[n][page, :, slot] = rounded(rows)
        got[n] = got[n].unflatten(-1, (-1, 32))
    return got


def _exact_read(c, s):
    page, slot, _ = _places(c, s)
    return {n: _blocks(s[n + "_pages"], s["d"])[page, :, slot] for n in ("k", "v")}


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = _inputs(case, seed)
    return {"attn": _exact_attn, "append": _exact_append, "read": _exact_read}[case["op"]](case, s)
