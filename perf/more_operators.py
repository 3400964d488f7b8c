"""More operators of a serving step, as timed and compared cases: rotary tables
scaled for long contexts, head norms with the position rotation in one pass,
and a paged cache that holds keys and values in 4 bits, with attention over it.

The model's own sizes are 16 query and 4 kv heads of 256 elements, sliding
windows of 512 positions, a rotated share of a quarter or all of a head, chunks
of up to 512 prompt tokens, blocks of 8 verified tokens and contexts of up to
131072 positions; other heads are generic.

What the listed cases stand for:

  table-4k       a table for a short context, frequencies scaled by wavelength: start-up of a small server
  table-128k     the table of the longest context, frequencies interpolated by band
  rope-1         one decoded token's queries and keys, a quarter of the head turned: latency
  rope-chunk     a prompt chunk with head norms and interleaved pairs
  rope-8192      a long prompt of a model with many smaller heads, with norms
  append-1       one token of one conversation: latency
  append-64      a decode step of 64 conversations of any length, with head norms
  append-chunk   a whole prompt chunk, bf16 activations, interleaved pairs and head norms
  attend-1       one token early in a conversation: latency
  attend-far     one token at the end of the longest context
  attend-48      a decode step of 48 conversations of very unequal lengths
  attend-chunk   a prompt chunk deep in a long document

Rotation. Row p of a table holds the cosines, then the sines of p f_i, i < d / 2,
times the attention factor a; with f0_i = theta^(-2 i / d)
  linear  f = f0 / factor
  ntk     theta * factor^(d / (d - 2)) in place of theta
  yarn    c(r) = d ln(original / (2 pi r)) / (2 ln theta); lo = max(floor c(beta_fast), 0),
          hi = min(ceil c(beta_slow), d - 1); t = clamp((i - lo) / max(hi - lo, 0.001), 0, 1);
          f = f0 (1 - t) + f0 t / factor; a = 0.1 ln(factor) + 1
  bands   w = original f0 / (2 pi); f = f0 where w > high, f0 / factor where w < low, between
          them f0 ((1 - s) / factor + s) with s = (w - low) / (high - low).
Elements (e, e + d / 2) of a head turn together, interleaved (2 e, 2 e + 1); a norm
comes first: x / sqrt(mean x^2 + eps) * weight.

The cache. A page holds 64 positions of every kv head. 32 elements of a position
and head share one power of two 2^(byte - 127), the smallest with amax <= 7 * 2^e,
-120 <= e <= 125; an element is a sign and one of 0 0.5 1 1.5 2 3 4 6 (codes 0..7, 8
added for the sign) times it, the nearest, of two as near the even code; the even
element's code is the low half of its byte. A page's kv head is 68 head_dim bytes:
  key codes     position 16 t + c, part g = bytes of 4 (j = 0 ..): head_dim >= 128: [t][j][g][c][16 bytes], elements
                32 (4 j + g) ..; 64: [t][g][c][8 bytes], elements 16 g ..
  value codes   position 32 u + 16 a + 4 g + b; with n = head_dim / 16 a lane c has elements n c ..; the 4 n bytes
                [a][b][n / 2] of (u, g, c) are cut in 16: [u][piece][g][c][16]
  key scales    [g][c][t][j], head_dim 64: [g 2][c][t]
  value scales  [g][block][u][a][b]
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

HEADS, KV_HEADS, HEAD_DIM, WINDOW = 16, 4, 256, 512
PAGE = 64
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    m = {"heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM}
    return [
        {"name": "table-4k", "op": "table", "rows": 4096, "pdim": 64, "theta": 5e6, "kind": "bands", "factor": 8.0,
         "original": 1024},
        {"name": "table-128k", "op": "table", "rows": 131072, "pdim": 256, "theta": 1e4, "kind": "yarn", "factor": 32.0,
         "original": 4096},
        {"name": "rope-1", "op": "rope", **m, "tokens": 1, "pdim": 64, "inter": False, "norm": False, "x": "f32"},
        {"name": "rope-chunk", "op": "rope", **m, "tokens": 512, "pdim": 256, "inter": True, "norm": True, "x": "f32"},
        {"name": "rope-8192", "op": "rope", "heads": 32, "kv_heads": 8, "head_dim": 128, "tokens": 8192, "pdim": 128,
         "inter": False, "norm": True, "x": "bf16"},
        {"name": "append-1", "op": "append", **m, "nseq": 1, "tokens": 1, "ctx": 1003, "pdim": 64, "inter": False,
         "norm": False, "x": "f32"},
        {"name": "append-64", "op": "append", **m, "nseq": 64, "tokens": 1, "ctx": 8000, "pdim": 64, "inter": False,
         "norm": True, "x": "f32"},
        {"name": "append-chunk", "op": "append", **m, "nseq": 1, "tokens": 512, "ctx": 1000, "pdim": 256, "inter": True,
         "norm": True, "x": "bf16"},
        {"name": "attend-1", "op": "attend", **m, "nseq": 1, "tokens": 1, "ctx": 1003, "window": 0, "gate": False,
         "x": "f32", "out": "f32"},
        {"name": "attend-far", "op": "attend", **m, "nseq": 1, "tokens": 1, "ctx": 131071, "window": 0, "gate": False,
         "x": "f32", "out": "f32"},
        {"name": "attend-48", "op": "attend", **m, "nseq": 48, "tokens": 1, "ctx": 12000, "window": 0, "gate": True,
         "x": "f32", "out": "bf16"},
        {"name": "attend-chunk", "op": "attend", **m, "nseq": 1, "tokens": 512, "ctx": 16384, "window": 0,
         "gate": False, "x": "bf16", "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("table", "rope", "append", "append", "attend", "attend", "attend", "attend"))
    if op == "table":
        return {"op": op, "rows": _log(rng, 100, 131072), "pdim": 2 * rng.randint(2, 128), "theta": rng.choice((1e4, 5e5, 5e6)),
                "kind": rng.choice(("none", "linear", "ntk", "yarn", "bands")), "factor": rng.choice((1.5, 2.0, 4.0, 8.0, 32.0)),
                "original": rng.choice((1024, 4096, 8192))}
    hd = rng.choice((64, 128, 256, 256) if op != "rope" else (64, 80, 96, 128, 256))
    kvh = rng.choice((1, 2, 4, 4, 8)) if hd < 256 else rng.choice((1, 2, 4, 4))
    group = rng.choice((1, 2, 4, 4, 8)) if hd < 256 else rng.choice((1, 2, 4, 4))
    c = {"op": op, "heads": kvh * group, "kv_heads": kvh, "head_dim": hd, "x": rng.choice(("f32", "bf16"))}
    turn = {"pdim": rng.choice((0, hd // 4 // 2 * 2, hd // 2, hd)), "inter": rng.random() < 0.4, "norm": rng.random() < 0.5}
    if op == "rope":
        c.update(turn, tokens=_log(rng, 1, 8192))
        while c["tokens"] * (c["heads"] + kvh) * hd > 8192 * 40 * 64:
            c["tokens"] //= 2
        return c
    form = rng.choice(("decode", "decode", "block", "chunk"))
    if op == "append":
        c.update(turn)
        c["nseq"] = _log(rng, 1, 64) if form == "decode" else _log(rng, 1, 8)
        c["tokens"] = {"decode": 1, "block": rng.randint(2, 16), "chunk": _log(rng, 17, 512)}[form]
        c["ctx"] = _log(rng, 1, 30000 if form == "decode" else 8000)
        while c["nseq"] * c["tokens"] > 1024:
            c["nseq"] //= 2
        return c
    c["nseq"] = _log(rng, 1, 64) if form == "decode" else _log(rng, 1, 6)
    c["tokens"] = {"decode": 1, "block": rng.randint(2, 8), "chunk": _log(rng, 9, 300)}[form]
    c["ctx"] = _log(rng, 1, 100000 if form == "decode" else 8000)
    c["window"] = rng.choice((0, 0, WINDOW, _log(rng, 1, 4000)))
    c["gate"] = rng.random() < 0.3
    c["out"] = rng.choice(("f32", "bf16"))
    most = 131072 if form == "decode" else 16384
    while c["nseq"] > 1 and c["nseq"] * c["ctx"] > most:
        c["nseq"] //= 2
    return c


# ------------------------------------------------------------------ shapes


def _shape(c):
    """Positions cached before the call and new tokens, per sequence: unequal where there are several."""
    rng = random.Random(c["nseq"] * 1000003 + c["ctx"] * 101 + c["tokens"])
    pos, new = [c["ctx"]], [c["tokens"]]
    for _ in range(c["nseq"] - 1):
        pos.append(int(round(math.exp(rng.uniform(0.0, math.log(c["ctx"] + 1.0)))) - 1) if rng.random() < 0.6
                   else rng.randint(0, c["ctx"]))
        new.append(rng.randint(max(1, c["tokens"] // 2), c["tokens"]))
    return pos, new


def _visible(c):
    """Positions read by each sequence, and (query, position) pairs of each."""
    pos, new = _shape(c)
    w, spans, pairs = c["window"], [], []
    for p, t in zip(pos, new):
        first = max(0, p + 1 - w) if w else 0
        spans.append(p + t - first)
        pairs.append(sum(min(p + j + 1, w) if w else p + j + 1 for j in range(t)))
    return spans, pairs


def work(case):
    c = case
    if c["op"] == "table":
        return {"bytes": c["rows"] * c["pdim"] * 4, "flops": 3.0 * c["rows"] * c["pdim"]}
    size = 4 if c["x"] == "f32" else 2
    qd, kvd = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    if c["op"] == "rope":
        n = c["tokens"]
        return {"bytes": n * (2 * (qd + kvd) * size + c["pdim"] * 4 + 4), "flops": 7.0 * n * (qd + kvd)}
    pos, new = _shape(c)
    n = sum(new)
    if c["op"] == "append":
        # the rows in, the turned queries and the codes out, and the touched pages read back as bf16
        touched = sum((p + t - 1) // PAGE - p // PAGE + 1 for p, t in zip(pos, new))
        back = touched * (68 * kvd + PAGE * 2 * kvd * 2)
        return {"bytes": n * (2 * qd + 2 * kvd) * size + n * 68 * kvd // 64 + n * c["pdim"] * 4 + back,
                "flops": 7.0 * n * (qd + 2 * kvd)}
    spans, pairs = _visible(c)
    osize = 4 if c["out"] == "f32" else 2
    return {"bytes": sum(spans) * 68 * kvd // 64 + n * qd * (size + osize) + (n * c["heads"] * 4 if c["gate"] else 0),
            "flops": 4.0 * qd * sum(pairs)}


# ------------------------------------------------------------------ inputs


def _sm():
    folder = os.path.join(os.getcwd(), "spark-x2.6-4b-q6k_amd")
    if folder not in sys.path:
        sys.path.insert(1, folder)
    import sparkmv
    return sparkmv


def _codes(n, gen):
    """n bytes of two codes each, as normal values under a power of two have them."""
    out = torch.empty(n, dtype=torch.uint8, device="cuda")
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    for a in range(0, n, 1 << 24):
        m = min(1 << 24, n - a)
        x = 1.7 * torch.randn(m, 2, generator=gen, device="cuda")
        code = torch.bucketize(x.abs(), bounds, out_int32=True) + 8 * (x < 0).int()
        out[a:a + m] = (code[:, 0] + 16 * code[:, 1]).to(torch.uint8)
    return out


def _cache(c, gen, extra):
    """A pool with the sequences' pages in random order."""
    pos, new = _shape(c)
    need = [(p + t + PAGE - 1) // PAGE for p, t in zip(pos, new)]
    npages, kvh, hd = sum(need) + extra, c["kv_heads"], c["head_dim"]
    order = torch.randperm(npages, generator=gen, device="cuda").to(torch.int32)
    pages = torch.full((c["nseq"], max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(need):
        pages[i, :m] = order[at:at + m]
        at += m
    data = torch.empty(npages, kvh, 68 * hd, dtype=torch.uint8, device="cuda")
    data[:, :, :64 * hd] = _codes(npages * kvh * 64 * hd, gen).reshape(npages, kvh, 64 * hd)
    data[:, :, 64 * hd:] = (124 + torch.randint(0, 5, (npages, kvh, 4 * hd), generator=gen, device="cuda")).to(torch.uint8)
    starts = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    return {"data": data, "pages": pages, "pos": torch.tensor(pos, dtype=torch.int32, device="cuda"), "qstart": starts,
            "ntok": sum(new), "max_q": max(new), "max_len": max(p + t for p, t in zip(pos, new))}


def _rope(rows, pdim):
    """cos and sin of position * 10000^(-2 i / pdim), [rows][pdim]: the cosines, then the sines."""
    i = torch.arange(pdim // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * torch.pow(1.0e4, -2.0 * i / pdim)
    return torch.cat([a.cos(), a.sin()], dim=1).float().contiguous()


def _norms(c, gen):
    one = lambda: 1.0 + 0.3 * torch.randn(c["head_dim"], generator=gen, device="cuda")  # noqa: E731
    return {"q_norm": one() if c["norm"] else None, "k_norm": one() if c["norm"] else None, "eps": 1e-6}


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "table":
        # a table has no inputs but its frequencies: another seed, another base
        s["theta"] = c["theta"] * (1.0 + 0.01 * (seed % 97) / 97.0)
        s["table"] = torch.empty(c["rows"], c["pdim"], device="cuda")
        if own:
            sm = _sm()
            s["call"] = sm.rope_table_op(s["table"], s["theta"], sm.RopeScaling(c["kind"], c["factor"], c["original"]))
        return s
    heads, kvh, hd, x = c["heads"], c["kv_heads"], c["head_dim"], TYPES[c["x"]]
    if c["op"] == "rope":
        n = c["tokens"]
        s["qkv"] = torch.randn(n, heads + 2 * kvh, hd, generator=gen, device="cuda").to(x)
        first = int(torch.randint(0, 3000, (1,), generator=gen, device="cuda"))
        s["pos"] = (first + torch.arange(n, device="cuda")).to(torch.int32)
        s["rope"] = _rope(first + n, c["pdim"]) if c["pdim"] else None
        s.update(_norms(c, gen))
        s["q_out"] = torch.empty(n, heads, hd, dtype=x, device="cuda")
        s["k_out"] = torch.empty(n, kvh, hd, dtype=x, device="cuda")
        if own:
            q, k, _ = s["qkv"].split([heads, kvh, kvh], 1)
            s["call"] = _sm().qk_rope_op(s["pos"], q, s["q_out"], k, s["k_out"], rope=s["rope"], interleaved=c["inter"],
                                         q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"])
        return s
    s.update(_cache(c, gen, 7))
    ntok = s["ntok"]
    if own:
        sm = _sm()
        kv = sm.PagedKV4(kvh, hd, s["data"].shape[0], *s["pages"].shape, pages=s["pages"], data=s["data"])
        batch = sm.KVBatch(s["pos"], ntok, qstart=s["qstart"], max_q=s["max_q"], max_len=s["max_len"])
    if c["op"] == "append":
        qkv = torch.randn(ntok, heads + 2 * kvh, hd, generator=gen, device="cuda")
        # a few key channels are much larger than the others
        qkv[:, heads:heads + kvh] *= 1.0 + 5.0 * (torch.rand(kvh, hd, generator=gen, device="cuda") < 0.02)
        s["qkv"] = qkv.to(x)
        s["rope"] = _rope(s["pages"].shape[1] * PAGE, c["pdim"]) if c["pdim"] else None
        s.update(_norms(c, gen))
        s["q_out"] = torch.empty(ntok, heads, hd, dtype=x, device="cuda")
        pos, new = _shape(c)
        s["blocks"] = max((p + t - 1) // PAGE - p // PAGE + 1 for p, t in zip(pos, new))
        s["from"] = s["pos"] // PAGE * PAGE
        s["back"] = torch.zeros(2, c["nseq"], s["blocks"] * PAGE, kvh, hd, dtype=torch.bfloat16, device="cuda")
        if own:
            q, k, v = s["qkv"].split([heads, kvh, kvh], 1)
            s["call"] = kv.append_op(batch, q, k, v, s["rope"], s["q_out"], interleaved=c["inter"], q_norm=s["q_norm"],
                                     k_norm=s["k_norm"], eps=s["eps"])
            s["read"] = kv.read_op(s["from"], s["back"][0], s["back"][1])
        return s
    s["q"] = (1.5 * torch.randn(ntok, heads, hd, generator=gen, device="cuda")).to(x)
    s["gate"] = torch.randn(ntok, heads, generator=gen, device="cuda") if c["gate"] else None
    s["out"] = torch.empty(ntok, heads, hd, dtype=TYPES[c["out"]], device="cuda")
    if own:
        s["call"] = kv.attend_op(batch, s["q"], s["out"], scale=hd ** -0.5, window=c["window"], gate=s["gate"])
    return s


# ------------------------------------------------------------------ plain forms


def _plain_table(s):
    c = s["case"]
    d, theta, factor, original = c["pdim"], s["theta"], c["factor"], float(c["original"])
    i = torch.arange(d // 2, dtype=torch.float64, device="cuda")
    a = 1.0
    if c["kind"] == "ntk" and d > 2:
        theta = theta * factor ** (d / (d - 2))
    f = torch.pow(theta, -2.0 * i / d)
    if c["kind"] == "linear":
        f = f / factor
    elif c["kind"] == "yarn":
        at = lambda r: d * math.log(original / (2.0 * math.pi * r)) / (2.0 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        t = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        f = f * (1.0 - t) + f / factor * t
        a = 0.1 * math.log(factor) + 1.0
    elif c["kind"] == "bands":
        w = original * f / (2.0 * math.pi)
        t = (w - 1.0) / (4.0 - 1.0)
        f = torch.where(w > 4.0, f, torch.where(w < 1.0, f / factor, f * ((1.0 - t) / factor + t)))
    # positions of 131072 turn many times: angles in 64 bits
    p = torch.arange(c["rows"], dtype=torch.float64, device="cuda")[:, None] * f
    s["table"].copy_(torch.cat([p.cos() * a, p.sin() * a], 1))
    return s["table"]


def _turned(x, rows, inter):
    """x [n, heads, hd] turned by the table's rows, in x's type"""
    d = rows.shape[1]
    cos, sin = rows[:, None, :d // 2].to(x.dtype), rows[:, None, d // 2:].to(x.dtype)
    a, b = (x[..., 0:d:2], x[..., 1:d:2]) if inter else (x[..., :d // 2], x[..., d // 2:d])
    ya, yb = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([ya, yb], -1).flatten(-2) if inter else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., d:]], -1)


def _normed(x, w, eps):
    return x * (x * x).mean(-1, keepdim=True).add(eps).rsqrt() * w.to(x.dtype)


def _plain_rope(s):
    c = s["case"]
    q, k, _ = s["qkv"].float().split([c["heads"], c["kv_heads"], c["kv_heads"]], 1)
    for x, w, out in ((q, s["q_norm"], s["q_out"]), (k, s["k_norm"], s["k_out"])):
        if c["norm"]:
            x = _normed(x, w, s["eps"])
        if c["pdim"]:
            x = _turned(x, s["rope"][s["pos"].long()], c["inter"])
        out.copy_(x)
    return {"q": s["q_out"], "k": s["k_out"]}


def _tokens(s):
    """Each token's sequence, its place among the sequence's new ones, and its position."""
    t = torch.arange(s["ntok"], device="cuda")
    seq = torch.searchsorted(s["qstart"][1:].long(), t, right=True)
    at = t - s["qstart"].long()[seq]
    return seq, at, s["pos"].long()[seq] + at


def _key_bytes(hd):
    """Offsets of the code bytes and scales of keys in a page's kv head: [64][hd / 2], [64][hd / 32]"""
    p, i, b = torch.arange(PAGE)[:, None], torch.arange(hd // 2), torch.arange(hd // 32)
    t, c, part = p // 16, p % 16, hd // 8 if hd < 128 else 16
    g, j = i // part % 4, i // part // 4
    codes = (((t * max(hd // 128, 1) + j) * 4 + g) * 16 + c) * part + i % part
    scales = ((b % 4 * 16 + c) * 4 + t) * max(hd // 128, 1) + b // 4
    return codes.cuda(), (64 * hd + scales).cuda()


def _value_bytes(hd):
    p, i, b, n = torch.arange(PAGE)[:, None], torch.arange(hd // 2), torch.arange(hd // 32), hd // 16
    u, a, g, r = p // 32, p // 16 % 2, p // 4 % 4, p % 4
    c, byte = i // (n // 2), (a * 4 + r) * (n // 2) + i % (n // 2)
    codes = (((u * (n // 4) + byte // 16) * 4 + g) * 16 + c) * 16 + byte % 16
    scales = (g * (hd // 32) + b) * 16 + u * 8 + a * 4 + r
    return (32 * hd + codes).cuda(), (66 * hd + scales).cuda()


def _values(data, where, hd):
    """[n, kv head, position, hd] values of pages' data [n, kv head, 68 hd]"""
    codes, scales = data[:, :, where[0]], data[:, :, where[1]]
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device="cuda")
    x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    scale = torch.pow(2.0, scales.float() - 127.0).masked_fill(scales == 255, math.nan)
    return (x.unflatten(-1, (hd // 32, 32)) * scale[..., None]).flatten(-2)


def _held(x):
    """x [.., hd] in f32 as code bytes [.., hd / 2] and scale bytes [.., hd / 32]"""
    x = x.unflatten(-1, (-1, 32))
    most = x.abs().amax(-1)
    m, e = torch.frexp(most)
    e = torch.where(m <= 0.875, e - 3, e - 2)
    e = torch.where(most > 0, e, -120).clamp(-120, 125)
    y = x.abs().double() * torch.pow(2.0, -e.double())[..., None]
    code = ((y > 0.25).int() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0) + 8 * (x < 0)).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), (e + 127).to(torch.uint8)


def _plain_append(s):
    c = s["case"]
    heads, kvh, hd, nb, nseq = c["heads"], c["kv_heads"], c["head_dim"], s["blocks"], c["nseq"]
    _, _, p = _tokens(s)
    seq = _tokens(s)[0]
    # in 64 bits and rounded once: a code next to a border depends on it
    q, k, v = s["qkv"].double().split([heads, kvh, kvh], 1)
    if c["norm"]:
        q, k = _normed(q, s["q_norm"], s["eps"]), _normed(k, s["k_norm"], s["eps"])
    if c["pdim"]:
        q, k = _turned(q, s["rope"][p], c["inter"]), _turned(k, s["rope"][p], c["inter"])
    s["q_out"].copy_(q)
    page, h = s["pages"].long()[seq, p // PAGE], torch.arange(kvh, device="cuda")
    flat = s["data"].view(-1)
    base = ((page[:, None] * kvh + h) * (68 * hd))[:, :, None]
    where = _key_bytes(hd), _value_bytes(hd)
    for x, (codes, scales) in ((k, where[0]), (v, where[1])):
        code, scale = _held(x.float())
        flat[base + codes[p % PAGE][:, None, :]] = code
        flat[base + scales[p % PAGE][:, None, :]] = scale
    # read back: the touched pages
    at = s["from"].long()[:, None] // PAGE + torch.arange(nb, device="cuda")
    there = at < s["pages"].shape[1]
    page = s["pages"].long().gather(1, at.clamp(max=s["pages"].shape[1] - 1))
    there &= page >= 0
    for i in range(2):
        x = _values(s["data"][page.clamp(min=0).reshape(-1)], where[i], hd).reshape(nseq, nb, kvh, PAGE, hd)
        x = torch.where(there[:, :, None, None, None], x, 0.0)
        s["back"][i].copy_(x.transpose(2, 3).reshape(nseq, nb * PAGE, kvh, hd))
    return {"q": s["q_out"], "k": s["back"][0], "v": s["back"][1]}


def _plain_attend(s):
    c = s["case"]
    heads, kvh, hd, nseq = c["heads"], c["kv_heads"], c["head_dim"], c["nseq"]
    group, most = heads // kvh, s["max_q"]
    seq, at, p = _tokens(s)
    q = torch.zeros(nseq, most, heads, hd, device="cuda")
    q[seq, at] = s["q"].float()
    q = q.reshape(nseq, most, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(nseq, kvh, most * group, hd)
    npos = s["pages"].shape[1] * PAGE
    pages = s["data"][s["pages"].long().clamp(min=0).reshape(-1)]
    k = _values(pages, _key_bytes(hd), hd).reshape(nseq, -1, kvh, PAGE, hd).transpose(1, 2).reshape(nseq, kvh, npos, hd)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (hd ** -0.5)
    del k
    j = torch.arange(npos, device="cuda")
    where = s["pos"].long()[:, None] + torch.arange(most, device="cuda")
    seen = (j <= where[:, :, None]) & (j > where[:, :, None] - (c["window"] or npos + 1))
    x = x.reshape(nseq, kvh, most, group, npos).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    v = _values(pages, _value_bytes(hd), hd).reshape(nseq, -1, kvh, PAGE, hd).transpose(1, 2).reshape(nseq, kvh, npos, hd)
    y = torch.matmul(x.reshape(nseq, kvh, most * group, npos), v).reshape(nseq, kvh, most, group, hd) / total
    y = y.permute(0, 2, 1, 3, 4).reshape(nseq, most, heads, hd)[seq, at]
    if c["gate"]:
        y = y / (1.0 + (-s["gate"]).exp())[:, :, None]
    s["out"].copy_(y)
    return s["out"]


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"table": _plain_table, "rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[op](s)
    s["call"]()
    if op == "table":
        return s["table"]
    if op == "rope":
        return {"q": s["q_out"], "k": s["k_out"]}
    if op == "append":
        s["read"]()
        return {"q": s["q_out"], "k": s["back"][0], "v": s["back"][1]}
    return s["out"]


# ------------------------------------------------------------------ from the definitions, in 64 bits


def _exact_table(c, s):
    d, half = c["pdim"], c["pdim"] // 2
    theta, factor, original, out = s["theta"], c["factor"], c["original"], 1.0
    freq = []
    for i in range(half):
        base = theta * factor ** (d / (d - 2.0)) if c["kind"] == "ntk" and d > 2 else theta
        f = 1.0 / base ** (2.0 * i / d)
        turns = original * f / (2.0 * math.pi)       # of the original context
        if c["kind"] == "linear":
            f /= factor
        elif c["kind"] == "yarn":
            dims = [d * math.log(original / (n * 2.0 * math.pi)) / (2.0 * math.log(theta)) for n in (32.0, 1.0)]
            first, last = max(0, math.floor(dims[0])), min(d - 1, math.ceil(dims[1]))
            share = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = (1.0 - share) * f + share * (f / factor)
        elif c["kind"] == "bands":
            if turns < 1.0:
                f /= factor
            elif turns <= 4.0:
                share = (turns - 1.0) / 3.0
                f = share * f + (1.0 - share) * f / factor
        freq.append(f)
    if c["kind"] == "yarn":
        out = 1.0 + 0.1 * math.log(factor)
    angle = torch.outer(torch.arange(c["rows"], dtype=torch.float64, device="cuda"),
                        torch.tensor(freq, dtype=torch.float64, device="cuda"))
    table = torch.empty(c["rows"], d, dtype=torch.float64, device="cuda")
    table[:, :half], table[:, half:] = torch.cos(angle) * out, torch.sin(angle) * out
    return table


def _exact_heads(x, weight, eps, rope, pos, inter):
    """x [n, heads, hd] in numpy f64: normed and turned"""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt(np.mean(y ** 2, axis=2, keepdims=True) + eps) * weight
    if rope is not None:
        d = rope.shape[1]
        for i in range(d // 2):
            a, b = (2 * i, 2 * i + 1) if inter else (i, i + d // 2)
            cos, sin = rope[pos, i][:, None], rope[pos, i + d // 2][:, None]
            y[..., a], y[..., b] = y[..., a] * cos - y[..., b] * sin, y[..., b] * cos + y[..., a] * sin
    return y


def _exact_rope(c, s):
    wide = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    qkv, rope, pos, heads, kvh = wide(s["qkv"]), wide(s["rope"]), s["pos"].cpu().numpy(), c["heads"], c["kv_heads"]
    return {"q": _exact_heads(qkv[:, :heads], wide(s["q_norm"]), s["eps"], rope, pos, c["inter"]),
            "k": _exact_heads(qkv[:, heads:heads + kvh], wide(s["k_norm"]), s["eps"], rope, pos, c["inter"])}


def _place(position, d, hd):
    """Byte and half of element d's key code and value code, and the places of their scales, from the layout's definition"""
    t, c = divmod(position, 16)
    if hd == 64:
        g, rest = divmod(d, 16)
        key = ((t * 4 + g) * 16 + c) * 8 + rest // 2
        key_scale = (d // 32 * 16 + c) * 4 + t
    else:
        block, rest = divmod(d, 32)
        j, g = divmod(block, 4)
        key = (((t * (hd // 128) + j) * 4 + g) * 16 + c) * 16 + rest // 2
        key_scale = ((g * 16 + c) * 4 + t) * (hd // 128) + j
    n = hd // 16
    u, rest = divmod(position, 32)
    a, rest = divmod(rest, 16)
    g, b = divmod(rest, 4)
    lane, rest = divmod(d, n)
    piece, byte = divmod((a * 4 + b) * (n // 2) + rest // 2, 16)
    value = (((u * (n // 4) + piece) * 4 + g) * 16 + lane) * 16 + byte
    value_scale = ((g * (hd // 32) + d // 32) * 2 + u) * 8 + a * 4 + b
    return key, 64 * hd + key_scale, 32 * hd + value, 66 * hd + value_scale, d % 2


_PLACES = {}


def _places(hd):
    if hd not in _PLACES:
        _PLACES[hd] = np.array([[_place(p, d, hd) for d in range(hd)] for p in range(PAGE)])
    return _PLACES[hd]


def _read(data, hd):
    """Keys and values [64, hd] of a page's kv head (68 hd bytes, numpy)"""
    at = _places(hd)
    out = []
    for code, scale in ((at[..., 0], at[..., 1]), (at[..., 2], at[..., 3])):
        nibble = data[code].astype(np.int64) >> (4 * at[..., 4]) & 15
        out.append(np.array(VALUES)[nibble & 7] * np.where(nibble > 7, -1.0, 1.0) * np.exp2(data[scale].astype(np.float64) - 127.0))
    return out


def _nearest(x):
    """Values [.., 32] as the cache holds them, in f64"""
    most = np.abs(x).max(-1, keepdims=True)
    e = np.ceil(np.log2(np.where(most > 0, most, 1.0) / 7.0))
    e = np.where(most > 7.0 * np.exp2(e), e + 1, np.where(most <= 3.5 * np.exp2(e), e - 1, e))     # log2 rounds
    step = np.exp2(np.where(most > 0, np.clip(e, -120, 125), -120))
    levels = np.array(VALUES)
    y = np.abs(x) / step
    up = np.clip(np.searchsorted(levels, y, side="left"), 1, 7)
    low, high = levels[up - 1], levels[up]
    take = (y - low > high - y) | ((y - low == high - y) & (up % 2 == 0))
    return np.where(x < 0, -1.0, 1.0) * np.where(take, high, low) * step


def _exact_append(c, s):
    heads, kvh, hd = c["heads"], c["kv_heads"], c["head_dim"]
    wide = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    qkv, rope = wide(s["qkv"]), wide(s["rope"])
    pos, new = _shape(c)
    at = np.concatenate([np.arange(p, p + n) for p, n in zip(pos, new)])
    q = _exact_heads(qkv[:, :heads], wide(s["q_norm"]), s["eps"], rope, at, c["inter"])
    k = _exact_heads(qkv[:, heads:heads + kvh], wide(s["k_norm"]), s["eps"], rope, at, c["inter"])
    rows = k.astype(np.float32).astype(np.float64), qkv[:, heads + kvh:]
    held = [_nearest(x.reshape(-1, kvh, hd // 32, 32)).reshape(-1, kvh, hd) for x in rows]
    pages = s["pages"].cpu().numpy()
    back = np.zeros((2, c["nseq"], s["blocks"] * PAGE, kvh, hd))
    token = 0
    for n, (p, count) in enumerate(zip(pos, new)):
        first = p // PAGE
        for b in range(first, min(first + s["blocks"], pages.shape[1])):
            if pages[n, b] >= 0:
                data = s["data"][int(pages[n, b])].cpu().numpy()
                for h in range(kvh):
                    for i, x in enumerate(_read(data[h], hd)):
                        back[i, n, (b - first) * PAGE:(b - first + 1) * PAGE, h] = x
        for i in range(2):
            back[i, n, p - first * PAGE:p - first * PAGE + count] = held[i][token:token + count]
        token += count
    return {"q": q, "k": back[0], "v": back[1]}


def _exact_attend(c, s):
    """Sequence by sequence and kv head by kv head."""
    heads, kvh, hd = c["heads"], c["kv_heads"], c["head_dim"]
    at = torch.from_numpy(_places(hd)).cuda()
    level = torch.tensor(VALUES, dtype=torch.float64, device="cuda")
    pos, new = _shape(c)
    out = torch.zeros(s["ntok"], heads, hd, dtype=torch.float64, device="cuda")
    token = 0
    for n, (p, count) in enumerate(zip(pos, new)):
        last = p + count
        pages = s["pages"][n, :(last + PAGE - 1) // PAGE].long()
        sees = torch.arange(last, device="cuda")[None, :] <= p + torch.arange(count, device="cuda")[:, None]
        if c["window"]:
            sees &= torch.arange(last, device="cuda")[None, :] + c["window"] > p + torch.arange(count, device="cuda")[:, None]
        for h in range(kvh):
            data, kv = s["data"][pages, h], []
            for i in (0, 2):
                nibble = (data[:, at[..., i]].int() >> (4 * at[..., 4].int())) & 15
                x = level[nibble & 7] * torch.where(nibble > 7, -1.0, 1.0)
                kv.append((x * torch.exp2(data[:, at[..., i + 1]].double() - 127.0)).reshape(-1, hd)[:last])
            for j in range(h * (heads // kvh), (h + 1) * (heads // kvh)):
                score = s["q"][token:token + count, j].double() @ kv[0].T.contiguous() / math.sqrt(hd)
                weight = torch.softmax(score.masked_fill(~sees, -math.inf), 1)
                out[token:token + count, j] = weight @ kv[1]
        token += count
    if c["gate"]:
        out *= torch.sigmoid(s["gate"].double())[:, :, None]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"table": _exact_table, "rope": _exact_rope, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)
