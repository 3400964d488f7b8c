"""Operators of a serving step over several sequences, as timed and compared cases.

A step appends the new tokens' keys and values to a paged cache that holds
them in 8 bits (with the position rotation applied on the way), attends over
that cache, and answers with log probabilities. The model's own sizes are 16
query and 4 kv heads of 256 elements, sliding windows of 512 positions, a
rotated share of a quarter (full layers) or all (sliding layers) of a head,
chunks of up to 512 prompt tokens, blocks of 8 verified tokens and a
vocabulary of 131072; smaller heads are generic.

What the listed cases stand for:

  append-1         one token of one conversation: latency
  append-64        a decode step of 64 conversations of any length
  append-chunk     a whole prompt chunk of a sliding layer, bf16 activations
  append-ragged    several users' turns in one call, small heads
  attend-1         one token early in a conversation: latency
  attend-far       one token at the end of the longest context
  attend-48        a decode step of 48 conversations of very unequal lengths
  attend-window    a decode step of a sliding layer with its head gates
  attend-verify    blocks of 8 drafted tokens of three conversations
  attend-chunk     a prompt chunk deep in a long document
  logprobs-1       one decode step's answer, with alternatives
  logprobs-512     the scoring of a prompt chunk

The cache. A page holds 64 positions of every kv head; per page and kv head
there is one scale for the keys and one for the values, and a value is its
code (-127..127) times the scale. Codes of a page's kv head lie as
  keys    [head_dim / 64][position 64][64]
  values  [g 4][head_dim][t 4][i 4]       position = 16 t + 4 g + i.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

HEADS, KV_HEADS, HEAD_DIM, WINDOW, VOCAB = 16, 4, 256, 512, 131072
PAGE = 64
HEADROOM = 1.25     # a page that is not full yet gets a scale this much larger than its values need
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    m = {"heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM}
    return [
        {"name": "append-1", "op": "append", **m, "nseq": 1, "tokens": 1, "ctx": 1003, "pdim": 64, "x": "f32"},
        {"name": "append-64", "op": "append", **m, "nseq": 64, "tokens": 1, "ctx": 8000, "pdim": 64, "x": "f32"},
        {"name": "append-chunk", "op": "append", **m, "nseq": 1, "tokens": 512, "ctx": 1000, "pdim": 256, "x": "bf16"},
        {"name": "append-ragged", "op": "append", "heads": 8, "kv_heads": 8, "head_dim": 128, "nseq": 5, "tokens": 411,
         "ctx": 2000, "pdim": 128, "x": "bf16"},
        {"name": "attend-1", "op": "attend", **m, "nseq": 1, "tokens": 1, "ctx": 1003, "window": 0, "gate": False,
         "x": "f32", "out": "f32"},
        {"name": "attend-far", "op": "attend", **m, "nseq": 1, "tokens": 1, "ctx": 131071, "window": 0, "gate": False,
         "x": "f32", "out": "f32"},
        {"name": "attend-48", "op": "attend", **m, "nseq": 48, "tokens": 1, "ctx": 12000, "window": 0, "gate": False,
         "x": "f32", "out": "bf16"},
        {"name": "attend-window", "op": "attend", **m, "nseq": 24, "tokens": 1, "ctx": 5000, "window": WINDOW,
         "gate": True, "x": "f32", "out": "f32"},
        {"name": "attend-verify", "op": "attend", **m, "nseq": 3, "tokens": 8, "ctx": 6001, "window": 0, "gate": False,
         "x": "f32", "out": "f32"},
        {"name": "attend-chunk", "op": "attend", **m, "nseq": 1, "tokens": 512, "ctx": 16384, "window": 0,
         "gate": False, "x": "bf16", "out": "bf16"},
        {"name": "logprobs-1", "op": "logprobs", "rows": 1, "n": VOCAB, "k": 8, "x": "f32", "masked": False},
        {"name": "logprobs-512", "op": "logprobs", "rows": 512, "n": VOCAB, "k": 20, "x": "f32", "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "logprobs"))
    if op == "logprobs":
        return {"op": op, "rows": _log(rng, 1, 512), "n": _log(rng, 500, VOCAB), "k": rng.choice((0, 1, 5, 8, 20, 32)),
                "x": rng.choice(("f32", "f32", "bf16")), "masked": rng.random() < 0.3}
    hd = rng.choice((64, 128, 256, 256))
    kvh = rng.choice((1, 2, 4, 4, 8)) if hd < 256 else rng.choice((1, 2, 4, 4))
    group = rng.choice((1, 2, 4, 4, 8)) if hd < 256 else rng.choice((1, 2, 4, 4))
    heads = kvh * group
    c = {"op": op, "heads": heads, "kv_heads": kvh, "head_dim": hd, "x": rng.choice(("f32", "bf16"))}
    form = rng.choice(("decode", "decode", "block", "chunk"))
    if op == "append":
        c["nseq"] = _log(rng, 1, 64) if form == "decode" else _log(rng, 1, 8)
        c["tokens"] = {"decode": 1, "block": rng.randint(2, 16), "chunk": _log(rng, 17, 512)}[form]
        c["ctx"] = _log(rng, 1, 30000 if form == "decode" else 8000)
        c["pdim"] = rng.choice((0, hd // 4, hd // 2, hd))
        while c["nseq"] * c["tokens"] > 2048:
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
    if c["op"] == "logprobs":
        size = 4 if c["x"] == "f32" else 2
        return {"bytes": c["rows"] * (c["n"] * size + 4 + 8 + 8 * c["k"]), "flops": 4.0 * c["rows"] * c["n"]}
    qd, kvd = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    size = 4 if c["x"] == "f32" else 2
    pos, new = _shape(c)
    n = sum(new)
    if c["op"] == "append":
        # the rows in, the rotated queries and the codes out, the scales, and the touched pages read back as bf16
        touched = sum((p + t - 1) // PAGE - p // PAGE + 1 for p, t in zip(pos, new))
        back = touched * PAGE * 2 * kvd * 3
        return {"bytes": n * (2 * qd + 2 * kvd) * size + n * 2 * kvd + n * c["pdim"] * 4 + touched * c["kv_heads"] * 8 + back,
                "flops": 6.0 * n * (qd + 2 * kvd)}
    spans, pairs = _visible(c)
    osize = 4 if c["out"] == "f32" else 2
    return {"bytes": sum(spans) * 2 * kvd + sum(s // PAGE + 1 for s in spans) * c["kv_heads"] * 8 + n * qd * (size + osize)
            + (n * c["heads"] * 4 if c["gate"] else 0), "flops": 4.0 * qd * sum(pairs)}


# ------------------------------------------------------------------ inputs


def _sm():
    folder = os.path.join(os.getcwd(), "spark-x2.6-4b-q6k_amd")
    if folder not in sys.path:
        sys.path.insert(1, folder)
    import sparkmv
    return sparkmv


def _cache(c, gen, extra):
    """A pool with the sequences' pages in random order, codes as quantized normal values have them."""
    pos, new = _shape(c)
    need = [(p + t + PAGE - 1) // PAGE for p, t in zip(pos, new)]
    npages, kvh, hd = sum(need) + extra, c["kv_heads"], c["head_dim"]
    order = torch.randperm(npages, generator=gen, device="cuda").to(torch.int32)
    pages = torch.full((c["nseq"], max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(need):
        pages[i, :m] = order[at:at + m]
        at += m
    pool = []
    for _ in range(2):
        codes = torch.empty(npages, kvh, PAGE * hd, dtype=torch.int8, device="cuda")
        for a in range(0, npages, 256):
            n = min(256, npages - a)
            x = torch.randn(n, kvh, PAGE * hd, generator=gen, device="cuda")
            codes[a:a + n] = (x * 30.0).round_().clamp_(-127, 127).to(torch.int8)
        scale = (0.6 + 0.8 * torch.rand(npages, kvh, generator=gen, device="cuda")) / 30.0
        pool += [codes, scale]
    starts = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    return {"k": pool[0], "k_scale": pool[1], "v": pool[2], "v_scale": pool[3], "pages": pages,
            "pos": torch.tensor(pos, dtype=torch.int32, device="cuda"), "qstart": starts, "ntok": sum(new),
            "max_q": max(new), "max_len": max(p + t for p, t in zip(pos, new))}


def _rope(rows, pdim):
    """cos and sin of position * 10000^(-2 i / pdim), [rows][pdim]: the cosines, then the sines."""
    i = torch.arange(pdim // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * torch.pow(1.0e4, -2.0 * i / pdim)
    return torch.cat([a.cos(), a.sin()], dim=1).float().contiguous()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = TYPES[c["x"]]
    s = {"case": c}
    if c["op"] == "logprobs":
        rows, n, k = c["rows"], c["n"], c["k"]
        logits = torch.randn(rows, n, generator=gen, device="cuda") * 2.5
        peaks = torch.randint(0, n, (rows, 4), generator=gen, device="cuda")
        logits.scatter_add_(1, peaks, 9.0 * torch.rand(rows, 4, generator=gen, device="cuda"))
        if c["masked"]:       # a grammar leaves a part of the vocabulary
            logits[torch.rand(rows, n, generator=gen, device="cuda") < 0.4] = -math.inf
        s["logits"] = logits.to(x)
        # the given tokens: likely ones mostly
        t = torch.randint(0, n, (rows,), generator=gen, device="cuda")
        s["tokens"] = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.7, peaks[:, 0], t).to(torch.int32)
        s["tokens"] = torch.where(s["logits"].gather(1, s["tokens"].long()[:, None])[:, 0] == -math.inf,
                                  s["logits"].float().argmax(1).to(torch.int32), s["tokens"])
        s["logprob"] = torch.empty(rows, device="cuda")
        s["entropy"] = torch.empty(rows, device="cuda")
        s["top_id"] = torch.empty(rows, k, dtype=torch.int32, device="cuda")
        s["top_logprob"] = torch.empty(rows, k, device="cuda")
        if own:
            s["call"] = _sm().logprobs_op(s["logits"], s["tokens"], s["logprob"], s["entropy"], s["top_id"], s["top_logprob"])
        return s
    s.update(_cache(c, gen, 7))
    heads, kvh, hd, ntok = c["heads"], c["kv_heads"], c["head_dim"], s["ntok"]
    if own:
        sm = _sm()
        kv = sm.PagedKV(kvh, hd, s["k"].shape[0], *s["pages"].shape, pages=s["pages"], k=s["k"], v=s["v"],
                        k_scale=s["k_scale"], v_scale=s["v_scale"])
        batch = sm.KVBatch(s["pos"], ntok, qstart=s["qstart"], max_q=s["max_q"], max_len=s["max_len"])
    if c["op"] == "append":
        qkv = torch.randn(ntok, heads + 2 * kvh, hd, generator=gen, device="cuda")
        # a few key channels are much larger than the others
        qkv[:, heads:heads + kvh] *= 1.0 + 5.0 * (torch.rand(kvh, hd, generator=gen, device="cuda") < 0.02)
        s["qkv"] = qkv.to(x)
        s["rope"] = _rope(s["pages"].shape[1] * PAGE, c["pdim"]) if c["pdim"] else None
        s["q_out"] = torch.empty(ntok, heads, hd, dtype=x, device="cuda")
        pos, new = _shape(c)
        s["blocks"] = max((p + t - 1) // PAGE - p // PAGE + 1 for p, t in zip(pos, new))
        s["from"] = s["pos"] // PAGE * PAGE
        s["back"] = torch.zeros(2, c["nseq"], s["blocks"] * PAGE, kvh, hd, dtype=torch.bfloat16, device="cuda")
        if own:
            q, k, v = s["qkv"].split([heads, kvh, kvh], 1)
            s["call"] = kv.append_op(batch, q, k, v, s["rope"], s["q_out"])
            s["read"] = kv.read_op(s["from"], s["back"][0], s["back"][1])
        return s
    s["q"] = (1.5 * torch.randn(ntok, heads, hd, generator=gen, device="cuda")).to(x)
    s["gate"] = torch.randn(ntok, heads, generator=gen, device="cuda") if c["gate"] else None
    s["out"] = torch.empty(ntok, heads, hd, dtype=TYPES[c["out"]], device="cuda")
    if own:
        s["call"] = kv.attend_op(batch, s["q"], s["out"], scale=hd ** -0.5, window=c["window"], gate=s["gate"])
    return s


# ------------------------------------------------------------------ plain forms


def _tokens(s):
    """Each token's sequence, its place among the sequence's new ones, and its position."""
    t = torch.arange(s["ntok"], device="cuda")
    seq = torch.searchsorted(s["qstart"][1:].long(), t, right=True)
    at = t - s["qstart"].long()[seq]
    return seq, at, s["pos"].long()[seq] + at


def _key_codes(codes, hd):
    """[n, kv head, 64 * hd] codes of keys as [n, kv head, position, hd]."""
    return codes.reshape(*codes.shape[:2], hd // 64, PAGE, 64).permute(0, 1, 3, 2, 4).reshape(*codes.shape[:2], PAGE, hd)


def _value_codes(codes, hd):
    return codes.reshape(*codes.shape[:2], 4, hd, 4, 4).permute(0, 1, 4, 2, 5, 3).reshape(*codes.shape[:2], PAGE, hd)


def _key_layout(x):
    n, h, _, hd = x.shape
    return x.reshape(n, h, PAGE, hd // 64, 64).permute(0, 1, 3, 2, 4).reshape(n, h, PAGE * hd)


def _value_layout(x):
    n, h, _, hd = x.shape
    return x.reshape(n, h, 4, 4, 4, hd).permute(0, 1, 3, 5, 2, 4).reshape(n, h, PAGE * hd)


def _plain_append(s):
    c = s["case"]
    heads, kvh, hd, half, nseq, nb = c["heads"], c["kv_heads"], c["head_dim"], c["pdim"] // 2, c["nseq"], s["blocks"]
    seq, at, p = _tokens(s)
    # rotated in 64 bits and rounded once: a code next to a border depends on it
    q, k, v = s["qkv"].double().split([heads, kvh, kvh], 1)
    if half:
        cos, sin = s["rope"].double()[p][:, None, :half], s["rope"].double()[p][:, None, half:]
        turn = lambda x: torch.cat([x[..., :half] * cos - x[..., half:2 * half] * sin,  # noqa: E731
                                    x[..., half:2 * half] * cos + x[..., :half] * sin, x[..., 2 * half:]], -1)
        q, k = turn(q), turn(k)
    s["q_out"].copy_(q)
    block, row = p // PAGE - s["pos"].long()[seq] // PAGE, p % PAGE
    index = torch.arange(nb, device="cuda")
    first, end = s["pos"].long()[:, None] // PAGE + index, (s["pos"].long() + (s["qstart"][1:] - s["qstart"][:-1]).long())[:, None]
    touched = first * PAGE < end
    page = s["pages"].long().gather(1, first.clamp(max=s["pages"].shape[1] - 1))[touched]
    held = (s["pos"].long()[:, None] - first * PAGE).clamp(0, PAGE)[touched]
    full = ((first + 1) * PAGE <= end)[touched]
    isnew = torch.zeros(nseq, nb, PAGE, dtype=torch.bool, device="cuda")
    isnew[seq, block, row] = True
    isnew = isnew[touched]
    isold = torch.arange(PAGE, device="cuda") < held[:, None]
    for x, codes, scale, of, lay in ((k, s["k"], s["k_scale"], _key_codes, _key_layout),
                                     (v, s["v"], s["v_scale"], _value_codes, _value_layout)):
        new = torch.zeros(nseq, nb, PAGE, kvh, hd, dtype=torch.float64, device="cuda")
        new[seq, block, row] = x.float().double()
        new = new[touched].transpose(1, 2)
        was, step = of(codes[page], hd), scale[page].double()
        need = new.abs().amax((2, 3))
        keep = (held > 0)[:, None] & (need <= 127.0 * step)
        room = torch.where(full, 1.0, HEADROOM).double()[:, None]
        now = torch.where(keep, step, (need * room / 127.0).float().double())
        div = torch.where(now > 0, now, 1.0)[:, :, None, None]
        old = torch.where(keep[:, :, None, None], was.double(), (was.double() * step[:, :, None, None] / div).round())
        fresh = (new / div).round()
        got = torch.where(isnew[:, None, :, None], fresh, torch.where(isold[:, None, :, None], old, was.double()))
        codes[page] = lay(got.to(torch.int8))
        scale[page] = now.float()
    at = s["from"].long()[:, None] + torch.arange(nb * PAGE, device="cuda")
    inside = at < (end + PAGE - 1) // PAGE * PAGE
    page = s["pages"].long().gather(1, (at // PAGE).clamp(max=s["pages"].shape[1] - 1))[:, ::PAGE]
    for k, (codes, scale, of) in enumerate(((s["k"], s["k_scale"], _key_codes), (s["v"], s["v_scale"], _value_codes))):
        page_at = page.reshape(-1).clamp(min=0)
        x = of(codes[page_at], hd).float() * scale[page_at][:, :, None, None]
        x = x.transpose(1, 2).reshape(nseq, nb * PAGE, kvh, hd)
        s["back"][k].copy_(torch.where((inside & page.repeat_interleave(PAGE, 1).ge(0))[:, :, None, None], x, 0.0))
    return s


def _plain_attend(s):
    c = s["case"]
    heads, kvh, hd, nseq = c["heads"], c["kv_heads"], c["head_dim"], c["nseq"]
    group, most = heads // kvh, s["max_q"]
    seq, at, p = _tokens(s)
    q = torch.zeros(nseq, most, heads, hd, device="cuda")
    q[seq, at] = s["q"].float()
    q = q.reshape(nseq, most, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(nseq, kvh, most * group, hd)
    npos = s["pages"].shape[1] * PAGE
    page = s["pages"].long().clamp(min=0).reshape(-1)
    k = _key_codes(s["k"][page], hd).float() * s["k_scale"][page][:, :, None, None]
    k = k.reshape(nseq, -1, kvh, PAGE, hd).transpose(1, 2).reshape(nseq, kvh, npos, hd)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (hd ** -0.5)
    del k
    j = torch.arange(npos, device="cuda")
    where = s["pos"].long()[:, None] + torch.arange(most, device="cuda")
    seen = (j <= where[:, :, None]) & (j > where[:, :, None] - (c["window"] or npos + 1))
    x = x.reshape(nseq, kvh, most, group, npos).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    v = _value_codes(s["v"][page], hd).float() * s["v_scale"][page][:, :, None, None]
    v = v.reshape(nseq, -1, kvh, PAGE, hd).transpose(1, 2).reshape(nseq, kvh, npos, hd)
    y = torch.matmul(x.reshape(nseq, kvh, most * group, npos), v).reshape(nseq, kvh, most, group, hd) / total
    y = y.permute(0, 2, 1, 3, 4).reshape(nseq, most, heads, hd)[seq, at]
    if c["gate"]:
        y = y / (1.0 + (-s["gate"]).exp())[:, :, None]
    s["out"].copy_(y)
    return s


def _plain_logprobs(s):
    x = s["logits"].float()
    k = s["case"]["k"]
    most = x.amax(1, keepdim=True)
    e = (x - most).exp()
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    lse = most.double() + total.log()
    s["logprob"].copy_(x.gather(1, s["tokens"].long()[:, None]).double()[:, 0] - lse[:, 0])
    mean = torch.where(e > 0, e * (x - most), 0.0).sum(1, dtype=torch.float64) / total[:, 0]
    s["entropy"].copy_(total[:, 0].log() - mean)
    if k:
        top, at = torch.sort(x, dim=1, descending=True, stable=True)
        s["top_id"].copy_(at[:, :k])
        s["top_logprob"].copy_(top[:, :k].double() - lse)
    return s


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        s["call"]()
        if op == "append":
            s["read"]()
    else:
        {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[op](s)
    if op == "append":
        return {"q": s["q_out"], "k": s["back"][0], "v": s["back"][1], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "attend":
        return s["out"]
    return {"logprob": s["logprob"], "entropy": s["entropy"], "top_id": s["top_id"], "top_logprob": s["top_logprob"]}


# ------------------------------------------------------------------ from the definitions, in 64 bits


def _where(position, hd):
    """Offsets of a position's hd keys and hd values in their page's codes, from the layouts' definition."""
    d = np.arange(hd)
    t, g, i = position // 16, position % 16 // 4, position % 4
    return (d // 64) * (PAGE * 64) + position * 64 + d % 64, ((g * hd + d) * 4 + t) * 4 + i


def _exact_append(c, s):
    heads, kvh, hd, pdim = c["heads"], c["kv_heads"], c["head_dim"], c["pdim"]
    qkv = s["qkv"].double().cpu().numpy()
    rope = s["rope"].double().cpu().numpy() if pdim else None
    scales = {"k": s["k_scale"].cpu().numpy().copy(), "v": s["v_scale"].cpu().numpy().copy()}
    pages = s["pages"].cpu().numpy()
    pos, new = _shape(c)
    off = np.array([_where(r, hd) for r in range(PAGE)])     # [position][keys, values][hd]
    q_out = qkv[:, :heads].copy()
    back = {x: np.zeros((c["nseq"], s["blocks"] * PAGE, kvh, hd)) for x in "kv"}
    token = 0
    for n, (p, count) in enumerate(zip(pos, new)):
        at = token + np.arange(count)
        turned = qkv[at, :heads + kvh]
        if pdim:
            half = pdim // 2
            cos, sin = rope[p:p + count, None, :half], rope[p:p + count, None, half:]
            a, b = turned[..., :half].copy(), turned[..., half:pdim].copy()
            turned[..., :half], turned[..., half:pdim] = a * cos - b * sin, b * cos + a * sin
        q_out[at] = turned[:, :heads]
        rows = {"k": turned[:, heads:], "v": qkv[at, heads + kvh:]}
        token += count
        for b in range(p // PAGE, (p + count - 1) // PAGE + 1):
            lo, hi = max(p, b * PAGE), min(p + count, (b + 1) * PAGE)
            page, held = pages[n, b], lo - b * PAGE
            for which, name in enumerate("kv"):
                codes = s[name][int(page)].cpu().numpy()[:, off[:, which]].astype(np.float64)     # [kv head][position][hd]
                x = rows[name][lo - p:hi - p].astype(np.float32).astype(np.float64).transpose(1, 0, 2)
                for h in range(kvh):
                    big, step = np.abs(x[h]).max(), float(scales[name][page, h])
                    if not held or big > 127.0 * step:
                        wide = float(np.float32(big * (1.0 if hi == (b + 1) * PAGE else HEADROOM) / 127.0))
                        if held:
                            codes[h, :held] = np.rint(codes[h, :held] * step / wide)
                        step = wide
                        scales[name][page, h] = np.float32(step)
                    codes[h, held:held + hi - lo] = np.rint(x[h] / step) if step else 0.0
                    at_block = (b - p // PAGE) * PAGE
                    back[name][n, at_block:at_block + PAGE, h] = codes[h] * step
    return {"q": q_out, "k": back["k"], "v": back["v"], "k_scale": scales["k"].astype(np.float64),
            "v_scale": scales["v"].astype(np.float64)}


def _exact_attend(c, s):
    """Sequence by sequence and kv head by kv head."""
    heads, kvh, hd = c["heads"], c["kv_heads"], c["head_dim"]
    off = np.array([_where(r, hd) for r in range(PAGE)])
    off = torch.from_numpy(off).cuda()
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
            kd = (s["k"][pages, h][:, off[:, 0]].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, hd)[:last]
            vd = (s["v"][pages, h][:, off[:, 1]].double() * s["v_scale"][pages, h].double()[:, None, None]).reshape(-1, hd)[:last]
            for j in range(h * (heads // kvh), (h + 1) * (heads // kvh)):
                score = s["q"][token:token + count, j].double() @ kd.T.contiguous() / math.sqrt(hd)
                weight = torch.softmax(score.masked_fill(~sees, -math.inf), 1)
                out[token:token + count, j] = weight @ vd
        token += count
    if c["gate"]:
        out *= torch.sigmoid(s["gate"].double())[:, :, None]
    return out


def _exact_logprobs(c, s):
    x = s["logits"].double()
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    # the value first, then the lower index: one key of both
    n = x.shape[1]
    level = torch.unique(x, return_inverse=True)[1]
    at = (level * n + (n - 1 - torch.arange(n, device="cuda"))).topk(c["k"], 1)[1] if c["k"] else torch.empty(c["rows"], 0, dtype=torch.int64, device="cuda")
    return {"logprob": lp[torch.arange(c["rows"], device="cuda"), s["tokens"].long()],
            "entropy": -torch.where(p > 0, p * lp, 0.0).sum(1), "top_id": at.to(torch.int32), "top_logprob": lp.gather(1, at)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["op"]](case, s)
