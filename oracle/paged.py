"""The paged 8-bit cache, attention over it and log probabilities from their
definitions (include/sparkmv.h), in numpy and 64 bits. Test infrastructure."""
import numpy as np

PAGE = 64


def key_at(pos, d):
    return (d // 64) * (PAGE * 64) + pos * 64 + d % 64


def value_at(pos, d, hd):
    return ((pos // 4 % 4 * hd + d) * 4 + pos // 16) * 4 + pos % 4


def offsets(hd):
    """[2][position][hd]: where a page's keys and values lie."""
    p, d = np.arange(PAGE)[:, None], np.arange(hd)[None, :]
    return np.stack([key_at(p, d), value_at(p, d, hd)])


def rotate(x, row):
    """x [heads, hd] (f64) turned by a table row [rope_dim]."""
    half = row.shape[0] // 2
    c, s = row[:half].astype(np.float64), row[half:].astype(np.float64)
    out = x.copy()
    out[:, :half] = x[:, :half] * c - x[:, half:2 * half] * s
    out[:, half:2 * half] = x[:, half:2 * half] * c + x[:, :half] * s
    return out


def sequences(cache, pos, qstart, slot, ntok, max_q):
    """(slot, first position, first row, tokens) of the sequences a call serves."""
    out = []
    for i, p in enumerate(pos):
        a, b = (i, i + 1) if qstart is None else (int(qstart[i]), int(qstart[i + 1]))
        s = i if slot is None else int(slot[i])
        nslots, max_pages = cache["pages"].shape
        if not 0 <= s < nslots or p < 0 or a < 0 or b > ntok:
            continue
        n = min(b - a, max_q, max_pages * PAGE - p)
        if n > 0:
            out.append((s, int(p), a, n))
    return out


def append(cache, q, k, v, rope, pos, qstart=None, slot=None, max_q=1 << 30):
    """Updates cache (dict of k, v int8 [npages, kvh, 64 hd], k_scale, v_scale f32,
    pages) in place; returns q rotated (f64, [ntok, heads, hd]; rows of no
    sequence are NaN). q, k, v are f64 arrays of the inputs' values."""
    npages, kvh, _ = cache["k"].shape
    hd = k.shape[2]
    off = offsets(hd)
    q_out = np.full(q.shape, np.nan) if q is not None else None
    for s, p0, row, n in sequences(cache, pos, qstart, slot, k.shape[0], max_q if qstart is not None else 1):
        turn = (lambda x, p: rotate(x, rope[p])) if rope is not None else (lambda x, p: x)
        if q is not None:
            for j in range(n):
                q_out[row + j] = turn(q[row + j], p0 + j)
        for blk in range(p0 // PAGE, (p0 + n - 1) // PAGE + 1):
            page = int(cache["pages"][s, blk])
            if not 0 <= page < npages:
                continue
            lo, hi = max(p0, blk * PAGE), min(p0 + n, (blk + 1) * PAGE)
            held, full = lo - blk * PAGE, hi == (blk + 1) * PAGE
            for which, (name, x) in enumerate((("k", k), ("v", v))):
                with np.errstate(over="ignore"):
                    rows = np.stack([(turn(x[row + p - p0], p) if name == "k" else x[row + p - p0]) for p in range(lo, hi)])
                    rows = rows.astype(np.float32).astype(np.float64)
                scales = cache[name + "_scale"]
                for h in range(kvh):
                    codes = cache[name][page, h]
                    here = off[which]
                    was = float(scales[page, h]) if held else 0.0
                    need = float(np.abs(rows[:, h]).max()) if np.isfinite(rows[:, h]).all() else np.inf
                    if not np.isfinite(need) or np.isnan(was):
                        scales[page, h] = np.nan
                        codes[here[held:held + hi - lo]] = 0
                        continue
                    now = was
                    if not was > 0 or need > 127.0 * was:
                        now = max(float(np.float32(need * (1.0 if full else 1.25) / 127.0)), 2.0 ** -126)
                        scales[page, h] = now
                        old = codes[here[:held]].astype(np.float64)
                        codes[here[:held]] = np.rint(old * was / now)
                    new = np.rint(rows[:, h] / now)
                    assert np.abs(new).max() <= 127
                    codes[here[held:held + hi - lo]] = new
    return q_out


def read(cache, slot, p, hd):
    """(k, v) [kvh, hd] of a position; zeros without a page."""
    npages, kvh, _ = cache["k"].shape
    nslots, max_pages = cache["pages"].shape
    page = -1
    if 0 <= slot < nslots and 0 <= p < max_pages * PAGE:
        page = int(cache["pages"][slot, p // PAGE])
    if not 0 <= page < npages:
        return np.zeros((kvh, hd)), np.zeros((kvh, hd))
    off = offsets(hd)[:, p % PAGE]
    return tuple(cache[n][page][:, off[w]].astype(np.float64) * cache[n + "_scale"][page].astype(np.float64)[:, None]
                 for w, n in enumerate("kv"))


def attend(cache, q, hd, scale, window, gate, pos, qstart=None, slot=None, max_q=1 << 30):
    """(out, size): attention of q [ntok, heads, hd] (f64); rows of no sequence
    are NaN. size: per row and head, the largest sum of |q_d k_d| * scale over
    the seen positions, the weighted sum of |v| and the largest |q| sum |k| *
    scale, for error bounds."""
    npages, kvh, _ = cache["k"].shape
    ntok, heads, _ = q.shape
    out, size = np.full(q.shape, np.nan), np.zeros((ntok, heads, 3))
    off = offsets(hd)
    group = heads // kvh
    for s, p0, row, n in sequences(cache, pos, qstart, slot, ntok, max_q if qstart is not None else 1):
        last = p0 + n
        blocks = np.arange((last + PAGE - 1) // PAGE)
        page = cache["pages"][s, blocks].astype(int)
        ok = (page >= 0) & (page < npages)
        pg = np.where(ok, page, 0)
        for h in range(kvh):
            kd = cache["k"][pg, h][:, off[0]].astype(np.float64) * cache["k_scale"][pg, h].astype(np.float64)[:, None, None]
            vd = cache["v"][pg, h][:, off[1]].astype(np.float64) * cache["v_scale"][pg, h].astype(np.float64)[:, None, None]
            kd, vd, there = kd.reshape(-1, hd), vd.reshape(-1, hd), np.repeat(ok, PAGE)
            for j in range(n):
                p = p0 + j
                first = max(0, p + 1 - window) if window else 0
                at = np.arange(first, p + 1)
                at = at[there[at]]
                for g in range(h * group, (h + 1) * group):
                    if not len(at):
                        out[row + j, g] = 0.0
                        continue
                    x = q[row + j, g]
                    sc = kd[at] @ x * scale
                    w = np.exp(sc - sc.max())
                    w /= w.sum()
                    f = 1.0 / (1.0 + np.exp(-gate[row + j, g])) if gate is not None else 1.0
                    out[row + j, g] = w @ vd[at] * f
                    ak = np.abs(kd[at])
                    size[row + j, g] = ((ak @ np.abs(x)).max() * abs(scale), (w @ np.abs(vd[at])).max(),
                                        np.abs(x).max() * ak.sum(1).max() * abs(scale))
    return out, size


def seen_rows(cache, hd, window, pos, qstart=None, slot=None, max_q=1 << 30, ntok=None):
    """(row, kv head, keys, values) of every token of a call and kv head: what it
    sees, [positions, hd] in f64."""
    npages, kvh, _ = cache["k"].shape
    off = offsets(hd)
    for s, p0, row, n in sequences(cache, pos, qstart, slot, ntok, max_q if qstart is not None else 1):
        for j in range(n):
            p = p0 + j
            at = np.arange(max(0, p + 1 - window) if window else 0, p + 1)
            page = cache["pages"][s, at // PAGE].astype(int)
            at, page = at[(page >= 0) & (page < npages)], page[(page >= 0) & (page < npages)]
            for h in range(kvh):
                yield (row + j, h) + tuple(
                    np.take_along_axis(cache[m][page, h], off[w][at % PAGE], 1).astype(np.float64)
                    * cache[m + "_scale"][page, h].astype(np.float64)[:, None] for w, m in enumerate("kv"))


def attend_one(q, k, v, scale):
    """(out, weights, scores) of one query [hd] over keys and values [n, hd]."""
    s = k @ q * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    return w @ v, w, s


def attend_digits(q, k, v, scale, q_bits, w_bits, of_sum):
    """attend_one with the query and the weights as integers: q_bits below the
    power of two over the largest element; w_bits of each 64 positions' largest
    weight or, with of_sum, of their sum. Everything else in 64 bits."""
    ex = np.frexp(np.abs(q).max())[1]
    s = k @ np.rint(np.ldexp(q, q_bits - ex)) * np.ldexp(scale, int(ex) - q_bits)
    o, l, M = 0.0, 0.0, s.max()
    for a in range(0, len(s), PAGE):
        m = s[a:a + PAGE].max()
        p = np.exp(s[a:a + PAGE] - m)
        unit = 2.0 ** -w_bits * (p.sum() if of_sum else 1.0)
        o = o + np.exp(m - M) * (np.rint(p / unit) * unit @ v[a:a + PAGE])
        l = l + np.exp(m - M) * p.sum()
    return o / l


def attend_bound(q, k, v, scale, bf16):
    """How far an element of attend_one may be off, from the roundings that the
    call makes, u = 2^-24. With S the largest |score|, Q = largest |q| times the
    largest sum |k|, scaled, W the weighted sum of |v|, V the largest |v|, n positions:
      scores: the query's integer 2^-30 Q; three sums of digits' products, which
      are |score| and Q / 31 at most; five roundings of factors; the reference's
      and the difference's, 3 S; in the exponents of a page's, a share's and the
      join's factors 3 S each; each exponential 2 u: (21 S + Q / 8 + 10) u in all.
      A weight is off by that, relative to it, and so is their sum;
      sums over positions: two roundings a page in each of the two sums, and as
      many in a join, n / 16, and 32 for lanes, factors, division and gate;
      weights: 2^-30 of the largest of 64, u V.
    With bf16 outputs the query may be held to 2^-22 of its largest element, a
    weight to half of 2^-22.9 of its 64 positions' sum, 2^-17 V of all 64, and the
    output is rounded to half a step, 2^-8."""
    out, w, s = attend_one(q, k, v, scale)
    S, W, V = np.abs(s).max(), w @ np.abs(v), np.abs(v).max(0)
    Q = np.abs(q).max() * np.abs(k).sum(1).max() * abs(scale)
    b = 2.0 ** -24 * (W * (2 * (21 * S + Q / 8 + 10) + len(s) / 16 + 32) + V)
    if bf16:
        b = b + 2 * 2.0 ** -22 * Q * W + 2.0 ** -17 * V
        b = b + 2.0 ** -8 * (np.abs(out) + b)
    return b


def logprobs(x, tokens, k):
    """Rows of logits (f64): log probabilities of tokens, entropies, and the k
    largest logits' ids and log probabilities."""
    rows, n = x.shape
    lp, ent = np.full(rows, np.nan), np.full(rows, np.nan)
    ids, tops = np.full((rows, k), -1), np.full((rows, k), -np.inf)
    for r in range(rows):
        v = x[r]
        bad = np.isnan(v).any() or (v == np.inf).any()
        m = -np.inf if bad else v.max()
        with np.errstate(divide="ignore"):
            if m > -np.inf:
                lse = m + np.log(np.exp(v - m).sum())
                all_lp = v - lse
                p = np.exp(all_lp)
                ent[r] = -(p[p > 0] * all_lp[p > 0]).sum()
            else:
                all_lp, ent[r] = np.full(n, -np.inf), 0.0
        if bad:
            all_lp, ent[r] = np.full(n, np.nan), np.nan
        if tokens is not None and 0 <= tokens[r] < n:
            lp[r] = all_lp[tokens[r]]
        order = np.lexsort((np.arange(n), -np.where(np.isnan(v), -np.inf, v)))
        order = order[~np.isnan(v[order])][:k]
        ids[r, :len(order)], tops[r, :len(order)] = order, all_lp[order]
        if bad:
            tops[r] = np.nan
    return lp, ent, ids, tops


def model_step(f, caches, tables, tokens, slot, pos, qstart, after_append=None, of=None):
    """One paged step of a forward.Forward f (its weights and arithmetic; its f32
    cache is not touched): the final residual's logits of every token. caches:
    per layer, as append() takes them; tables: rope tables (full, sliding).
    after_append(li), when given, may put other codes into caches[li] before
    attention reads them. of: a module with another cache's append() and attend()."""
    import forward as fw
    put, look = (append, attend) if of is None else (of.append, of.attend)
    c = f.c
    hd, heads, kvh = c["head_dim"], c["heads"], c["kv_heads"]
    qd, kvd, n = heads * hd, kvh * hd, len(tokens)
    h = np.stack([f.embed[t].astype(np.float32) for t in tokens])
    for li, L in enumerate(f.layers):
        full = bool(L["full"])
        xn = np.stack([f.q(fw.rms_norm(x, L["in_norm"], c["eps"])) for x in h])
        qkv = np.stack([(L["qkv"] @ x).astype(np.float32) for x in xn]).astype(np.float64)
        gate = np.stack([(L["attn_gate"] @ x).astype(np.float32) for x in xn])
        q = put(caches[li], qkv[:, :qd].reshape(n, heads, hd), qkv[:, qd:qd + kvd].reshape(n, kvh, hd),
                   qkv[:, qd + kvd:].reshape(n, kvh, hd), tables[0 if full else 1], pos, qstart, slot)
        if after_append:
            after_append(li)
        out, _ = look(caches[li], q.astype(np.float32).astype(np.float64), hd, float(np.float32(1.0) / np.sqrt(np.float32(hd))),
                        0 if full else c["sliding_window"], gate.astype(np.float64), pos, qstart, slot)
        for t in range(n):
            a = out[t].reshape(qd).astype(np.float32)
            h[t] = (h[t] + (L["out"] @ f.q(a)).astype(np.float32)).astype(np.float32)
            x = f.q(fw.rms_norm(h[t], L["post_norm"], c["eps"]))
            act = (fw.gelu((L["gate"] @ x).astype(np.float32)) * (L["up"] @ x).astype(np.float32)).astype(np.float32)
            h[t] = (h[t] + (L["down"] @ f.q(act)).astype(np.float32)).astype(np.float32)
    return np.stack([(f.embed @ f.q(fw.rms_norm(x, f.norm, c["eps"]))).astype(np.float32) for x in h])
