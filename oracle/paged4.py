"""The paged 4-bit cache, attention over it, head norms with the rotation and
scaled rotary tables from their definitions (include/sparkmv.h), in numpy and 64
bits. Test infrastructure."""
import math

import numpy as np

from paged import PAGE, sequences

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def offsets(hd):
    """[4][position][hd]: the bytes of a page's kv head that hold the key code, key
    scale, value code and value scale of an element."""
    p, d = np.arange(PAGE)[:, None], np.arange(hd)[None, :]
    t, c, u, a, g, b, n, block = p // 16, p % 16, p // 32, p // 16 % 2, p // 4 % 4, p % 4, hd // 16, d // 32
    if hd == 64:
        kc, ks = ((t * 4 + d // 16) * 16 + c) * 8 + d % 16 // 2, (block * 16 + c) * 4 + t
    else:
        kc = (((t * (hd // 128) + block // 4) * 4 + block % 4) * 16 + c) * 16 + d % 32 // 2
        ks = ((block % 4 * 16 + c) * 4 + t) * (hd // 128) + block // 4
    y = (4 * a + b) * (n // 2) + d % n // 2
    vc = (((u * (n // 4) + y // 16) * 4 + g) * 16 + d // n) * 16 + y % 16
    vs = (g * (hd // 32) + block) * 16 + 8 * u + 4 * a + b
    return np.stack([kc, 64 * hd + ks, 32 * hd + vc, 66 * hd + vs])


def turn(x, row=None, interleaved=False, weight=None, eps=0.0):
    """x [heads, hd] (f64) normed by weight [hd] and turned by a table row [rope_dim]."""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight
    if row is None:
        return y
    half = row.shape[0] // 2
    c, s = row[:half].astype(np.float64), row[half:].astype(np.float64)
    a = np.arange(half) * 2 if interleaved else np.arange(half)
    b = a + 1 if interleaved else a + half
    out = y.copy()
    out[:, a], out[:, b] = y[:, a] * c - y[:, b] * s, y[:, b] * c + y[:, a] * s
    return out


def held(x):
    """x [.., 32 n] (f64 of f32 values) as codes 0..15 of the same shape and scale bytes [.., n]."""
    b = x.reshape(x.shape[:-1] + (-1, 32))
    most = np.abs(b).max(-1)
    bad = ~np.isfinite(most)
    m, e = np.frexp(np.where(bad | (most == 0), 1.0, most))
    e = np.where(m <= 0.875, e - 3, e - 2)
    e = np.clip(np.where(most == 0, -120, e), -120, 125)
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.abs(b) / np.exp2(e.astype(np.float64))[..., None]
        code = ((y > 0.25) * 1 + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)) + 8 * np.signbit(b)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(x.shape), np.where(bad, 255, e + 127)


def append(cache, q, k, v, rope, pos, qstart=None, slot=None, max_q=1 << 30, interleaved=False, q_norm=None, k_norm=None,
           eps=0.0):
    """Updates cache (dict of data uint8 [npages, kvh, 68 hd] and pages) in place;
    returns q turned (f64, [ntok, heads, hd]; rows of no sequence are NaN)."""
    npages, kvh, _ = cache["data"].shape
    hd = k.shape[2]
    off = offsets(hd)
    q_out = np.full(q.shape, np.nan) if q is not None else None
    for s, p0, row, n in sequences(cache, pos, qstart, slot, k.shape[0], max_q if qstart is not None else 1):
        for j in range(n):
            p = p0 + j
            r = None if rope is None else rope[p]
            if q is not None:
                q_out[row + j] = turn(q[row + j], r, interleaved, q_norm, eps)
            page = int(cache["pages"][s, p // PAGE])
            if not 0 <= page < npages:
                continue
            with np.errstate(over="ignore", invalid="ignore"):
                kt = turn(k[row + j], r, interleaved, k_norm, eps).astype(np.float32).astype(np.float64)
            for x, w in ((kt, 0), (v[row + j], 2)):
                code, scale = held(x)
                data = cache["data"][page]
                data[:, off[w, p % PAGE, ::2]] = code[:, ::2] + 16 * code[:, 1::2]
                data[:, off[w + 1, p % PAGE, ::32]] = scale
    return q_out


def values(cache, page, hd):
    """(keys, values) [pages, kvh, 64, hd] that pages hold, NaN where a scale says so."""
    off, data = offsets(hd), cache["data"][page]
    out = []
    for w in (0, 2):
        nibble = data[..., off[w]] >> (np.arange(hd) % 2 * 4).astype(np.uint8) & 15
        scale = data[..., off[w + 1]].astype(np.float64)
        x = LEVELS[nibble & 7] * np.where(nibble > 7, -1.0, 1.0) * np.exp2(scale - 127.0)
        out.append(np.where(scale > 252, np.nan, x))
    return out


def read(cache, slot, p, hd):
    """(k, v) [kvh, hd] of a position; zeros without a page."""
    npages, kvh, _ = cache["data"].shape
    nslots, max_pages = cache["pages"].shape
    page = -1
    if 0 <= slot < nslots and 0 <= p < max_pages * PAGE:
        page = int(cache["pages"][slot, p // PAGE])
    if not 0 <= page < npages:
        return np.zeros((kvh, hd)), np.zeros((kvh, hd))
    return tuple(x[0][:, p % PAGE] for x in values(cache, [page], hd))


def attend(cache, q, hd, scale, window, gate, pos, qstart=None, slot=None, max_q=1 << 30):
    """(out, size): attention of q [ntok, heads, hd] (f64); rows of no sequence are
    NaN, and so is a row that sees a position with a NaN in it. size: per row and
    head the largest sum of |q_d k_d| * scale over the seen positions and the
    largest weighted sum of |v|, for error bounds."""
    npages, kvh, _ = cache["data"].shape
    ntok, heads, _ = q.shape
    out, size = np.full(q.shape, np.nan), np.zeros((ntok, heads, 2))
    group = heads // kvh
    for s, p0, row, n in sequences(cache, pos, qstart, slot, ntok, max_q if qstart is not None else 1):
        page = cache["pages"][s, :(p0 + n + PAGE - 1) // PAGE].astype(int)
        ok = (page >= 0) & (page < npages)
        kd, vd = (x.transpose(1, 0, 2, 3).reshape(kvh, -1, hd) for x in values(cache, np.where(ok, page, 0), hd))
        there = np.repeat(ok, PAGE)
        for j in range(n):
            p = p0 + j
            at = np.arange(max(0, p + 1 - window) if window else 0, p + 1)
            at = at[there[at]]
            for g in range(heads):
                k, v, x = kd[g // group][at], vd[g // group][at], q[row + j, g]
                if not len(at):
                    out[row + j, g] = 0.0
                    continue
                sc = k @ x * scale
                if not (np.isfinite(sc).all() and np.isfinite(v).all()):
                    continue
                w = np.exp(sc - sc.max())
                w /= w.sum()
                f = 1.0 / (1.0 + np.exp(-gate[row + j, g])) if gate is not None else 1.0
                out[row + j, g] = w @ v * f
                size[row + j, g] = (np.abs(k) @ np.abs(x)).max() * abs(scale), (w @ np.abs(v)).max()
    return out, size


def table(rows, d, theta, kind="none", factor=1.0, original=0.0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0, attention=None):
    """[rows, d] in f64: cosines, then sines of the scaled frequencies."""
    i = np.arange(d // 2)
    base = theta * factor ** (d / (d - 2.0)) if kind == "ntk" and d > 2 else theta
    f = base ** (-2.0 * i / d)
    if kind == "linear":
        f = f / factor
    elif kind == "yarn":
        at = [d * math.log(original / (r * 2.0 * math.pi)) / (2.0 * math.log(theta)) for r in (beta_fast, beta_slow)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
        t = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        f = (1.0 - t) * f + t * f / factor
    elif kind == "bands":
        turns = original * f / (2.0 * math.pi)
        s = (turns - low) / (high - low)
        f = np.where(turns > high, f, np.where(turns < low, f / factor, s * f + (1.0 - s) * f / factor))
    if attention is None:
        attention = 0.1 * math.log(factor) + 1.0 if kind == "yarn" else 1.0
    angle = np.arange(rows)[:, None] * f
    return np.concatenate([np.cos(angle) * attention, np.sin(angle) * attention], 1)
