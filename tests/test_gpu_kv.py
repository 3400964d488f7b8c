"""GPU tests of the paged 8-bit cache: the append, reading back and attention
over it, against the definitions in 64 bits (oracle/paged.py).

The append's arithmetic is fixed to the bit, so codes, scales and rotated
queries have to be equal. Attention's bound, per row and head, with u = 2^-24
(half a step of f32), S = the largest sum of |q_d k_d| * scale of a seen
position, W = the weighted sum of |v| and n positions:
  a score is off by at most (hd + 8) u S (hd products and sums, the scales), so
  a weight by twice that relative to the sum of weights, and the two sums over
  positions (in pages of 64 and then page by page, with a rescale each) by
  2 (80 + 2 n / 64) u: |out - exact| <= W (2 (hd + 8) S + 160 + n / 16) u.
A bf16 output is rounded once more (2^-8 of the value), and its scores and
weights may be held in 14 bits and more: a query element to 2^-15 of the row's
largest (Q = that times the sum of |k|, scaled, so a score by 2^-15 Q) and a
weight to 2^-15 of its page's largest, 64 of them at most: 2^-9 W in all."""
import numpy as np
import pytest

import paged

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Case:
    """A cache of random pages in random order, with nslots sequences of up to max_pages pages."""

    def __init__(self, sm, dev, kvh, hd, nslots, max_pages, seed, spare=3, fill=True):
        import torch
        self.rng = rng = np.random.default_rng(seed)
        self.sm, self.dev, self.kvh, self.hd = sm, dev, kvh, hd
        npages = nslots * max_pages + spare
        order = rng.permutation(npages)[:nslots * max_pages].reshape(nslots, max_pages)
        self.host = {"pages": order.astype(np.int32)}
        for n in "kv":
            codes = np.clip(np.rint(rng.standard_normal((npages, kvh, 64 * hd)) * 30), -127, 127)
            self.host[n] = (codes if fill else 0 * codes).astype(np.int8)
            self.host[n + "_scale"] = ((0.5 + rng.random((npages, kvh))) / 30).astype(np.float32)
        self.put()

    def put(self):
        import torch
        t = {n: torch.from_numpy(a.copy()).to(self.dev) for n, a in self.host.items()}
        self.kv = self.sm.PagedKV(self.kvh, self.hd, self.host["k"].shape[0], *self.host["pages"].shape, **t)
        return self.kv

    def ints(self, x):
        import torch
        return None if x is None else torch.tensor(np.asarray(x), dtype=torch.int32, device=self.dev)

    def batch(self, pos, ntok=None, qstart=None, slot=None, **kw):
        return self.sm.KVBatch(self.ints(pos), ntok, self.ints(qstart), self.ints(slot), **kw)

    def same(self):
        """The device's cache equals the host's."""
        for n in ("k_scale", "v_scale"):
            got, want = getattr(self.kv, n).cpu().numpy(), self.host[n]
            assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)]), n
        for n in "kv":
            assert np.array_equal(getattr(self.kv, n).cpu().numpy(), self.host[n]), n


def rows(dev, x, dtype):
    """numpy values as a device tensor of the type, and the type's values in f64"""
    import torch
    t = torch.from_numpy(np.asarray(x, np.float32)).to(dev).to(dtype)
    return t, t.double().cpu().numpy()


def types():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16}


SCENES = {   # (pos, count) per sequence; None counts: one token each
    "decode": ([0, 1, 62, 63, 64, 190, 127, 128], None),
    "chunks": ([0, 5, 63, 64, 100], [64, 3, 66, 128, 60]),
    "left out": ([3, -1, 70, 10, 5], [2, 4, 0, 1, 7]),
    "long": ([17], [190]),
}


@pytest.mark.parametrize("scene", list(SCENES))
@pytest.mark.parametrize("kvh,group,hd,rope,x", [(2, 4, 256, 64, "f32"), (4, 1, 64, 64, "bf16"), (1, 8, 128, 0, "f32"),
                                                (3, 2, 128, 90, "bf16"), (2, 2, 256, 256, "f32")])
def test_append_equals_the_definition(sm, dev, scene, kvh, group, hd, rope, x):
    import torch
    pos, count = SCENES[scene]
    c = Case(sm, dev, kvh, hd, len(pos), 4, 100 + len(pos) + hd)
    qstart = None if count is None else np.concatenate([[1], 1 + np.cumsum(count)])   # row 0 belongs to nobody
    ntok = len(pos) if count is None else int(qstart[-1]) + 2
    dt = types()[x]
    q, qf = rows(dev, c.rng.standard_normal((ntok, kvh * group, hd)), dt)
    k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)) * np.exp(c.rng.standard_normal((ntok, 1, 1))), dt)
    v, vf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), dt)
    table = sm.rope_table(4 * 64, rope, 1e4, dev) if rope else None
    q_out = torch.full((ntok, kvh * group, hd), 7.0, dtype=dt, device=dev)
    c.kv.append(c.batch(pos, ntok, qstart), q, k, v, table, q_out)
    want = paged.append(c.host, qf, kf, vf, table.cpu().numpy() if rope else None, pos, qstart)
    c.same()
    got = q_out.double().cpu().numpy()
    none = np.isnan(want)
    assert np.all(got[none] == 7.0)
    exact = torch.from_numpy(np.where(none, 7.0, want))
    if x == "f32":
        assert np.array_equal(got, exact.float().double().numpy())
    else:   # one rounding from 64 bits: half a step of bf16
        assert np.all(np.abs(got - exact.numpy()) <= 2.0 ** -8 * np.abs(exact.numpy()) * (1 + 1e-9) + 1e-40)


def test_append_one_by_one_and_cut_back(sm, dev):
    """Growing magnitudes grow a page's scale again and again; cut back, the
    page keeps its scale; cut back to its start, it is opened anew."""
    kvh, hd = 2, 128
    import torch
    c = Case(sm, dev, kvh, hd, 1, 2, 5, fill=False)
    for step, (p, f) in enumerate([(p, 1.2 ** (p % 20)) for p in range(70)] + [(66, 0.1), (67, 0.2), (64, 0.3), (65, 2.0), (9, 1e3)]):
        k, kf = rows(dev, c.rng.standard_normal((1, kvh, hd)) * f, torch.float32)
        v, vf = rows(dev, c.rng.standard_normal((1, kvh, hd)), torch.float32)
        c.kv.append(c.batch([p]), None, k, v)
        paged.append(c.host, None, kf, vf, None, [p])
        if step % 10 == 9 or step >= 70:
            c.same()


def test_append_many_sequences(sm, dev):
    """More sequences than a workgroup has threads, each with a few tokens."""
    import torch
    n, kvh, hd = 300, 1, 64
    c = Case(sm, dev, kvh, hd, n, 1, 83, fill=False)
    counts = c.rng.integers(0, 4, n)
    pos = c.rng.integers(-1, 60, n)
    qstart = np.concatenate([[0], np.cumsum(counts)])
    ntok = int(qstart[-1])
    q, qf = rows(dev, c.rng.standard_normal((ntok, 3, hd)), torch.bfloat16)
    k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.bfloat16)
    table = sm.rope_table(64, 32, 1e4, dev)
    q_out = torch.full_like(q, 5.0)
    c.kv.append(c.batch(pos, ntok, qstart), q, k, k, table, q_out)
    want = paged.append(c.host, qf, kf, kf, table.cpu().numpy(), pos, qstart)
    c.same()
    got, none = q_out.double().cpu().numpy(), np.isnan(want)
    assert np.all(got[none] == 5.0)
    assert np.all(np.abs(got - want)[~none] <= 2.0 ** -8 * np.abs(want[~none]) * (1 + 1e-9))


@pytest.mark.parametrize("what", ["nan", "inf", "zero", "tiny", "denormal", "huge", "ties", "f32 to bf16"])
def test_append_of_unusual_values(sm, dev, what):
    import torch
    kvh, hd = 2, 64
    c = Case(sm, dev, kvh, hd, 2, 2, 11)
    x = c.rng.standard_normal((80, kvh, hd))
    if what in ("nan", "inf"):
        x[3, 1, 5] = np.nan if what == "nan" else -np.inf
    elif what == "zero":
        x[:] = 0
    elif what == "tiny":
        x *= 1e-33
    elif what == "denormal":
        x *= 2e-44
    elif what == "huge":
        x *= 3.0e37
    elif what == "ties":       # the scale comes out as 2^-6 exactly (127 * 2^-6 is the largest), with halves of it about
        x = c.rng.integers(-254, 255, x.shape) / 128.0
        x[0, :, 0] = 254 / 128.0
    k, kf = rows(dev, x, torch.float32)
    b = c.batch([0, 30], 80, [0, 64, 80])
    for again in range(2):     # the second time over the first one's pages
        c.kv.append(b, None, k, k)
        paged.append(c.host, None, kf, kf, None, [0, 30], [0, 64, 80])
        c.same()


def test_append_leaves_bad_entries_out(sm, dev):
    """Slots outside the table, pages outside the pool, positions past the
    table, rows outside the call's, more tokens than max_q."""
    import torch
    kvh, hd = 2, 64
    c = Case(sm, dev, kvh, hd, 4, 2, 13)
    c.host["pages"][1] = [-1, 2]
    c.host["pages"][2] = [c.host["k"].shape[0], 1 << 30]
    c.host["pages"][3] = [-(1 << 31), 4]
    c.put()
    pos, slot = [60, 60, 60, 60, 0, 0, 127, 128, 5], [0, 1, 2, 3, 4, -1, 0, 1, 3]
    slot[6], pos[6] = 1, 127
    slot[0], slot[7] = 0, 2
    qstart = [0, 9, 18, 27, 36, 40, 44, 50, 55, 70]
    k, kf = rows(dev, c.rng.standard_normal((60, kvh, hd)), torch.float32)
    q, qf = rows(dev, c.rng.standard_normal((60, kvh, hd)), torch.float32)
    q_out = torch.full_like(q, 3.0)
    table = sm.rope_table(128, 64, 1e4, dev)
    # slot 1 twice, on pages of its own each time: 60 .. 67 and 127
    pos[1] = 56
    c.kv.append(c.batch(pos, 60, qstart, slot, max_q=8), q, k, k, table, q_out)
    want = paged.append(c.host, qf, kf, kf, table.cpu().numpy(), pos, qstart, slot, 8)
    c.same()
    got = q_out.double().cpu().numpy()
    assert np.array_equal(got, np.where(np.isnan(want), 3.0, want).astype(np.float32).astype(np.float64))


def test_append_from_one_matrix_and_in_place(sm, dev):
    """The forward's layout: q, k and v beside each other in a row, the queries
    rotated where they are."""
    import torch
    kvh, heads, hd = 2, 8, 128
    c = Case(sm, dev, kvh, hd, 3, 2, 17)
    qkv, f = rows(dev, c.rng.standard_normal((3, (heads + 2 * kvh) * hd + 8)), torch.float32)
    qd, kvd = heads * hd, kvh * hd
    table = sm.rope_table(128, 32, 5e6, dev)
    q = qkv[:, :qd]
    c.kv.append(c.batch([0, 64, 100]), q, qkv[:, qd:qd + kvd], qkv[:, qd + kvd:qd + 2 * kvd], table, q)
    want = paged.append(c.host, f[:, :qd].reshape(3, heads, hd), f[:, qd:qd + kvd].reshape(3, kvh, hd),
                        f[:, qd + kvd:qd + 2 * kvd].reshape(3, kvh, hd), table.cpu().numpy(), [0, 64, 100])
    c.same()
    assert np.array_equal(q.cpu().numpy().reshape(3, heads, hd), want.astype(np.float32))
    assert np.array_equal(qkv[:, qd:].double().cpu().numpy(), f[:, qd:])


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 256])
def test_read(sm, dev, x, hd):
    import torch
    kvh = 3
    c = Case(sm, dev, kvh, hd, 3, 3, 19)
    c.host["pages"][1, 1] = -1
    c.host["pages"][2, 0] = c.host["k"].shape[0] + 5
    c.put()
    slot, start, n = [0, 1, 2, 7, 0], [-70, 30, 50, 3, 150], 130
    k = torch.full((5, n, kvh, hd), 9.0, dtype=types()[x], device=dev)
    v = torch.full_like(k, 9.0)
    c.kv.read(c.ints(start), k, v, c.ints(slot))
    for got, w in ((k, 0), (v, 1)):
        want = np.stack([[paged.read(c.host, s, f + j, hd)[w] for j in range(n)] for s, f in zip(slot, start)])
        want = torch.from_numpy(want.astype(np.float32)).to(types()[x]).double().numpy()   # code * scale in f32, as said
        assert np.array_equal(got.double().cpu().numpy(), want)
    one = torch.full((5, n, kvh, hd), 9.0, dtype=types()[x], device=dev)
    c.kv.read(c.ints(start), None, one, c.ints(slot))
    assert torch.equal(one, v)


def check_attention(c, q, qf, out, scale, window, gate, pos, qstart, slot, max_q=1 << 30, note=""):
    want, size = paged.attend(c.host, qf, c.hd, scale, window, gate, pos, qstart, slot, max_q)
    got = out.double().cpu().numpy()
    none = np.isnan(want).all(-1)
    served = np.zeros(len(qf), bool)
    for _, _, a, n in paged.sequences(c.host, pos, qstart, slot, len(qf), max_q if qstart is not None else 1):
        served[a:a + n] = True
    assert np.all(got[~served] == 7.0), "rows of no sequence"
    bf16 = str(out.dtype).endswith("bfloat16")
    S, W, Q = size[..., 0], size[..., 1], size[..., 2]
    n = max(pos) + 1 + len(qf)
    bound = W * (2 * (c.hd + 8) * S + 160 + n / 16) * U
    if bf16:
        bound = bound + W * (2.0 ** -14 * Q + 2.0 ** -9) + 2.0 ** -8 * np.abs(np.nan_to_num(want)).max(-1)
    assert np.array_equal(np.isnan(got[served]), np.isnan(want[served])), note
    err = np.abs(np.where(np.isnan(want), 0, got - want))[served]
    bound = np.nan_to_num(bound)     # of a row that is NaN, whose error is taken as 0
    assert np.all(err <= bound[served][..., None] + 1e-30), (note, float((err / (bound[served][..., None] + 1e-30)).max()))
    norm = np.linalg.norm(np.nan_to_num(want[served]))
    rel = np.linalg.norm(err) / norm if norm else 0.0
    print(f"{note}: relL2 {rel:.2e}")
    return got, want


def attend(c, pos, qstart, slot, heads, x="f32", o="f32", window=0, gate=False, scale=None, max_q=None, q_scale=1.5, note=""):
    import torch
    ntok = len(pos) if qstart is None else int(qstart[-1]) + 1     # the last row belongs to nobody
    q, qf = rows(c.dev, c.rng.standard_normal((ntok, heads, c.hd)) * q_scale, types()[x])
    g = torch.from_numpy(c.rng.standard_normal((ntok, heads)).astype(np.float32)).to(c.dev) if gate else None
    out = torch.full((ntok, heads, c.hd), 7.0, dtype=types()[o], device=c.dev)
    c.kv.attend(c.batch(pos, ntok, qstart, slot, max_q=max_q, max_len=max(pos) + ntok), q, out, scale, window, g)
    return check_attention(c, q, qf, out, c.hd ** -0.5 if scale is None else scale, window,
                           None if g is None else g.double().cpu().numpy(), pos, qstart, slot,
                           1 << 30 if max_q is None else max_q, note)


@pytest.mark.parametrize("x,o", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("kvh,group,hd", [(2, 4, 256), (1, 1, 64), (2, 2, 128), (1, 3, 256), (2, 8, 64), (1, 16, 128), (1, 5, 256)])
def test_attend_decode(sm, dev, kvh, group, hd, x, o):
    """One token each, at every kind of length; slots in another order."""
    pos = [0, 1, 15, 16, 62, 63, 64, 65, 127, 128, 300, 700]
    c = Case(sm, dev, kvh, hd, len(pos), 11, 23 + hd)
    slot = list(c.rng.permutation(len(pos)))
    attend(c, pos, None, slot, kvh * group, x, o, note=f"kvh {kvh} group {group} hd {hd} {x} {o}")


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 100000])
@pytest.mark.parametrize("form", ["decode", "block", "chunk"])
def test_attend_window_and_gate(sm, dev, form, window):
    c = Case(sm, dev, 2, 128, 4, 10, 29)
    pos = [0, 70, 300, 511]
    qstart = {"decode": None, "block": [0, 5, 6, 13, 21], "chunk": [0, 90, 97, 230, 250]}[form]
    attend(c, pos, qstart, None, 8, window=window, gate=True, note=f"{form} window {window}")


@pytest.mark.parametrize("x,o", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("kvh,group,hd", [(2, 4, 256), (1, 1, 64), (2, 2, 128), (1, 3, 256), (1, 16, 64), (2, 5, 128)])
@pytest.mark.parametrize("counts", [[8, 1, 3], [2, 0, 2], [70, 33, 1], [150, 0, 64]])
def test_attend_several_tokens(sm, dev, kvh, group, hd, counts, x, o):
    c = Case(sm, dev, kvh, hd, 3, 6, 31 + hd)
    qstart = np.concatenate([[1], 1 + np.cumsum(counts)])
    attend(c, [0, 190, 130], qstart, None, kvh * group, x, o, note=f"{counts} kvh {kvh} group {group} hd {hd} {x}")


@pytest.mark.parametrize("x,o", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("kvh,group,hd,most,longest", [
    (2, 8, 64, 13, 700), (2, 8, 128, 13, 700), (2, 8, 256, 13, 700),     # up to 104 columns a sequence, split
    (4, 4, 64, 8, 700), (4, 4, 128, 8, 700), (4, 4, 256, 8, 700),        # up to 32
    (8, 8, 64, 17, 300), (8, 8, 128, 17, 300), (8, 4, 256, 8, 300)])     # short: whole
def test_attend_blocks_that_fill_the_card(sm, dev, kvh, group, hd, most, longest, x, o):
    """Enough tokens that a workgroup takes as many columns as a sequence gives;
    fewer tokens are taken in smaller tiles."""
    n = 16 if longest > 512 else 20
    c = Case(sm, dev, kvh, hd, n, longest // 64 + 2, 51 + hd + kvh)
    counts = [most - i % 4 for i in range(n)]
    counts[3], counts[7] = 0, 1
    pos = c.rng.integers(0, longest + 1, n).tolist()
    pos[0], pos[1] = longest, 0
    qstart = np.concatenate([[1], 1 + np.cumsum(counts)])
    attend(c, pos, qstart, None, kvh * group, x, o, note=f"kvh {kvh} group {group} hd {hd} blocks of up to {most}")


def test_attend_prompt_of_many_tiles(sm, dev):
    """A prompt from its first position: tiles of one page up to all."""
    c = Case(sm, dev, 2, 64, 2, 18, 57)
    attend(c, [0, 5], [0, 1100, 1117], None, 16, "bf16", "bf16", note="a prompt of 1100")


@pytest.mark.parametrize("o", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [None, [4, 9, 40]])
def test_attend_sharp_and_flat(sm, dev, counts, o):
    """Scores of hundreds, where one position has all the weight, and of zero."""
    qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    for q_scale in (40.0, 0.0):
        c = Case(sm, dev, 2, 128, 3, 12, 37)
        attend(c, [600, 64, 300], qstart, None, 8, "f32", o, q_scale=q_scale, note=f"queries of {q_scale}")
    c = Case(sm, dev, 2, 128, 3, 12, 38)
    attend(c, [600, 64, 300], qstart, None, 8, "f32", o, scale=-0.3, note="a negative scale")


@pytest.mark.parametrize("counts", [None, [1, 20, 20, 70]])
def test_attend_leaves_bad_entries_out(sm, dev, counts):
    """Missing pages are left out, a token with none gets zeros; bad slots and
    negative positions leave a sequence's rows alone."""
    c = Case(sm, dev, 2, 64, 4, 4, 41)
    c.host["pages"][0, 1] = -1
    c.host["pages"][1, :] = c.host["k"].shape[0]
    c.host["pages"][2, 0] = -5
    c.put()
    qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    got, _ = attend(c, [140, 100, 70, 180], qstart, None, 4, note="pages missing")
    row = 1
    assert np.all(got[row] == 0.0)
    attend(c, [140, 100, 70, 180], qstart, [9, -1, 2, 3], 4, note="slots missing")
    attend(c, [140, -3, 70, 180], qstart, [3, 0, 3, 3], 4, note="one slot three times")
    attend(c, [250, 255, 256, 1000], qstart, [3, 2, 1, 0], 4, note="past the table")
    if counts:
        attend(c, [140, 100, 70, 180], qstart, None, 4, max_q=6, note="max_q")


@pytest.mark.parametrize("counts", [None, [6, 6, 80]])
@pytest.mark.parametrize("window", [0, 40])
def test_attend_nan_pages(sm, dev, counts, window):
    """A page whose scale is NaN is NaN for the tokens that see any of it, and
    nothing for those that do not: behind them, or out of their window."""
    c = Case(sm, dev, 2, 128, 3, 5, 43)
    for s, blk, n in ((0, 1, "k_scale"), (1, 0, "v_scale"), (2, 3, "v_scale")):
        c.host[n][c.host["pages"][s, blk], 1] = np.nan
    c.put()
    qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    got, want = attend(c, [125, 90, 150], qstart, None, 8, window=window, note=f"NaN pages, window {window}")
    assert np.isnan(want).any() or window


def test_attend_bad_queries(sm, dev):
    """A query that is not finite makes its own head's output NaN and no other."""
    import torch
    for counts in (None, [3, 20]):
        c = Case(sm, dev, 2, 64, 2, 3, 47)
        pos, qstart = [100, 70], None if counts is None else [0, 3, 23]
        ntok = 2 if counts is None else 23
        q, qf = rows(dev, c.rng.standard_normal((ntok, 8, 64)), torch.float32)
        good = torch.full((ntok, 8, 64), 7.0, device=dev)
        b = c.batch(pos, ntok, qstart)
        c.kv.attend(b, q, good)
        q[1, 3, 7], q[0, 5, 0] = float("nan"), float("inf")
        out = torch.full((ntok, 8, 64), 7.0, device=dev)
        c.kv.attend(b, q, out)
        got, good = out.cpu().numpy(), good.cpu().numpy()
        assert np.isnan(got[1, 3]).all() and np.isnan(got[0, 5]).all()
        got[1, 3], got[0, 5] = good[1, 3], good[0, 5]
        assert np.array_equal(got, good)


@pytest.mark.parametrize("counts", [None, [3, 1, 2], [40, 3, 70]])
def test_attend_longer_than_said(sm, dev, counts):
    """max_len only shapes launches: sequences far past it, and far below, are
    served in full; so are more sequences than a wave has lanes."""
    import torch
    c = Case(sm, dev, 2, 64, 3, 60, 73)
    pos = [3500, 1, 2000]
    qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    ntok = 3 if counts is None else int(qstart[-1])
    q, qf = rows(dev, c.rng.standard_normal((ntok, 8, 64)), torch.float32)
    for max_len in (1, 0, 1 << 20):
        out = torch.full((ntok, 8, 64), 7.0, device=dev)
        c.kv.attend(c.batch(pos, ntok, qstart, max_len=max_len), q, out)
        check_attention(c, q, qf, out, 0.125, 0, None, pos, qstart, None, note=f"max_len {max_len}")


def test_attend_many_sequences(sm, dev):
    """More sequences than a wave has lanes, idle ones among them, over shared
    pages: decode steps short and long, and ragged blocks."""
    c = Case(sm, dev, 2, 64, 6, 40, 79)
    rng = np.random.default_rng(8)
    for n in (65, 300):
        slot = rng.integers(0, 6, n)
        for most in (200, 2400):
            pos = rng.integers(0, most, n)
            pos[rng.random(n) < 0.2] = -1
            attend(c, list(pos), None, list(slot), 4, note=f"{n} sequences up to {most}")
        counts = rng.integers(0, 4, n)
        pos = rng.integers(0, 600, n)
        attend(c, list(pos), np.concatenate([[0], np.cumsum(counts)]), list(slot), 4, "f32", "bf16", note=f"{n} ragged")


@pytest.mark.parametrize("form", ["one", "many", "block", "chunk"])
def test_attend_long(sm, dev, form):
    """Work split over a long axis and joined."""
    nseq = 1 if form != "many" else 9
    c = Case(sm, dev, 2, 128, nseq, 150, 53)
    pos = [9000] if nseq == 1 else [9000, 0, 64, 8000, 1, 2, 3, 500, 7000]
    qstart = {"one": None, "many": None, "block": [0, 7], "chunk": [0, 100]}[form]
    for o in ("f32", "bf16"):
        attend(c, pos, qstart, None, 8, "f32", o, note=f"long {form} {o}")
    attend(c, pos, qstart, None, 8, window=3000, note=f"long {form}, window")


def test_strides_streams_and_repeats(sm, dev):
    """Rows wider than their heads, a stream of the caller's, the same bits each time."""
    import torch
    c = Case(sm, dev, 2, 64, 5, 8, 59)
    pos, heads, ntok = [400, 3, 64, 200, 90], 8, 5
    q, qf = rows(dev, c.rng.standard_normal((ntok, heads * 64 + 24)), torch.float32)
    out = torch.full((ntok, heads * 64 + 8), 7.0, dtype=torch.bfloat16, device=dev)
    gate = torch.randn(ntok, heads + 3, device=dev)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream())
    b = c.batch(pos)
    c.kv.attend(b, q[:, :heads * 64], out[:, :heads * 64], gate=gate[:, :heads], stream=s)
    s.synchronize()
    assert torch.all(out[:, heads * 64:] == 7.0)
    check_attention(c, q, qf[:, :heads * 64].reshape(ntok, heads, 64), out[:, :heads * 64].reshape(ntok, heads, 64), 0.125, 0,
                    gate[:, :heads].double().cpu().numpy(), pos, None, None, note="strides")
    one = torch.empty(ntok, heads, 64, device=dev)
    two = torch.empty_like(one)
    qc = q[:, :heads * 64].contiguous()
    c.kv.attend(b, qc, one.view(ntok, -1))
    c.kv.attend(b, qc, two.view(ntok, -1))
    assert torch.equal(one, two)


@pytest.mark.parametrize("form", ["decode", "block"])
def test_capture_and_replay(sm, dev, form):
    """Append and attention recorded once and replayed as positions move, with
    eager calls on another cache between the replays."""
    import torch
    kvh, heads, hd, nseq = 2, 8, 128, 3
    c, e = (Case(sm, dev, kvh, hd, nseq, 6, 61, fill=False) for _ in range(2))
    per = 1 if form == "decode" else 5
    ntok = nseq * per
    qstart = None if form == "decode" else [0, 5, 10, 15]
    k, v = torch.zeros(ntok, kvh, hd, device=dev), torch.zeros(ntok, kvh, hd, device=dev)
    q, turned = torch.zeros(ntok, heads, hd, device=dev), torch.zeros(ntok, heads, hd, device=dev)
    out = torch.zeros(ntok, heads, hd, device=dev)
    pos = c.ints([0, 0, 0])
    table = sm.rope_table(6 * 64, hd, 1e4, dev)
    b = sm.KVBatch(pos, ntok, c.ints(qstart), max_q=per, max_len=384)
    ops = [c.kv.append_op(b, q, k, v, table, turned), c.kv.attend_op(b, turned, out)]
    eager = [e.kv.append_op(b, q, k, v, table, torch.zeros_like(turned))]
    eager_out, eager_q = torch.zeros_like(out), eager[0].keep[6]
    eager.append(e.kv.attend_op(b, eager_q, eager_out))
    stream = torch.cuda.Stream(device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for op in ops:
            op()
    at = np.array([0, 50, 120])
    for step in range(20):
        pos.copy_(torch.from_numpy(at.astype(np.int32)))
        for t in (q, k, v):
            t.copy_(torch.from_numpy(c.rng.standard_normal(t.shape).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        for op in eager:
            op()
        torch.cuda.synchronize()
        assert torch.equal(out, eager_out), step
        assert torch.equal(c.kv.k, e.kv.k) and torch.equal(c.kv.v_scale, e.kv.v_scale), step
        at = at + per
        if step == 10:
            at[1] -= 7      # a cut back sequence


def test_one_conversation(sm, dev):
    """A prompt in chunks, then tokens and verified blocks, two sequences at
    once: attention over the cache stays near attention over the values that
    were appended. Each cached value is off by at most 2.5 steps of its page's
    scale s, that is by 2.5 * 1.25 * (largest in the page) / 127 < 0.025 of it."""
    import torch
    kvh, heads, hd = 2, 8, 128
    c = Case(sm, dev, kvh, hd, 2, 8, 67, fill=False)
    table = sm.rope_table(8 * 64, hd, 1e4, dev)
    tab = table.cpu().numpy()
    lens, kept = [0, 0], [[], []]
    for counts in ([130, 40], [1, 1], [1, 0], [5, 8], [1, 1], [64, 3], [1, 1]):
        ntok = sum(counts)
        qstart = np.concatenate([[0], np.cumsum(counts)])
        q, qf = rows(dev, c.rng.standard_normal((ntok, heads, hd)), torch.float32)
        k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.float32)
        v, vf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.float32)
        out = torch.full((ntok, heads, hd), 7.0, device=dev)
        b = c.batch(lens, ntok, qstart)
        c.kv.append(b, q, k, v, table, q)
        c.kv.attend(b, q, out)
        want_q = paged.append(c.host, qf, kf, vf, tab, lens, qstart)
        c.same()
        got, want = check_attention(c, q, want_q, out, hd ** -0.5, 0, None, lens, qstart, None, note=str(counts))
        for s in range(2):
            for j in range(counts[s]):
                r = qstart[s] + j
                kept[s].append((paged.rotate(kf[r], tab[lens[s] + j]), vf[r]))
            for p in range(len(kept[s])):
                kc, vc = paged.read(c.host, s, p, hd)
                page = c.host["pages"][s, p // 64]
                assert np.all(np.abs(kc - kept[s][p][0]) <= 3 * c.host["k_scale"][page][:, None] * (1 + 1e-6))
                assert np.all(np.abs(vc - kept[s][p][1]) <= 3 * c.host["v_scale"][page][:, None] * (1 + 1e-6))
            lens[s] += counts[s]


def test_binding_refusals(sm, dev):
    import torch
    c = Case(sm, dev, 2, 64, 2, 2, 71)
    x = torch.zeros(2, 2, 64, device=dev)
    q = torch.zeros(2, 4, 64, device=dev)
    b = c.batch([0, 0])
    for call, text in (
            (lambda: c.kv.append(b, None, x.half(), x), "type"), (lambda: c.kv.append(b, None, x, x[:1]), "1 rows"),
            (lambda: c.kv.append(b, q, x, x), "do not agree"), (lambda: c.kv.append(b, None, x[:, :1], x), "shape"),
            (lambda: c.kv.append(b, None, x.cpu(), x), "on cpu"), (lambda: c.kv.attend(b, q[:, :3], q), "shape"),
            (lambda: c.kv.attend(b, q[:, :3].contiguous(), q[:, :3].contiguous()), "query heads"),
            (lambda: c.kv.attend(b, q, q.transpose(1, 2).contiguous().transpose(1, 2)), "side by side"),
            (lambda: c.kv.read(c.ints([0, 0])), "nothing"), (lambda: sm.KVBatch(c.ints([0, 0]).long()), "type"),
            (lambda: sm.KVBatch(c.ints([0, 0]), 2, c.ints([0, 1])), "shape"),
            (lambda: sm.PagedKV(2, 64, 9, 2, 2, pages=c.kv.pages, k=c.kv.k), "shape"),
            (lambda: c.kv.append(b, None, x, x, torch.zeros(127, 64, device=dev)), "does not cover")):
        with pytest.raises(sm.SparkmvError, match=text):
            call()
