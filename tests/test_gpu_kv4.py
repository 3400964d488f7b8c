"""GPU tests of the paged 4-bit cache: the append, reading back and attention over
it, against the definitions in 64 bits (oracle/paged4.py).

A key is rounded to f32 once after 64-bit arithmetic and everything behind it is
exact, so the cache has to be equal byte for byte, and so do the values read back.

Attention's bound, per row and head, with u = 2^-24 (half a step of f32), S the
largest sum of |q_d k_d| * scale of a seen position, W the weighted sum of |v|, n
positions. Every product of two bf16 numbers is exact in f32. The matrix
instruction's sums, four products at a time at least, each cut off (2 u) at worst:
hd / 4 of them in a score, n / 4 in an output; lower parts of a split number add
2^-8 of that. So a score is off by at most (hd + 8) u S with its factors, a weight
by twice that relative to the sum of weights (and 2 u for each exponential), the
sums by (n / 2 + 160) u with rescales, joins, division and gate:
  |out - exact| <= W (2 (hd + 8) S + 160 + n / 2) u.
bf16 outputs hold a weight to 2^-17 of itself (W 2^-17 more) and are rounded once
(2^-8 of the value)."""
import numpy as np
import pytest

import paged4
from paged import sequences
from test_gpu_kv import SCENES, rows, types

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Case:
    """A cache of random bytes, scales among them that no append writes, with
    nslots sequences of up to max_pages pages in random order; fill() gives the
    first positions of slots ordinary values."""

    def __init__(self, sm, dev, kvh, hd, nslots, max_pages, seed, spare=3):
        self.rng = rng = np.random.default_rng(seed)
        self.sm, self.dev, self.kvh, self.hd = sm, dev, kvh, hd
        npages = nslots * max_pages + spare
        order = rng.permutation(npages)[:nslots * max_pages].reshape(nslots, max_pages)
        self.host = {"pages": order.astype(np.int32), "data": rng.integers(0, 256, (npages, kvh, 68 * hd)).astype(np.uint8)}
        self.put()

    def put(self):
        import torch
        t = {n: torch.from_numpy(a.copy()).to(self.dev) for n, a in self.host.items()}
        self.kv = self.sm.PagedKV4(self.kvh, self.hd, self.host["data"].shape[0], *self.host["pages"].shape, **t)
        return self.kv

    def fill(self, lengths):
        """Ordinary values at positions 0 .. lengths[slot] - 1; what is behind them stays."""
        off, hd = paged4.offsets(self.hd), self.hd
        table = self.host["pages"]
        for s, n in enumerate(lengths):
            for blk in range((min(n, 64 * table.shape[1]) + 63) // 64):
                page, upto = table[s, blk], min(64, n - 64 * blk)
                if not 0 <= page < len(self.host["data"]):
                    continue
                for w in (1, 3):
                    at = off[w, :upto, ::32]
                    self.host["data"][page][:, at] = self.rng.integers(124, 129, (self.kvh,) + at.shape)
        self.put()

    def ints(self, x):
        import torch
        return None if x is None else torch.tensor(np.asarray(x), dtype=torch.int32, device=self.dev)

    def batch(self, pos, ntok=None, qstart=None, slot=None, **kw):
        return self.sm.KVBatch(self.ints(pos), ntok, self.ints(qstart), self.ints(slot), **kw)

    def same(self):
        assert np.array_equal(self.kv.data.cpu().numpy(), self.host["data"])


def check_rows(got, want, x, left=7.0):
    """Queries as tests/test_gpu_rope.py has them; rows of no sequence as they were."""
    import torch
    got, none = got.double().cpu().numpy(), np.isnan(want)
    assert np.all(got[none] == left)
    exact = np.where(none, left, want)
    # a turn keeps a pair's length: the largest turned element is the largest before it over
    # sqrt(2) at least
    most = np.abs(exact).max(-1, keepdims=True) * np.sqrt(2.0)
    half, small = (2.0 ** -24, 2.0 ** -49) if x == "f32" else (2.0 ** -8, 2.0 ** -20)
    assert np.all(np.abs(got - exact) <= half * np.abs(exact) * (1 + 1e-6) + small * most)


@pytest.mark.parametrize("scene", list(SCENES))
@pytest.mark.parametrize("kvh,group,hd,rope,inter,norm,x", [
    (2, 4, 256, 64, False, True, "f32"), (4, 1, 64, 64, True, False, "bf16"), (1, 8, 128, 0, False, True, "f32"),
    (3, 2, 128, 90, False, True, "bf16"), (2, 2, 256, 256, True, True, "f32"), (5, 3, 64, 6, False, False, "f32"),
    (1, 1, 128, 34, True, True, "bf16"), (2, 1, 256, 0, False, False, "bf16")])
def test_append_equals_the_definition(sm, dev, scene, kvh, group, hd, rope, inter, norm, x):
    import torch
    pos, count = SCENES[scene]
    c = Case(sm, dev, kvh, hd, len(pos), 4, 100 + len(pos) + hd)
    qstart = None if count is None else np.concatenate([[1], 1 + np.cumsum(count)])   # row 0 belongs to nobody
    ntok = len(pos) if count is None else int(qstart[-1]) + 2
    dt = types()[x]
    q, qf = rows(dev, c.rng.standard_normal((ntok, kvh * group, hd)), dt)
    k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)) * np.exp(3 * c.rng.standard_normal((ntok, 1, 1))), dt)
    v, vf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)) * np.exp(3 * c.rng.standard_normal((ntok, kvh, hd))), dt)
    table = sm.rope_table(4 * 64, rope, 1e4, dev, scaling=sm.RopeScaling()) if rope else None
    w = [rows(dev, 1 + 0.3 * c.rng.standard_normal(hd), torch.float32) if norm else (None, None) for _ in range(2)]
    q_out = torch.full((ntok, kvh * group, hd), 7.0, dtype=dt, device=dev)
    eps = float(np.float32(1e-5))
    c.kv.append(c.batch(pos, ntok, qstart), q, k, v, table, q_out, interleaved=inter, q_norm=w[0][0], k_norm=w[1][0], eps=eps)
    want = paged4.append(c.host, qf, kf, vf, table.cpu().numpy() if rope else None, pos, qstart, interleaved=inter,
                         q_norm=w[0][1], k_norm=w[1][1], eps=eps)
    c.same()
    check_rows(q_out, want, x)


def test_append_of_a_long_chunk_and_many_heads(sm, dev):
    """Enough work that a wave takes several heads, and more heads than fill one."""
    import torch
    for kvh, heads, hd, ntok, x in ((5, 25, 64, 700, "bf16"), (3, 9, 128, 900, "f32"), (4, 16, 256, 512, "f32")):
        c = Case(sm, dev, kvh, hd, 2, 16, 7 + hd)
        dt = types()[x]
        q, qf = rows(dev, c.rng.standard_normal((ntok, heads, hd)), dt)
        k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), dt)
        v, vf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), dt)
        nw, nwf = rows(dev, 1 + 0.3 * c.rng.standard_normal(hd), torch.float32)
        table = sm.rope_table(16 * 64, hd // 2, 1e4, dev)
        pos, qstart = [37, 5], [0, ntok - 60, ntok]
        q_out = torch.full_like(q, 7.0)
        c.kv.append(c.batch(pos, ntok, qstart), q, k, v, table, q_out, q_norm=nw, k_norm=nw, eps=0.25)
        want = paged4.append(c.host, qf, kf, vf, table.cpu().numpy(), pos, qstart, q_norm=nwf, k_norm=nwf, eps=0.25)
        c.same()
        check_rows(q_out, want, x)


def test_append_many_sequences(sm, dev):
    """More sequences than a wave has lanes, each with a few tokens, in any order of rows."""
    import torch
    n, kvh, hd = 300, 1, 64
    c = Case(sm, dev, kvh, hd, n, 1, 83)
    counts = c.rng.integers(0, 4, n)
    pos = c.rng.integers(-1, 60, n)
    qstart = np.concatenate([[0], np.cumsum(counts)])
    ntok = int(qstart[-1])
    q, qf = rows(dev, c.rng.standard_normal((ntok, 3, hd)), torch.bfloat16)
    k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.bfloat16)
    table = sm.rope_table(64, 32, 1e4, dev)
    q_out = torch.full_like(q, 7.0)
    c.kv.append(c.batch(pos, ntok, qstart), q, k, k, table, q_out)
    want = paged4.append(c.host, qf, kf, kf, table.cpu().numpy(), pos, qstart)
    c.same()
    check_rows(q_out, want, "bf16")


@pytest.mark.parametrize("what", ["nan", "inf", "zero", "tiny", "denormal", "huge", "ties", "minus zero"])
def test_append_of_unusual_values(sm, dev, what):
    import torch
    kvh, hd = 2, 64
    c = Case(sm, dev, kvh, hd, 2, 2, 11)
    x = c.rng.standard_normal((80, kvh, hd))
    if what in ("nan", "inf"):
        x[3, 1, 5] = np.nan if what == "nan" else -np.inf
    elif what == "zero":
        x[:] = 0
    elif what == "minus zero":
        x = np.where(c.rng.random(x.shape) < 0.5, -0.0, x)
    elif what in ("tiny", "denormal"):
        x *= 1e-36 if what == "tiny" else 2e-44
    elif what == "huge":
        x = np.clip(x * 2e38, -3.4e38, 3.4e38)
    elif what == "ties":
        x = c.rng.integers(-28, 29, x.shape) / 4.0
    k, kf = rows(dev, x, torch.float32)
    b = c.batch([0, 30], 80, [0, 64, 80])
    c.kv.append(b, None, k, k)
    paged4.append(c.host, None, kf, kf, None, [0, 30], [0, 64, 80])
    c.same()


def test_append_leaves_bad_entries_out(sm, dev):
    """Slots outside the table, pages outside the pool, positions past the
    table, rows outside the call's, more tokens than max_q."""
    import torch
    kvh, hd = 2, 64
    c = Case(sm, dev, kvh, hd, 4, 2, 13)
    c.host["pages"][1] = [-1, 2]
    c.host["pages"][2] = [c.host["data"].shape[0], 1 << 30]
    c.host["pages"][3] = [-(1 << 31), 4]
    c.put()
    pos, slot = [60, 56, 60, 60, 0, 0, 127, 128, 5, 3], [0, 1, 2, 3, 4, -1, 1, 2, 3, 1 << 30]
    low = -(1 << 31)
    qstart = [0, 9, 18, 27, 36, 40, 44, 50, 55, 70, low]
    k, kf = rows(dev, c.rng.standard_normal((60, kvh, hd)), torch.float32)
    q, qf = rows(dev, c.rng.standard_normal((60, kvh, hd)), torch.float32)
    q_out = torch.full_like(q, 7.0)
    table = sm.rope_table(128, 64, 1e4, dev)
    c.kv.append(c.batch(pos, 60, qstart, slot, max_q=8), q, k, k, table, q_out)
    want = paged4.append(c.host, qf, kf, kf, table.cpu().numpy(), pos, qstart, slot, 8)
    c.same()
    check_rows(q_out, want, "f32")


@pytest.mark.parametrize("inter", [False, True])
def test_append_with_a_table_and_weights_at_any_address(sm, dev, inter):
    import torch
    c = Case(sm, dev, 2, 128, 2, 4, 113)
    n, heads, rope = 9, 4, 128
    flat = torch.empty(4 * 64 * rope + 1, device=dev)
    table = flat[1:].view(4 * 64, rope)
    table.copy_(sm.rope_table(4 * 64, rope, 1e4, dev))
    w = torch.from_numpy(1 + 0.3 * c.rng.standard_normal(2 * 128 + 3).astype(np.float32)).to(dev)
    qn, kn = w[1:129], w[130:258]
    q, qf = rows(dev, c.rng.standard_normal((n, heads, 128)), torch.float32)
    k, kf = rows(dev, c.rng.standard_normal((n, 2, 128)), torch.float32)
    out, turned = torch.empty_like(q), torch.empty_like(q)
    pos, qstart, eps = [5, 70], [0, 4, 9], float(np.float32(1e-5))
    c.fill(pos)
    c.kv.append(c.batch(pos, n, qstart), q, k, k, table, out, inter, qn, kn, eps)
    at = torch.tensor([5, 6, 7, 8, 70, 71, 72, 73, 74], dtype=torch.int32, device=dev)
    sm.qk_rope(at, q, turned, None, None, table, inter, qn, None, eps)
    assert torch.equal(out, turned)
    want = np.stack([paged4.turn(qf[t], table.cpu().numpy()[int(at[t])], inter, qn.double().cpu().numpy(), eps) for t in range(n)])
    size = np.abs(want).max(-1, keepdims=True)
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -24 * np.abs(want) * (1 + 1e-6) + 2.0 ** -48 * size)
    aligned = [t.clone() for t in (table, kn)]
    other = Case(sm, dev, 2, 128, 2, 4, 113)
    other.host = {n: a.copy() for n, a in c.host.items()}
    other.put()
    other.kv.append(other.batch(pos, n, qstart), None, k, k, aligned[0], None, inter, None, aligned[1], eps)
    assert torch.equal(c.kv.data, other.kv.data) and not np.array_equal(c.kv.data.cpu().numpy(), c.host["data"])


def test_append_from_one_matrix_and_in_place(sm, dev):
    """The forward's layout: q, k and v beside each other in a row, the queries turned where they are."""
    import torch
    kvh, heads, hd = 2, 8, 128
    c = Case(sm, dev, kvh, hd, 3, 2, 17)
    for inter in (False, True):
        qkv, f = rows(dev, c.rng.standard_normal((3, (heads + 2 * kvh) * hd + 8)), torch.float32)
        qd, kvd = heads * hd, kvh * hd
        table = sm.rope_table(128, 90, 5e6, dev)
        q = qkv[:, :qd]
        c.kv.append(c.batch([0, 64, 100]), q, qkv[:, qd:qd + kvd], qkv[:, qd + kvd:qd + 2 * kvd], table, q, interleaved=inter)
        want = paged4.append(c.host, f[:, :qd].reshape(3, heads, hd), f[:, qd:qd + kvd].reshape(3, kvh, hd),
                             f[:, qd + kvd:qd + 2 * kvd].reshape(3, kvh, hd), table.cpu().numpy(), [0, 64, 100], interleaved=inter)
        c.same()
        check_rows(q.reshape(3, heads, hd), want, "f32")
        assert np.array_equal(qkv[:, qd:].double().cpu().numpy(), f[:, qd:])


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_read(sm, dev, x, hd):
    import torch
    kvh = 3
    c = Case(sm, dev, kvh, hd, 3, 3, 19)
    c.fill([192, 192, 100])
    off = paged4.offsets(hd)
    c.host["pages"][1, 1] = -1
    c.host["pages"][2, 0] = c.host["data"].shape[0] + 5
    for w in (1, 3):       # a NaN here and there
        at = off[w, 20, ::32][:1]
        c.host["data"][c.host["pages"][0, 0], 1, at] = 255
    c.put()
    slot, start, n = [0, 1, 2, 7, 0], [-70, 30, 50, 3, 100], 90
    k = torch.full((5, n, kvh, hd), 9.0, dtype=types()[x], device=dev)
    v = torch.full_like(k, 9.0)
    c.kv.read(c.ints(start), k, v, c.ints(slot))
    for got, w in ((k, 0), (v, 1)):
        want = np.stack([[paged4.read(c.host, s, f + j, hd)[w] for j in range(n)] for s, f in zip(slot, start)])
        assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)
        assert np.isnan(want).any()
    one = torch.full((5, n, kvh, hd), 9.0, dtype=types()[x], device=dev)
    c.kv.read(c.ints(start), None, one, c.ints(slot))
    assert np.array_equal(one.float().cpu().numpy(), v.float().cpu().numpy(), equal_nan=True)


def check_attention(c, q, qf, out, scale, window, gate, pos, qstart, slot, max_q=1 << 30, note=""):
    want, size = paged4.attend(c.host, qf, c.hd, scale, window, gate, pos, qstart, slot, max_q)
    got = out.double().cpu().numpy()
    served = np.zeros(len(qf), bool)
    for _, _, a, n in sequences(c.host, pos, qstart, slot, len(qf), max_q if qstart is not None else 1):
        served[a:a + n] = True
    assert np.all(got[~served] == 7.0), "rows of no sequence"
    bf16 = str(out.dtype).endswith("bfloat16")
    S, W = size[..., 0], size[..., 1]
    n = max(pos) + 1 + len(qf)
    bound = W * (2 * (c.hd + 8) * S + 160 + n / 2) * U
    if bf16:
        bound = bound + W * 2.0 ** -17 + 2.0 ** -8 * np.abs(np.nan_to_num(want)).max(-1)
    assert np.array_equal(np.isnan(got[served]), np.isnan(want[served])), note
    err = np.abs(np.where(np.isnan(want), 0, got - want))[served]
    assert np.all(err <= bound[served][..., None] + 1e-30), (note, float((err / (bound[served][..., None] + 1e-30)).max()))
    norm = np.linalg.norm(np.nan_to_num(want[served]))
    print(f"{note}: relL2 {np.linalg.norm(err) / norm if norm else 0.0:.2e}")
    return got, want


def attend(c, pos, qstart, slot, heads, x="f32", o="f32", window=0, gate=False, scale=None, max_q=None, q_scale=1.5, note="",
           max_len=None):
    import torch
    ntok = len(pos) if qstart is None else int(qstart[-1]) + 1     # the last row belongs to nobody
    q, qf = rows(c.dev, c.rng.standard_normal((ntok, heads, c.hd)) * q_scale, types()[x])
    g = torch.from_numpy(c.rng.standard_normal((ntok, heads)).astype(np.float32)).to(c.dev) if gate else None
    out = torch.full((ntok, heads, c.hd), 7.0, dtype=types()[o], device=c.dev)
    b = c.batch(pos, ntok, qstart, slot, max_q=max_q, max_len=max(pos) + ntok if max_len is None else max_len)
    c.kv.attend(b, q, out, scale, window, g)
    return check_attention(c, q, qf, out, c.hd ** -0.5 if scale is None else scale, window,
                           None if g is None else g.double().cpu().numpy(), pos, qstart, slot,
                           1 << 30 if max_q is None else max_q, note)


def lengths(pos, qstart, slot, nslots):
    """How much of each slot the call's tokens may see"""
    n = [0] * nslots
    for i, p in enumerate(pos):
        s = i if slot is None else int(slot[i])
        if 0 <= s < nslots and p >= 0:
            n[s] = max(n[s], int(p) + (1 if qstart is None else max(0, int(qstart[i + 1]) - int(qstart[i]))))
    return n


@pytest.mark.parametrize("x,o", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("kvh,group,hd", [(2, 4, 256), (1, 1, 64), (2, 2, 128), (1, 3, 256), (2, 8, 64), (1, 16, 128), (1, 5, 256),
                                          (1, 16, 256), (1, 16, 64)])
def test_attend_decode(sm, dev, kvh, group, hd, x, o):
    """One token each, at every kind of length; slots in another order."""
    pos = [0, 1, 15, 16, 62, 63, 64, 65, 127, 128, 300, 700]
    c = Case(sm, dev, kvh, hd, len(pos), 11, 23 + hd)
    slot = list(c.rng.permutation(len(pos)))
    c.fill(lengths(pos, None, slot, len(pos)))
    for max_len in (700, 4000):     # whole contexts a workgroup, and shares
        attend(c, pos, None, slot, kvh * group, x, o, note=f"kvh {kvh} group {group} hd {hd} {x} {o} {max_len}", max_len=max_len)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 100000, (1 << 31) - 1])
@pytest.mark.parametrize("form", ["decode", "block", "chunk"])
def test_attend_window_and_gate(sm, dev, form, window):
    c = Case(sm, dev, 2, 128, 4, 12, 29)
    pos = [0, 70, 300, 511]
    qstart = {"decode": None, "block": [0, 5, 6, 13, 21], "chunk": [0, 90, 97, 230, 250]}[form]
    c.fill(lengths(pos, qstart, None, 4))
    attend(c, pos, qstart, None, 8, window=window, gate=True, note=f"{form} window {window}")
    attend(c, pos, qstart, None, 4, "bf16", "bf16", window=window, gate=True, note=f"{form} window {window}, bf16", max_len=9000)


@pytest.mark.parametrize("x,o", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("kvh,group,hd", [(2, 4, 256), (1, 1, 64), (2, 2, 128), (1, 3, 256), (1, 16, 64), (2, 5, 128)])
@pytest.mark.parametrize("counts", [[8, 1, 3], [2, 0, 2], [70, 33, 1], [150, 0, 64]])
def test_attend_several_tokens(sm, dev, kvh, group, hd, counts, x, o):
    c = Case(sm, dev, kvh, hd, 3, 6, 31 + hd)
    qstart = np.concatenate([[1], 1 + np.cumsum(counts)])
    pos = [0, 190, 130]
    c.fill(lengths(pos, qstart, None, 3))
    attend(c, pos, qstart, None, kvh * group, x, o, note=f"{counts} kvh {kvh} group {group} hd {hd} {x}")


def test_attend_prompt_of_many_tiles(sm, dev):
    """A prompt from its first position: tiles of one page up to all."""
    c = Case(sm, dev, 2, 64, 2, 18, 57)
    qstart = [0, 1100, 1117]
    c.fill(lengths([0, 5], qstart, None, 2))
    attend(c, [0, 5], qstart, None, 16, "bf16", "bf16", note="a prompt of 1100")


@pytest.mark.parametrize("o", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [None, [4, 9, 40]])
def test_attend_sharp_and_flat(sm, dev, counts, o):
    """Scores of hundreds, where one position has all the weight, and of zero."""
    qstart, pos = None if counts is None else np.concatenate([[0], np.cumsum(counts)]), [600, 64, 300]
    c = Case(sm, dev, 2, 128, 3, 12, 37)
    c.fill(lengths(pos, qstart, None, 3))
    for q_scale in (40.0, 0.0):
        attend(c, pos, qstart, None, 8, "f32", o, q_scale=q_scale, note=f"queries of {q_scale}")
    attend(c, pos, qstart, None, 8, "f32", o, scale=-0.3, note="a negative scale")
    attend(c, pos, qstart, None, 8, "f32", o, scale=0.0, note="a scale of zero")


@pytest.mark.parametrize("counts", [None, [1, 20, 20, 70]])
def test_attend_leaves_bad_entries_out(sm, dev, counts):
    """Missing pages are left out, a token with none gets zeros; bad slots and
    negative positions leave a sequence's rows alone."""
    c = Case(sm, dev, 2, 64, 4, 4, 41)
    c.fill([256] * 4)
    c.host["pages"][0, 1] = -1
    c.host["pages"][1, :] = c.host["data"].shape[0]
    c.host["pages"][2, 0] = -5
    c.put()
    qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    got, _ = attend(c, [140, 100, 70, 180], qstart, None, 4, note="pages missing")
    assert np.all(got[1] == 0.0)
    attend(c, [140, 100, 70, 180], qstart, [9, -1, 2, 3], 4, note="slots missing")
    attend(c, [140, -3, 70, 180], qstart, [3, 0, 3, 3], 4, note="one slot three times")
    attend(c, [250, 255, 256, 1000], qstart, [3, 2, 1, 0], 4, note="past the table")
    if counts:
        attend(c, [140, 100, 70, 180], qstart, None, 4, max_q=6, note="max_q")
        low = -(1 << 31)
        attend(c, [140, 100, 70, 180, 5], [0, 4, low, 4, 9, 30], None, 4, note="rows that fall")


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("counts", [None, [6, 6, 80]])
@pytest.mark.parametrize("window", [0, 40])
def test_attend_nan(sm, dev, counts, window, hd):
    """32 elements that read as NaN are NaN for the tokens that see them, and nothing
    for those that do not: behind them, or out of their window."""
    c = Case(sm, dev, 2, hd, 3, 5, 43)
    pos = [125, 90, 150]
    qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    c.fill(lengths(pos, qstart, None, 3))
    off = paged4.offsets(hd)
    for s, p, w, block in ((0, 100, 1, 0), (1, 95, 3, 1), (2, 153, 3, 0), (2, 0, 1, 1)):
        c.host["data"][c.host["pages"][s, p // 64], 1, off[w, p % 64, 32 * block]] = 255
    c.put()
    for o in ("f32", "bf16"):
        got, want = attend(c, pos, qstart, None, 8, o=o, window=window, note=f"NaN, window {window}")
    assert np.isnan(want[:, 4:]).any() and not np.isnan(want[:3 if counts is None else 92, :4]).any()


def test_attend_bad_queries(sm, dev):
    """A query that is not finite makes its own head's output NaN and no other."""
    import torch
    for counts in (None, [3, 20]):
        c = Case(sm, dev, 2, 64, 2, 3, 47)
        pos, qstart = [100, 70], None if counts is None else [0, 3, 23]
        c.fill(lengths(pos, qstart, None, 2))
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


@pytest.mark.parametrize("counts", [None, [1, 0, 5], [40, 3, 70]])
def test_attend_outliers(sm, dev, counts):
    """Query elements hundreds of times the others, keys and values of far apart
    magnitudes, a first position with nearly all the weight and next to no value."""
    import torch
    kvh, hd, heads = 2, 128, 8
    c = Case(sm, dev, kvh, hd, 3, 12, 91)
    pos, qstart = [600, 64, 300], None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    ntok = 3 if counts is None else int(qstart[-1])
    last = [p + (1 if counts is None else n) for p, n in zip(pos, counts or [1] * 3)]
    for s, n in enumerate(last):
        k = c.rng.standard_normal((n, kvh, hd))
        v = c.rng.standard_normal((n, kvh, hd)) * np.exp2(c.rng.integers(-12, 13, (n, kvh, 1)))
        k[0], v[0] = 4.0, v[0] * 1e-4
        kd, vd = (torch.from_numpy(x.astype(np.float32)).to(dev) for x in (k, v))
        c.kv.append(c.batch([0], n, [0, n], [s]), None, kd, vd)
        paged4.append(c.host, None, k.astype(np.float32).astype(float), v.astype(np.float32).astype(float), None, [0], [0, n], [s])
    c.same()
    for o in ("f32", "bf16"):
        q, qf = rows(dev, c.rng.standard_normal((ntok, heads, hd)) + 0.3, torch.float32)
        q[:, :, 5] *= 300.0
        q[:, ::2, 7] *= 1e-6
        qf = q.double().cpu().numpy()
        out = torch.full((ntok, heads, hd), 7.0, dtype=types()[o], device=dev)
        c.kv.attend(c.batch(pos, ntok, qstart, max_len=700), q, out)
        check_attention(c, q, qf, out, hd ** -0.5, 0, None, pos, qstart, None, note=f"outliers {o}")


@pytest.mark.parametrize("counts", [None, [3, 1, 2], [40, 3, 70]])
def test_attend_longer_than_said(sm, dev, counts):
    """max_len only shapes launches: sequences far past it, and far below, are served in full."""
    import torch
    c = Case(sm, dev, 2, 64, 3, 60, 73)
    pos = [3500, 1, 2000]
    qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    c.fill(lengths(pos, qstart, None, 3))
    ntok = 3 if counts is None else int(qstart[-1])
    q, qf = rows(dev, c.rng.standard_normal((ntok, 8, 64)), torch.float32)
    for max_len in (1, 0, 1 << 20):
        out = torch.full((ntok, 8, 64), 7.0, device=dev)
        c.kv.attend(c.batch(pos, ntok, qstart, max_len=max_len), q, out)
        check_attention(c, q, qf, out, 0.125, 0, None, pos, qstart, None, note=f"max_len {max_len}")


@pytest.mark.parametrize("max_q", [5, 512, 20000, 1 << 30, (1 << 31) - 1])
@pytest.mark.parametrize("counts,group", [([1], 4), ([2], 2), ([1, 2, 1], 1), ([0, 1], 4), ([5, 9], 4)])
def test_max_q_far_above_the_rows(sm, dev, counts, group, max_q):
    import torch
    kvh, hd, n = 2, 64, len(counts)
    c = Case(sm, dev, kvh, hd, n, 50, 97)
    qstart, pos = np.concatenate([[0], np.cumsum(counts)]), [3000, 40, 2900][:n]
    c.fill(lengths(pos, qstart, None, n))
    ntok = int(qstart[-1])
    q, qf = rows(dev, c.rng.standard_normal((ntok, kvh * group, hd)), torch.float32)
    k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.float32)
    b = c.batch(pos, ntok, qstart, max_q=max_q, max_len=3100)
    c.kv.append(b, None, k, k)
    paged4.append(c.host, None, kf, kf, None, pos, qstart, None, max_q)
    c.same()
    out = torch.full_like(q, 7.0)
    c.kv.attend(b, q, out)
    check_attention(c, q, qf, out, 0.125, 0, None, pos, qstart, None, max_q, f"{counts} group {group} max_q {max_q}")


def test_attend_many_sequences(sm, dev):
    """More sequences than a wave has lanes, idle ones among them, over shared
    pages: decode steps short and long, and ragged blocks."""
    c = Case(sm, dev, 2, 64, 6, 40, 79)
    c.fill([2560] * 6)
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
    c.fill(lengths(pos, qstart, None, nseq))
    for o in ("f32", "bf16"):
        attend(c, pos, qstart, None, 8, "f32", o, note=f"long {form} {o}")
    attend(c, pos, qstart, None, 8, window=3000, note=f"long {form}, window")


def test_attend_blocks_of_more_sequences_than_shares_hold(sm, dev):
    """2100 blocks of three tokens, whose tiles are too many to share out evenly: a
    workgroup a tile, one of them over more pages than it holds numbers of."""
    c = Case(sm, dev, 1, 64, 3, 270, 101)
    c.fill([70, 17000, 200])
    n = 2100
    slot, counts = np.zeros(n, int), np.full(n, 3)
    pos = c.rng.integers(0, 60, n)
    slot[[7, 2000]], pos[[7, 2000]] = 1, [16990, 9000]
    slot[5::9], pos[5::9] = 2, c.rng.integers(0, 190, len(pos[5::9]))
    counts[11::50] = 0
    attend(c, list(pos), np.concatenate([[0], np.cumsum(counts)]), list(slot), 16, "bf16", "f32", note="2100 blocks", max_len=17000)


@pytest.mark.parametrize("x,o", [("f32", "f32"), ("bf16", "bf16")])
def test_attend_short_blocks_of_many_sequences(sm, dev, x, o):
    """More sequences than a wave has lanes, each with up to three tiles of sixteen columns."""
    c = Case(sm, dev, 1, 128, 5, 20, 109)
    c.fill([1200] * 5)
    n = 90
    slot, counts, pos = c.rng.integers(0, 5, n), c.rng.integers(0, 13, n), c.rng.integers(0, 1100, n)
    qstart = np.concatenate([[0], np.cumsum(counts)])
    for window, most in ((0, 1200), (70, 1200), (0, 100)):
        attend(c, list(pos), qstart, list(slot), 4, x, o, window=window, max_q=12, max_len=most, note=f"window {window} {x}")


def test_attend_shares_of_many_pages(sm, dev):
    """A length said far too small makes few shares, of more pages than a workgroup holds numbers of."""
    c = Case(sm, dev, 1, 64, 2, 330, 103)
    pos, qstart = [20900, 300], [0, 100, 140]
    c.fill(lengths(pos, qstart, None, 2))
    for x in ("f32", "bf16"):
        attend(c, pos, qstart, None, 4, x, "f32", note=f"few shares {x}", max_len=1)
        attend(c, pos, qstart, None, 4, x, "f32", window=19000, note=f"few shares, window {x}", max_len=1)


@pytest.mark.parametrize("counts", [None, [3, 9], [20, 40]])
def test_pages_past_32_bits(sm, dev, counts):
    """Pages on both sides of 2^31 and 2^32 bytes give the bits that a small pool gives."""
    import torch
    kvh, hd, heads, n = 4, 256, 8, 2
    size = kvh * 68 * hd
    at = [(1 << 31) // size, (1 << 31) // size + 1, (1 << 32) // size, (1 << 32) // size + 3, (1 << 32) // size - 1, 2]
    npages = at[3] + 1
    pos = [100, 70]
    qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
    ntok = n if counts is None else int(qstart[-1])
    g = torch.Generator(device=dev).manual_seed(5)
    q, k = (torch.randn(ntok, h, hd, generator=g, device=dev) for h in (heads, kvh))
    data = torch.empty(npages, kvh, 68 * hd, dtype=torch.uint8, device=dev)
    small = sm.PagedKV4(kvh, hd, 6, n, 3, pages=torch.arange(6, dtype=torch.int32, device=dev).view(n, 3))
    large = sm.PagedKV4(kvh, hd, npages, n, 3, pages=torch.tensor(at, dtype=torch.int32, device=dev).view(n, 3), data=data)
    small.data.random_(0, 256, generator=g)
    for i, p in enumerate(at):
        data[p].copy_(small.data[i])
    got, old = [], torch.randn(sum(pos), kvh, hd, generator=g, device=dev)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for kv in (small, large):
        kv.append(sm.KVBatch(ints([0, 0]), sum(pos), ints([0, pos[0], sum(pos)]), max_q=max(pos), max_len=192), None, old, old)
        b = sm.KVBatch(torch.tensor(pos, dtype=torch.int32, device=dev), ntok,
                       None if qstart is None else torch.tensor(qstart, dtype=torch.int32, device=dev), max_q=64, max_len=192)
        out, rk, rv = torch.empty_like(q), *(torch.empty(n, 64, kvh, hd, device=dev) for _ in range(2))
        kv.append(b, None, k, k)
        kv.attend(b, q, out)
        kv.read(torch.tensor(pos, dtype=torch.int32, device=dev), rk, rv)
        assert torch.isfinite(out).all() and out.abs().max() > 0.1
        got.append([t.view(torch.int32) for t in (out, rk, rv)])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert all(torch.equal(data[p], small.data[i]) for i, p in enumerate(at))


def test_attend_two_at_once(sm, dev):
    """Two streams, each with a workspace of its own, the same bits as alone."""
    import torch
    c = Case(sm, dev, 2, 128, 4, 40, 107)
    c.fill([2500] * 4)
    calls = []
    for counts in (None, [30, 20, 9, 50]):
        qstart = None if counts is None else np.concatenate([[0], np.cumsum(counts)])
        n = 4 if counts is None else int(qstart[-1])
        q, _ = rows(dev, c.rng.standard_normal((n, 8, 128)), torch.float32)
        out, alone = torch.zeros_like(q), torch.zeros_like(q)
        b = c.batch([2000, 5, 2300, 700], n, qstart, max_len=2400)
        c.kv.attend(b, q, alone)
        calls.append((c.kv.attend_op(b, q, out), torch.cuda.Stream(device=dev), out, alone))
    torch.cuda.synchronize()
    for _ in range(5):
        for op, s, out, _ in calls:
            with torch.cuda.stream(s):
                out.zero_()
            op(s)
        torch.cuda.synchronize()
        assert all(torch.equal(out, alone) for _, _, out, alone in calls)


def test_rows_claimed_twice_stay_in_bounds(sm, dev):
    """Every sequence claims all rows, which the call does not serve as asked: it
    ends, and the rows next to the call's are left alone."""
    import torch
    kvh, hd, heads, n, ntok = 2, 64, 8, 200, 90
    c = Case(sm, dev, kvh, hd, 4, 6, 89)
    c.fill([384] * 4)
    qstart, slot = np.tile([0, ntok], n // 2 + 1)[:n + 1], np.arange(n) % 4
    q, _ = rows(dev, c.rng.standard_normal((ntok + 2, heads, hd)), torch.float32)
    out = torch.full_like(q, 7.0)
    b = sm.KVBatch(c.ints([100] * n), ntok, c.ints(qstart), c.ints(slot), max_len=200)
    c.kv.attend(b, q[1:-1], out[1:-1])
    torch.cuda.synchronize()
    assert torch.all(out[0] == 7.0) and torch.all(out[-1] == 7.0)


def test_strides_streams_and_repeats(sm, dev):
    """Rows wider than their heads, a stream of the caller's, the same bits each time."""
    import torch
    c = Case(sm, dev, 2, 64, 5, 8, 59)
    pos, heads, ntok = [400, 3, 64, 200, 90], 8, 5
    c.fill(lengths(pos, None, None, 5))
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


@pytest.mark.parametrize("form", ["decode", "block", "chunk"])
def test_capture_and_replay(sm, dev, form):
    """Append, attention and reading back recorded once and replayed as positions
    move, with eager calls on another cache between the replays."""
    import torch
    kvh, heads, hd, nseq = 2, 8, 128, 3
    c, e = (Case(sm, dev, kvh, hd, nseq, 8, 61) for _ in range(2))
    per = {"decode": 1, "block": 5, "chunk": 22}[form]
    ntok = nseq * per
    qstart = None if form == "decode" else [0, per, 2 * per, 3 * per]
    k, v = torch.zeros(ntok, kvh, hd, device=dev), torch.zeros(ntok, kvh, hd, device=dev)
    q = torch.zeros(ntok, heads, hd, device=dev)
    pos, start = c.ints([0, 0, 0]), c.ints([0, 0, 0])
    table, w = sm.rope_table(8 * 64, hd, 1e4, dev), torch.ones(hd, device=dev)
    b = sm.KVBatch(pos, ntok, c.ints(qstart), max_q=per, max_len=512)
    sides = []
    for kv in (c.kv, e.kv):
        turned, out = torch.zeros_like(q), torch.zeros_like(q)
        back = torch.zeros(2, nseq, 30, kvh, hd, device=dev)
        sides.append(([kv.append_op(b, q, k, v, table, turned, q_norm=w, k_norm=w), kv.attend_op(b, turned, out),
                       kv.read_op(start, back[0], back[1])], out, back, kv))
    stream = torch.cuda.Stream(device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for op in sides[0][0]:
            op()
    at = np.array([0, 50, 120])
    for step in range(14):
        pos.copy_(torch.from_numpy(at.astype(np.int32)))
        start.copy_(torch.from_numpy(np.maximum(at - 8, 0).astype(np.int32)))
        for t in (q, k, v):
            t.copy_(torch.from_numpy(c.rng.standard_normal(t.shape).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        for op in sides[1][0]:
            op()
        torch.cuda.synchronize()
        # positions that were never appended are random bytes, NaN among them
        same = lambda x, y: np.array_equal(x.cpu().numpy(), y.cpu().numpy(), equal_nan=True)  # noqa: E731
        assert same(sides[0][1], sides[1][1]), step
        assert same(sides[0][2], sides[1][2]) and torch.equal(c.kv.data, e.kv.data), step
        at = at + per
        if step == 10:
            at[1] -= 7      # a cut back sequence


def test_one_conversation(sm, dev):
    """A prompt in chunks, then tokens and verified blocks, two sequences at once, with
    norms and interleaved pairs: each cached value is off by at most one scale, the
    scale at most 2 / 7 of the block's largest element."""
    import torch
    kvh, heads, hd = 2, 8, 128
    c = Case(sm, dev, kvh, hd, 2, 8, 67)
    table = sm.rope_table(8 * 64, hd, 1e4, dev, scaling=sm.RopeScaling("yarn", 4, 128))
    tab = table.cpu().numpy()
    nw, nwf = rows(dev, 1 + 0.2 * c.rng.standard_normal(hd), torch.float32)
    eps = float(np.float32(1e-6))
    lens = [0, 0]
    for counts in ([130, 40], [1, 1], [1, 0], [5, 8], [1, 1], [64, 3], [1, 1]):
        ntok = sum(counts)
        qstart = np.concatenate([[0], np.cumsum(counts)])
        q, qf = rows(dev, c.rng.standard_normal((ntok, heads, hd)), torch.float32)
        k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.float32)
        v, vf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.float32)
        out = torch.full((ntok, heads, hd), 7.0, device=dev)
        b = c.batch(lens, ntok, qstart)
        c.kv.append(b, q, k, v, table, q, interleaved=True, q_norm=nw, k_norm=nw, eps=eps)
        c.kv.attend(b, q, out)
        paged4.append(c.host, qf, kf, vf, tab, lens, qstart, interleaved=True, q_norm=nwf, k_norm=nwf, eps=eps)
        c.same()
        check_attention(c, q, q.double().cpu().numpy(), out, hd ** -0.5, 0, None, lens, qstart, None, note=str(counts))
        for s in range(2):
            for j in range(counts[s]):
                r = qstart[s] + j
                kc, vc = paged4.read(c.host, s, lens[s] + j, hd)
                for x, y in ((kc, paged4.turn(kf[r], tab[lens[s] + j], True, nwf, eps)), (vc, vf[r])):
                    most = np.abs(y).reshape(kvh, -1, 32).max(-1)
                    assert np.all(np.abs(x - y).reshape(kvh, -1, 32).max(-1) <= 2 / 7 * most * (1 + 1e-6))
            lens[s] += counts[s]


def test_binding_refusals(sm, dev):
    import torch
    c = Case(sm, dev, 2, 64, 2, 2, 71)
    x = torch.zeros(2, 2, 64, device=dev)
    q = torch.zeros(2, 4, 64, device=dev)
    w = torch.ones(64, device=dev)
    b = c.batch([0, 0])
    for call, text in (
            (lambda: c.kv.append(b, None, x.half(), x), "type"), (lambda: c.kv.append(b, None, x, x[:1]), "1 rows"),
            (lambda: c.kv.append(b, q, x, x), "do not agree"), (lambda: c.kv.append(b, None, x[:, :1], x), "shape"),
            (lambda: c.kv.append(b, None, x.cpu(), x), "on cpu"), (lambda: c.kv.attend(b, q[:, :3], q), "shape"),
            (lambda: c.kv.append(b, None, x, x, k_norm=w[:63]), "shape"), (lambda: c.kv.append(b, None, x, x, k_norm=w.half()), "type"),
            (lambda: c.kv.append(b, None, x, x, k_norm=w, eps=0.0), "eps"),
            (lambda: c.kv.append(b, q, x, x, q_out=q, q_norm=w.cpu()), "on cpu"),
            (lambda: c.kv.attend(b, q[:, :3].contiguous(), q[:, :3].contiguous()), "query heads"),
            (lambda: c.kv.attend(b, q, q.transpose(1, 2).contiguous().transpose(1, 2)), "side by side"),
            (lambda: c.kv.read(c.ints([0, 0])), "nothing"),
            (lambda: sm.PagedKV4(2, 64, 9, 2, 2, pages=c.kv.pages, data=c.kv.data), "shape"),
            (lambda: sm.PagedKV4(2, 64, 7, 2, 2, pages=c.kv.pages, data=c.kv.data.char()), "type"),
            (lambda: c.kv.append(b, None, x, x, torch.zeros(127, 64, device=dev)), "does not cover")):
        with pytest.raises(sm.SparkmvError, match=text):
            call()
