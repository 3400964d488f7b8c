"""GPU tests of the 4-bit cache's attention where a score is exact in f32, so that
what queries lose on their way shows, and of queries and keys of far apart magnitudes.

Queries here are small multiples of a power of two, of at most eight significant bits,
and keys are codes under one power of two, such that every partial sum of a score is
a multiple of one power of two g below 2^24 g: exact in f32, in any order. u = 2^-24
(half a step of f32). The score's factor and its product with it are rounded (2 u s of
the exponent), and so is the difference to the reference (2 u of the largest score):
with s the largest score a weight is off by 4 u s of itself, by twice that relative to
the sum of the weights, the sums of n positions by (n / 2 + 160) u as in test_gpu_kv4.py:
  |out - exact| <= W (8 s + 160 + n / 2) u, W the weighted sum of |v|;
bf16 outputs hold a weight to 2^-17 of itself (W 2^-17 more) and are rounded once."""
import numpy as np
import pytest

import paged4
from test_gpu_kv import rows, types
from test_gpu_kv4 import U, Case, attend, lengths

pytestmark = pytest.mark.gpu

# up to 48 columns of a kv head and sequence, and more
MAX_Q = {"decode": 1, "block": 7, "chunk": 60}
FORMS = {"decode": ([200, 3, 129], None), "block": ([200, 3, 129], [0, 5, 6, 13]), "chunk": ([140, 3, 70], [0, 60, 65, 95])}


def put_keys(c, length, byte):
    """Key scale bytes of positions 0 .. length[slot] - 1: byte(block) for each block of 32."""
    off = paged4.offsets(c.hd)
    for s, n in enumerate(length):
        for p in range(n):
            page = c.host["data"][c.host["pages"][s, p // 64]]
            for blk in range(c.hd // 32):
                page[:, off[1, p % 64, 32 * blk]] = byte(blk)


def check_exact(c, q, out, scale, pos, qstart):
    qf = q.double().cpu().numpy()
    want, size = paged4.attend(c.host, qf, c.hd, scale, 0, None, pos, qstart)
    got = out.double().cpu().numpy()
    assert np.isfinite(want).all() and np.isfinite(got).all()
    s, w, n = largest_score(c, qf, scale, pos, qstart), size[..., 1], max(pos) + len(qf)
    assert 1.0 < s < 100.0      # scores matter
    bound = w * (8 * s + 160 + n / 2) * U
    if str(out.dtype).endswith("bfloat16"):
        bound = bound + w * 2.0 ** -17 + 2.0 ** -8 * np.abs(want).max(-1)
    err = np.abs(got - want)
    print(f"relL2 {np.linalg.norm(err) / np.linalg.norm(want):.2e}, of the bound {(err / bound[..., None]).max():.2f}")
    assert np.all(err <= bound[..., None])


def largest_score(c, qf, scale, pos, qstart):
    """Of any row and position that it sees."""
    group, most = qf.shape[1] // c.kvh, 0.0
    for i, p0 in enumerate(pos):
        r = range(i, i + 1) if qstart is None else range(qstart[i], qstart[i + 1])
        n = p0 + len(r)
        page = c.host["pages"][i, :(n + 63) // 64].astype(int)
        k = paged4.values(c.host, page, c.hd)[0].transpose(1, 0, 2, 3).reshape(c.kvh, -1, c.hd)[:, :n]
        for t in r:
            for g in range(qf.shape[1]):
                most = max(most, np.abs(k[g // group] @ qf[t, g]).max() * abs(scale))
    return most


@pytest.mark.parametrize("x,o", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", list(FORMS))
def test_queries_enter_whole(sm, dev, form, hd, x, o):
    """Large elements beside small ones, each of which moves the scores: half the
    elements are 128 .. 255, the others 1 / 8 .. 15 / 8, down to 2^-11 of the largest. Sums
    are multiples of 1 / 16 below 256 * 255 * 6 < 2^19."""
    import torch
    pos, qstart = FORMS[form]
    c = Case(sm, dev, 2, hd, 3, 5, 201 + hd)
    length = lengths(pos, qstart, None, 3)
    c.fill(length)
    put_keys(c, length, lambda blk: 127)
    c.put()
    ntok = 3 if qstart is None else qstart[-1]
    shape = (ntok, 8, hd)
    big = c.rng.integers(128, 256, shape) * np.where(c.rng.random(shape) < 0.5, -1, 1)
    small = c.rng.integers(-15, 16, shape) / 8.0
    q, qf = rows(dev, np.where(c.rng.random(shape) < 0.5, big, small), types()[x])
    out = torch.full(shape, 7.0, dtype=types()[o], device=dev)
    scale = 2.0 ** (-10 if hd == 64 else -11)
    c.kv.attend(c.batch(pos, ntok, qstart, max_q=MAX_Q[form], max_len=300), q, out, scale)
    check_exact(c, q, out, scale, pos, qstart)


def apart(sm, dev, form, hd, x, q_exp, key_byte, scale, keep=None, seed=0):
    """Queries of +-1 .. 15 times 2^q_exp(block) and keys with scale byte key_byte(block)."""
    import torch
    pos, qstart = FORMS[form]
    c = Case(sm, dev, 2, hd, 3, 5, 301 + hd + seed)
    length = lengths(pos, qstart, None, 3)
    c.fill(length)
    put_keys(c, length, key_byte)
    if keep:
        off = paged4.offsets(hd)
        for blk in range(hd // 32):
            if not keep(blk):
                c.host["data"][:, :, off[0, :, 32 * blk:32 * blk + 32].ravel()] = 0
    c.put()
    ntok = 3 if qstart is None else qstart[-1]
    shape = (ntok, 8, hd)
    f = np.array([2.0 ** q_exp(d // 32) for d in range(hd)])
    q, _ = rows(dev, c.rng.integers(1, 16, shape) * np.where(c.rng.random(shape) < 0.5, -1, 1) * f, types()[x])
    out = torch.full(shape, 7.0, device=dev)
    c.kv.attend(c.batch(pos, ntok, qstart, max_q=MAX_Q[form], max_len=300), q, out, scale)
    check_exact(c, q, out, scale, pos, qstart)


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("q_exp,key_byte,scale_exp", [(-90, 252, -44), (-122, 252, -11), (100, 20, -1), (118, 7, -6), (-20, 127, 12)])
def test_queries_and_keys_of_any_magnitude(sm, dev, q_exp, key_byte, scale_exp, form, hd, x):
    """Down to 2^-122 and up to 2^122, under keys that bring the scores near 1: they
    are multiples of one power of two up to 256 * 15 * 12 of them."""
    apart(sm, dev, form, hd, x, lambda blk: q_exp, lambda blk: key_byte, 2.0 ** scale_exp)


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("span", [30, 89, 100, 108])
def test_blocks_of_queries_far_apart(sm, dev, span, form, hd, x):
    """32 elements 2^span times the others, under keys that are zero: the others make the scores."""
    apart(sm, dev, form, hd, x, lambda blk: span - 40 if blk == 0 else -40, lambda blk: 127 + 42, 2.0 ** -8, lambda blk: blk > 0, span)


@pytest.mark.parametrize("o", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("form", list(FORMS))
def test_bad_queries_without_pages(sm, dev, form, hd, o):
    """A token none of whose positions has a page is zeros, whatever its query holds."""
    import torch
    pos, qstart = FORMS[form]
    c = Case(sm, dev, 2, hd, 3, 5, 401)
    c.fill(lengths(pos, qstart, None, 3))
    c.host["pages"][1, :] = -1
    c.put()
    ntok = 3 if qstart is None else qstart[-1]
    at = slice(1, 2) if qstart is None else slice(qstart[1], qstart[2])
    q = torch.randn(ntok, 8, hd, device=dev)
    q[at, 1, 3], q[at, 2, 40], q[at, 7, 60] = float("nan"), float("inf"), -float("inf")
    out = torch.full(q.shape, 7.0, dtype=types()[o], device=dev)
    c.kv.attend(c.batch(pos, ntok, qstart, max_q=MAX_Q[form], max_len=300), q, out)
    assert torch.all(out[at] == 0.0) and torch.isfinite(out).all() and torch.all(out[0].abs().amax(-1) > 0)


@pytest.mark.parametrize("kvh,group,hd", [(2, 4, 256), (1, 1, 64), (2, 2, 128), (1, 3, 256), (1, 16, 64), (2, 5, 128), (1, 16, 256)])
@pytest.mark.parametrize("counts", [[8, 1, 3], [70, 33, 1], [150, 0, 64]])
def test_bf16_queries_with_f32_outputs(sm, dev, kvh, group, hd, counts):
    c = Case(sm, dev, kvh, hd, 3, 6, 501 + hd)
    qstart = np.concatenate([[1], 1 + np.cumsum(counts)])
    pos = [0, 190, 130]
    c.fill(lengths(pos, qstart, None, 3))
    attend(c, pos, qstart, None, kvh * group, "bf16", "f32", note=f"{counts} kvh {kvh} group {group} hd {hd}")


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", list(FORMS))
def test_outliers_under_keys_of_zero(sm, dev, form, hd, x):
    """One element 300 times the others, under keys that are zero, so that the others
    make the scores. Past 48 columns an element that needs more bits is off by 2^-24 of
    the largest of its 32 neighbours, a score by the sum of that times its keys, and a
    weight by twice that relative to the sum; the rest of the bound is
    test_gpu_kv4.py's."""
    import torch
    pos, qstart = FORMS[form]
    c = Case(sm, dev, 2, hd, 3, 5, 601 + hd)
    c.fill(lengths(pos, qstart, None, 3))
    off = paged4.offsets(hd)
    c.host["data"][:, :, off[0, :, 4:6].ravel()] = 0     # two elements of a byte
    c.put()
    ntok = 3 if qstart is None else qstart[-1]
    x0 = c.rng.standard_normal((ntok, 8, hd)) + 0.3
    x0[:, :, 5] *= 300.0
    x0[:, ::2, 7] *= 1e-3
    q, qf = rows(dev, x0, types()[x])
    out = torch.full(q.shape, 7.0, device=dev)
    scale = hd ** -0.5
    c.kv.attend(c.batch(pos, ntok, qstart, max_q=MAX_Q[form], max_len=300), q, out, scale)
    want, size = paged4.attend(c.host, qf, hd, scale, 0, None, pos, qstart)
    off_by = np.zeros(qf.shape)
    if form == "chunk":
        most = np.repeat(np.abs(qf).reshape(ntok, 8, -1, 32).max(-1), 32, -1)
        off_by = np.where((x == "bf16") & (np.abs(qf) >= 2.0 ** -17 * most), 0.0, 2.0 ** -24 * most)
    _, lost = paged4.attend(c.host, off_by, hd, scale, 0, None, pos, qstart)
    s, w, n = size[..., 0], size[..., 1], max(pos) + ntok
    bound = w * ((2 * (hd + 8) * s + 160 + n / 2) * U + 2 * lost[..., 0])
    err = np.abs(out.double().cpu().numpy() - want)
    print(f"relL2 {np.linalg.norm(err) / np.linalg.norm(want):.2e}, of the bound {(err / bound[..., None]).max():.2f}")
    assert np.all(err <= bound[..., None])
