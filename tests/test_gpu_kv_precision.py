"""GPU tests of what attention over the paged cache holds its queries and
weights to: the scenes and the bound of tests/test_kv_precision.py, which shows
on the CPU that narrower integers do not pass."""
import numpy as np
import pytest

import paged
from test_kv_precision import scene

pytestmark = pytest.mark.gpu

FORMS = {   # (pos, qstart); None: one token each
    "decode": ([50, 150, 61], None),
    "block": ([50, 150, 61], [0, 8, 9, 12]),
    "chunk": ([2, 0, 61], [0, 130, 177, 300]),
}


def run(sm, dev, c, q, hd, pos, qstart, x, o, scale=None):
    """(outputs, the queries' values) of one call."""
    import torch
    ints = lambda v: None if v is None else torch.tensor(np.asarray(v), dtype=torch.int32, device=dev)  # noqa: E731
    t = {n: torch.from_numpy(a.copy()).to(dev) for n, a in c.items()}
    kv = sm.PagedKV(c["k"].shape[1], hd, c["k"].shape[0], *c["pages"].shape, **t)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}
    qt = torch.from_numpy(q.astype(np.float32)).to(dev).to(dt[x])
    out = torch.full(q.shape, 7.0, dtype=dt[o], device=dev)
    kv.attend(sm.KVBatch(ints(pos), len(q), ints(qstart), max_len=192), qt, out, scale)
    return out.double().cpu().numpy(), qt.double().cpu().numpy()


@pytest.mark.parametrize("x,o", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("kvh,group,hd", [(2, 4, 256), (1, 16, 64), (2, 5, 128), (8, 4, 64), (8, 4, 256)])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("kind", ["outlier", "sink"])
def test_outliers_and_sinks(sm, dev, kind, form, kvh, group, hd, x, o):
    pos, qstart = FORMS[form]
    c, q = scene(kind, kvh, group, hd, hd + kvh, qstart or [0, 1, 2, 3])
    got, qf = run(sm, dev, c, q, hd, pos, qstart, x, o)
    most = 0.0
    for row, h, k, v in paged.seen_rows(c, hd, 0, pos, qstart, ntok=len(q)):
        for g in range(h * group, (h + 1) * group):
            want = paged.attend_one(qf[row, g], k, v, hd ** -0.5)[0]
            bound = paged.attend_bound(qf[row, g], k, v, hd ** -0.5, o == "bf16")
            most = max(most, (np.abs(got[row, g] - want) / np.maximum(bound, 1e-300)).max())   # 0 where every value is
    print(f"{kind} {form} kvh {kvh} group {group} hd {hd} {x} {o}: {most:.3f} of the bound")
    assert most <= 1


def check_one_position(sm, dev, form, kvh, group, hd, x, o, size):
    """Each query is a multiple of the key at one of its positions, with a score
    of `size` there: that position has all the weight, the others' scores being
    lower by a tenth of it at least, and the output is its value. Off by the
    weight's integer, 2^-23, the division and the gate, a few 2^-24, and a bf16
    output's half step."""
    pos, qstart = FORMS[form]
    c, q = scene("outlier", kvh, group, hd, 7 * hd + kvh, qstart or [0, 1, 2, 3])
    rng, want = np.random.default_rng(3), np.zeros(q.shape)
    for row, h, k, v in paged.seen_rows(c, hd, 0, pos, qstart, ntok=len(q)):
        for g in range(h * group, (h + 1) * group):
            at = rng.integers(len(k))
            unit = k[at] / (k[at] @ k[at] * hd ** -0.5)
            at = np.argmax(k @ unit)     # a longer key may score more
            q[row, g], want[row, g] = unit * size, v[at]
            s = np.sort(k @ unit)
            assert len(s) == 1 or s[-2] < s[-1] - 0.01
    got, _ = run(sm, dev, c, q, hd, pos, qstart, x, o)
    err = np.abs(got - want)
    assert np.all(err <= np.abs(want) * (8 * 2.0 ** -24 + 2.0 ** -22 + (2.0 ** -8 if o == "bf16" else 0.0))), float(err.max())


SHAPES = [(2, 4, 256), (1, 16, 64), (8, 4, 128)]


@pytest.mark.parametrize("size", [3.0e5, 3.0e8])
@pytest.mark.parametrize("x,o", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("kvh,group,hd", SHAPES)
@pytest.mark.parametrize("form", list(FORMS))
def test_very_large_scores(sm, dev, form, kvh, group, hd, x, o, size):
    check_one_position(sm, dev, form, kvh, group, hd, x, o, size)


@pytest.mark.parametrize("size", [1.0e10, 3.0e12, 1.0e25])
@pytest.mark.parametrize("x,o", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("kvh,group,hd", SHAPES)
@pytest.mark.parametrize("form", list(FORMS))
def test_scores_whose_last_place_is_more_than_an_exponent(sm, dev, form, kvh, group, hd, x, o, size):
    check_one_position(sm, dev, form, kvh, group, hd, x, o, size)
