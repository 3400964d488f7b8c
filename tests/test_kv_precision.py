"""CPU tests of the bound that tests/test_gpu_kv_precision.py holds attention
over the paged cache to (oracle/paged.py attend_bound): queries and weights as
integers of the kernels' widths stay within it, narrower ones do not.

Two scenes where widths matter. "outlier": one query element is 300 times the
others, in a channel where the keys are zero, so the scores are the others'.
"sink": the first position has nearly all the weight and next to no value; what
the output is made of has weights of e^-12."""
import numpy as np
import pytest

import paged

POS, QSTART = [50, 150, 61], [0, 8, 9, 12]


def scene(kind, kvh, group, hd, seed, qstart=QSTART):
    """(cache, q [tokens, heads, hd]) of three sequences."""
    rng = np.random.default_rng(seed)
    npages = 10
    c = {"pages": rng.permutation(npages)[:9].reshape(3, 3).astype(np.int32)}
    for n in "kv":
        c[n] = np.clip(np.rint(rng.standard_normal((npages, kvh, 64 * hd)) * 30), -127, 127).astype(np.int8)
        c[n + "_scale"] = ((0.5 + rng.random((npages, kvh))) / 30).astype(np.float32)
    off = paged.offsets(hd)
    q = rng.standard_normal((qstart[-1], kvh * group, hd)) * 1.5
    if kind == "outlier":
        c["k"][:, :, off[0][:, 3]] = 0
        q[:, :, 3] = 450 * np.sign(q[:, :, 3])
    else:
        q *= 0.1
        c["k"][:, :, off[0][:, 3]] = 0
        c["v"] = (np.abs(c["v"]) // 2 + 60).astype(np.int8)
        for s, (a, b) in enumerate(zip(qstart, qstart[1:])):
            page = c["pages"][s, 0]
            c["k"][page, :, off[0][0, 3]] = 120
            c["v"][page][:, off[1][0]] = 1
            for h in range(kvh):
                q[a:b, h * group:(h + 1) * group, 3] = 12 / (120 * float(c["k_scale"][page, h]) * hd ** -0.5)
    return c, q


SHAPES = [(2, 4, 256), (1, 16, 64), (2, 5, 128)]


def worst(kind, shape, bf16, *widths):
    """The largest share of the bound that integers of these widths take, with a
    bf16 output's own rounding."""
    kvh, group, hd = shape
    c, q = scene(kind, kvh, group, hd, hd)
    most = 0.0
    for row, h, k, v in paged.seen_rows(c, hd, 0, POS, QSTART, ntok=12):
        for g in range(h * group, (h + 1) * group):
            x = q[row, g].astype(np.float32).astype(np.float64)
            want = paged.attend_one(x, k, v, hd ** -0.5)[0]
            got = paged.attend_digits(x, k, v, hd ** -0.5, *widths)
            if bf16:
                step = np.exp2(np.floor(np.log2(np.abs(got))) - 7)
                got = np.rint(got / step) * step
            most = max(most, (np.abs(got - want) / paged.attend_bound(x, k, v, hd ** -0.5, bf16)).max())
    return most


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["outlier", "sink"])
def test_kernel_widths_are_within_the_bound(kind, shape):
    assert worst(kind, shape, False, 30, 30, False) < 1
    assert worst(kind, shape, True, 22, 22.9, True) < 1


@pytest.mark.parametrize("shape", SHAPES)
def test_narrower_queries_are_seen(shape):
    assert worst("outlier", shape, False, 14, 30, False) > 1
    assert worst("outlier", shape, True, 14, 22.9, True) > 1


@pytest.mark.parametrize("shape", SHAPES)
def test_narrower_weights_are_seen(shape):
    assert worst("sink", shape, False, 30, 15, False) > 1
    assert worst("sink", shape, True, 22, 15, False) > 1


@pytest.mark.parametrize("refills", [1, 5, 20, 60])
def test_a_page_cut_back_and_filled_again(refills):
    """Drafted tokens that end a page, rejected and drafted again with slightly
    larger values each time: the older values are rounded anew each time. After
    the first filling a value is off by 3 steps at most (tests/test_kv.py); each
    refill adds half a step and no step is smaller than those before it. The bound
    of a page that is filled once does not hold here."""
    rng = np.random.default_rng(5)
    hd = 64
    c = {"k": np.zeros((1, 1, 64 * hd), np.int8), "v": np.zeros((1, 1, 64 * hd), np.int8),
         "k_scale": np.zeros((1, 1), np.float32), "v_scale": np.zeros((1, 1), np.float32), "pages": np.zeros((1, 1), np.int32)}
    x = rng.standard_normal((64, 1, hd)).astype(np.float32).astype(np.float64)
    for p in range(60):
        paged.append(c, None, x[p:p + 1], x[p:p + 1], None, [p])
    most = 0.0
    for n in range(refills + 1):
        new = rng.uniform(-1, 1, (4, 1, hd)) * 6.0 * 1.01 ** n
        new[0, 0, 0] = 6.0 * 1.01 ** n
        new = new.astype(np.float32).astype(np.float64)
        before = c["k_scale"][0, 0]
        paged.append(c, None, new, new, None, [60], [0, 4])
        assert c["k_scale"][0, 0] > before
        x[60:] = new
        for p in range(64):
            k, v = paged.read(c, 0, p, hd)
            err = np.abs(k - x[p]).max() / c["k_scale"][0, 0]
            assert err <= (3 + n / 2) * (1 + 1e-6)
            assert np.array_equal(k, v)
            most = max(most, err)
    if refills >= 20:
        assert most > 3
