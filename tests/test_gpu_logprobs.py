"""GPU tests of sparkmv_logprobs against the definitions in 64 bits
(oracle/paged.py).

Bounds, with u = 2^-24 and the largest |x - max| = D where e^(x - max) counts:
a term e^(x - max) is off by a relative 4 u (1 + |x - max|) at most, terms
below e^-30 add up to less than u, so the sum by 4 * 31 u plus the additions'
depth (64 u for partial sums of a few thousand, then their sums), and a log
probability by that, the logarithm's own 4 u of its value and 2 u of x and max."""
import numpy as np
import pytest

import paged

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def make(dev, rows, n, seed, x="f32", scale=3.0, ld=0):
    import torch
    rng = np.random.default_rng(seed)
    v = (rng.standard_normal((rows, n)) * scale).astype(np.float32)
    t = torch.full((rows, max(ld, n)), 1e9, device=dev).to(torch.float32 if x == "f32" else torch.bfloat16)[:, :n]
    t.copy_(torch.from_numpy(v))
    return rng, t, t.double().cpu().numpy()


def check(sm, t, f, tokens, k):
    import torch
    rows, n = f.shape
    lp, ent, ids, tops = sm.logprobs(t, None if tokens is None else torch.tensor(tokens, dtype=torch.int32, device=t.device), k)
    w_lp, w_ent, w_ids, w_tops = paged.logprobs(f, tokens, k)
    assert np.array_equal(ids.cpu().numpy(), w_ids)
    big = np.abs(np.where(np.isfinite(f), f, 0)).max(1)
    for what, got, want in (("logprob", lp, w_lp), ("entropy", ent, w_ent), ("tops", tops, w_tops)):
        if got is None:
            continue
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want)), what
        inf = np.isinf(want)
        assert np.array_equal(got[inf], want[inf]), what
        ok = np.isfinite(want)
        room = (4 * 31 + 64 + 64) * U + 4 * U * (big if want.ndim == 1 else big[:, None]) + 4 * U * np.abs(np.where(ok, want, 0))
        if what == "entropy":   # its sum weighs each term by |x - max| <= 31
            room = room * 32
        err = np.abs(np.where(ok, got - np.where(ok, want, 0), 0))
        assert np.all(err <= room), (what, float((err / room).max()))
        print(f"{rows} x {n}, {what}: largest error {err.max() if err.size else 0:.2e}")


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(1, 131072, 8), (1, 1, 1), (3, 2, 5), (2, 63, 32), (7, 1000, 20), (1, 151936, 32), (5, 4097, 1),
                                      (64, 16384, 3), (2, 8192, 0), (300, 77, 4)])
def test_rows(sm, dev, rows, n, k, x):
    rng, t, f = make(dev, rows, n, rows * 7 + n, x)
    check(sm, t, f, rng.integers(0, n, rows), k)


def test_strides(sm, dev):
    """Rows that do not start on 16 bytes, and a last row that ends the buffer."""
    for x in ("f32", "bf16"):
        for n, ld in ((1001, 1003), (513, 600), (8191, 8191)):
            rng, t, f = make(dev, 5, n, n + ld, x, ld=ld)
            check(sm, t, f, rng.integers(0, n, 5), 9)
            check(sm, t[1:], f[1:], rng.integers(0, n, 4), 9)


def test_ties_go_to_the_lower_index(sm, dev):
    import torch
    rng = np.random.default_rng(5)
    v = rng.integers(-3, 4, (4, 20000)).astype(np.float32)
    v[1] = 2.0
    v[2] = np.where(rng.random(20000) < 0.5, 0.0, -0.0)
    v[3] = np.repeat(np.arange(200), 100)[::-1]
    check(sm, torch.from_numpy(v).to(dev), v.astype(np.float64), [0, 5, 19999, 3], 32)


def test_masked_rows(sm, dev):
    """-inf in most places, in all but fewer than k, in all; the type's lowest value."""
    for n in (70, 30000):
        rng, t, f = make(dev, 6, n, 9 + n)
        t[0, rng.random(n) < 0.9] = -np.inf
        t[1, :] = -np.inf
        t[1, n // 2], t[1, n - 1] = -5.0, 2.0
        t[2, :] = -np.inf
        t[3, :] = float(np.finfo(np.float32).min)
        t[4, ::2] = float(np.finfo(np.float32).min)
        t[5, :] = -np.inf
        t[5, 3] = 3.0e38
        check(sm, t, t.double().cpu().numpy(), [1, 0, 4, 2, 1, 3], 12)


def test_unusual_values(sm, dev):
    """NaN and +inf make a row NaN (and no other); large and equal logits."""
    for n in (100, 20000):
        rng, t, f = make(dev, 6, n, 13 + n)
        t[0, n // 3] = np.nan
        t[1, n // 3] = np.inf
        t[2, :] = np.nan
        t[3, :] = 3.0e38
        t[4, :] *= 1e30
        check(sm, t, t.double().cpu().numpy(), rng.integers(0, n, 6), 5)


def test_tokens_outside_the_row(sm, dev):
    rng, t, f = make(dev, 4, 500, 17)
    check(sm, t, f, [-1, 500, 2 ** 31 - 1, 499], 2)
    check(sm, t, f, None, 2)


def test_capture_and_stream(sm, dev):
    import torch
    rng, t, f = make(dev, 8, 20000, 19)
    rows, k = 8, 6
    tok = torch.tensor(rng.integers(0, 20000, rows), dtype=torch.int32, device=dev)
    outs = [torch.empty(rows, device=dev), torch.empty(rows, device=dev), torch.empty(rows, k, dtype=torch.int32, device=dev),
            torch.empty(rows, k, device=dev)]
    op = sm.logprobs_op(t, tok, *outs)
    s = torch.cuda.Stream(device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        op()
    for step in range(4):
        t.copy_(torch.from_numpy((rng.standard_normal((rows, 20000)) * 3).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = sm.logprobs(t, tok, k)
        for a, b in zip(outs, want):
            assert torch.equal(a, b), step


def test_argmax_is_the_first_alternative(sm, dev):
    rng, t, f = make(dev, 3, 151936, 23)
    ids = sm.logprobs(t, None, 1)[2]
    for r in range(3):
        assert int(sm.argmax(t[r].contiguous())[0]) == int(ids[r, 0])
