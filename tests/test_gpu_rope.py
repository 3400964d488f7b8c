"""GPU tests of scaled rotary tables and of head norms with the rotation, against
their definitions in 64 bits (oracle/paged4.py). Tables and f32 outputs are computed
in 64 bits and rounded once: half a step of the output's type, and 1e-6 of that for
what the 64-bit sums and roots may be off (where a sum cancels, 2^-49 of its terms).
bf16 outputs are computed in f32, in roundings of 2^-24: 9 at most in the sum of 256
squares, which the root halves, 2 in the root and its conversion, 4 in a term (its
factor, its product, the sum, the norm's product): 10.5 of the two terms' magnitudes,
which are sqrt 2 of the largest normed element of the head together, less than 2^-20 of
it beside the half step."""
import numpy as np
import pytest

import paged4
from test_gpu_kv import rows, types

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,d,theta", [(1, 2, 1e4), (4096, 64, 5e6), (513, 256, 1e4), (131072, 32, 5e5), (70, 6, 100.0), (65, 90, 1e4)])
@pytest.mark.parametrize("scaling", [
    None, {}, {"kind": "linear", "factor": 4}, {"kind": "ntk", "factor": 8}, {"kind": "yarn", "factor": 32, "original": 4096},
    {"kind": "yarn", "factor": 2, "original": 1024, "beta_fast": 8, "beta_slow": 2, "attention": 1.0},
    {"kind": "bands", "factor": 8, "original": 8192}, {"kind": "bands", "factor": 3, "original": 600, "low": 0.5, "high": 20, "attention": 0.7}])
def test_table(sm, dev, n, d, theta, scaling):
    import torch
    s = None if scaling is None else sm.RopeScaling(**scaling)
    got = torch.full((n + 1, d), 7.0, device=dev)
    sm.rope_table_op(got[:n], theta, s)()
    assert torch.all(got[n] == 7.0)
    want = paged4.table(n, d, theta, **(scaling or {}))
    # an angle of up to 131072 is off by 2^-36 in 64 bits, and so is a table entry
    assert np.all(np.abs(got[:n].double().cpu().numpy() - want) <= 2.0 ** -24 * np.abs(want) * (1 + 1e-6) + 2.0 ** -35)
    if s is not None:
        assert torch.equal(sm.rope_table(n, d, theta, dev, scaling=s), got[:n])


CASES = [(2, 1, 256, 64, 1), (16, 4, 256, 256, 5), (3, 5, 64, 64, 9), (1, 1, 4, 4, 3), (7, 2, 80, 80, 12), (4, 4, 96, 34, 6),
         (5, 1, 192, 6, 7), (2, 2, 128, 0, 4), (9, 3, 12, 2, 65), (32, 8, 128, 128, 700), (3, 3, 36, 30, 2000), (1, 2, 256, 90, 1300)]


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("heads,kvh,hd,rope,n", CASES)
def test_qk_rope(sm, dev, heads, kvh, hd, rope, n, inter, x):
    """Into other tensors and in place, with and without norms, q or k alone."""
    import torch
    rng = np.random.default_rng(heads + hd + rope)
    dt = types()[x]
    wide = 8 * ((hd * (heads + kvh) + 15) // 8)
    both, bf = rows(dev, rng.standard_normal((n, wide)) * np.exp(rng.standard_normal((n, 1))), dt)
    # a head's rows start 16-byte aligned: keys at the next multiple of eight elements
    kat = 8 * ((heads * hd + 7) // 8)
    q, k = both[:, :heads * hd].unflatten(1, (heads, hd)), both[:, kat:kat + kvh * hd].unflatten(1, (kvh, hd))
    qf, kf = bf[:, :heads * hd].reshape(n, heads, hd), bf[:, kat:kat + kvh * hd].reshape(n, kvh, hd)
    table = sm.rope_table(500, rope, 1e4, dev) if rope else None
    tab = table.cpu().numpy() if rope else None
    at = rng.integers(0, 500, n)
    pos = torch.tensor(at, dtype=torch.int32, device=dev) if rope else None
    eps = float(np.float32(1e-3))
    half = 2.0 ** -24 if x == "f32" else 2.0 ** -8
    for qn, kn in ((False, False), (True, True), (False, True)):
        w = [rows(dev, 1 + 0.3 * rng.standard_normal(hd), torch.float32) if on else (None, None) for on in (qn, kn)]
        want = [np.stack([paged4.turn(f[t], tab[at[t]] if rope else None, inter, wf, eps) for t in range(n)])
                for f, (_, wf) in zip((qf, kf), w)]
        size = [np.stack([np.abs(paged4.turn(f[t], None, inter, wf, eps)).max(-1, keepdims=True) for t in range(n)])
                for f, (_, wf) in zip((qf, kf), w)]

        def check(got, exact, most):
            got = got.double().cpu().numpy()
            assert np.all(np.abs(got - exact) <= half * np.abs(exact) * (1 + 1e-6) + (2.0 ** -49 if x == "f32" else 2.0 ** -20) * most)

        def room(h):    # rows that start 16-byte aligned
            return torch.full((n, 8 * ((h * hd + 7) // 8)), 7.0, dtype=dt, device=dev)[:, :h * hd].unflatten(1, (h, hd))

        qo, ko = room(heads), room(kvh)
        sm.qk_rope(pos, q, qo, k, ko, table, inter, w[0][0], w[1][0], eps)
        check(qo, want[0], size[0])
        check(ko, want[1], size[1])
        q2, k2 = room(heads).copy_(q), room(kvh).copy_(k)
        sm.qk_rope(pos, q2, q2, None, None, table, inter, w[0][0], None, eps)
        sm.qk_rope(pos, None, None, k2, k2, table, inter, None, w[1][0], eps)
        assert torch.equal(q2, qo) and torch.equal(k2, ko)
    assert np.array_equal(both.double().cpu().numpy(), bf)


def test_in_place_among_others(sm, dev):
    """Queries and keys turned where they lie beside the values, which stay."""
    import torch
    rng = np.random.default_rng(5)
    heads, kvh, hd, n = 8, 2, 128, 300
    qkv, f = rows(dev, rng.standard_normal((n, heads + 2 * kvh, hd)), torch.float32)
    q, k, _ = qkv.split([heads, kvh, kvh], 1)
    table = sm.rope_table(400, 64, 1e4, dev)
    at = rng.integers(0, 400, n)
    sm.qk_rope(torch.tensor(at, dtype=torch.int32, device=dev), q, q, k, k, table)
    want = np.stack([paged4.turn(f[t, :heads + kvh], table.cpu().numpy()[at[t]]) for t in range(n)])
    got = qkv.double().cpu().numpy()
    assert np.all(np.abs(got[:, :heads + kvh] - want) <= 2.0 ** -24 * np.abs(want) * (1 + 1e-6) + 2.0 ** -49 * np.abs(want).max())
    assert np.array_equal(got[:, heads + kvh:], f[:, heads + kvh:])


def test_positions_outside_the_table(sm, dev):
    """Their tokens stay as they were."""
    import torch
    x = torch.randn(6, 2, 64, device=dev)
    table = sm.rope_table(10, 64, 1e4, dev)
    pos = torch.tensor([-1, 0, 9, 10, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32, device=dev)
    out = torch.full_like(x, 7.0)
    sm.qk_rope(pos, x, out, rope=table)
    assert torch.all(out[[0, 3, 4, 5]] == 7.0) and torch.all(out[[1, 2]] != 7.0)
    y = x.clone()
    sm.qk_rope(pos, y, y, rope=table)
    assert torch.equal(y[[0, 3, 4, 5]], x[[0, 3, 4, 5]]) and torch.equal(y[[1, 2]], out[[1, 2]])


def test_unusual_values(sm, dev):
    """Zeros, huge and tiny heads under a norm; what is not finite stays in its own head."""
    import torch
    w = torch.ones(64, device=dev)
    x = torch.randn(1, 6, 64, device=dev)
    x[0, 0] = 0
    x[0, 1] *= 1e36
    x[0, 2] *= 1e-36
    x[0, 3, 5] = float("nan")
    x[0, 4, 5] = float("inf")
    out = torch.empty_like(x)
    eps = float(np.float32(1e-12))
    sm.qk_rope(None, x, out, q_norm=w, eps=eps)
    f, got = x.double().cpu().numpy()[0], out.double().cpu().numpy()[0]
    want = paged4.turn(f, None, False, np.ones(64), eps)
    for h in (0, 1, 2, 5):
        assert np.all(np.abs(got[h] - want[h]) <= 2.0 ** -24 * np.abs(want[h]) * (1 + 1e-6) + 2.0 ** -149)
    assert np.isnan(got[3]).all() and np.isnan(got[4, 5]) and np.all(got[4, np.arange(64) != 5] == 0)


def test_unusual_bf16_values(sm, dev):
    """Heads of any magnitude that bf16 holds, under a norm, whose squares no f32 does."""
    import torch
    rng = np.random.default_rng(9)
    w, wf = rows(dev, 1 + 0.3 * rng.standard_normal(64), torch.float32)
    x, f = rows(dev, rng.standard_normal((1, 8, 64)) * np.array([1e38, 1e30, 1e10, 1.0, 1e-10, 1e-20, 1e-30, 0.0])[None, :, None], torch.bfloat16)
    table, out = sm.rope_table(5, 64, 1e4, dev), torch.empty_like(x)
    eps = float(np.float32(1e-38))
    pos = torch.tensor([3], dtype=torch.int32, device=dev)
    for inter in (False, True):
        sm.qk_rope(pos, x, out, rope=table, interleaved=inter, q_norm=w, eps=eps)
        want = paged4.turn(f[0], table.cpu().numpy()[3], inter, wf, eps)
        size = np.abs(paged4.turn(f[0], None, inter, wf, eps)).max(-1, keepdims=True)
        assert np.all(np.abs(out[0].double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) * (1 + 1e-6) + 2.0 ** -20 * size)


def test_streams_and_capture(sm, dev):
    """On a stream of the caller's, and recorded and replayed as positions move."""
    import torch
    table = torch.empty(300, 64, device=dev)
    make = sm.rope_table_op(table, 1e4, sm.RopeScaling("linear", 2.0))
    make()
    x, out, eager = torch.randn(40, 3, 64, device=dev), torch.empty(40, 3, 64, device=dev), torch.empty(40, 3, 64, device=dev)
    pos = torch.zeros(40, dtype=torch.int32, device=dev)
    op, other = sm.qk_rope_op(pos, x, out, rope=table), sm.qk_rope_op(pos, x, eager, rope=table)
    s = torch.cuda.Stream(device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        make()
        op()
    for step in range(6):
        pos.copy_(torch.arange(40, dtype=torch.int32) * 7 + step)
        x.normal_()
        table.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        other(s)
        s.synchronize()
        assert torch.equal(out, eager) and table[0, 0] == 1.0


def test_binding_refusals(sm, dev):
    import torch
    x, pos, table = torch.zeros(3, 2, 64, device=dev), torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(9, 64, device=dev)
    for call, text in (
            (lambda: sm.qk_rope(pos, x, None, rope=table), "do not agree"), (lambda: sm.qk_rope(pos, rope=table), "do not agree"),
            (lambda: sm.qk_rope(None, x, x, rope=table), "without positions"), (lambda: sm.qk_rope(pos[:2], x, x, rope=table), "shape"),
            (lambda: sm.qk_rope(pos.long(), x, x, rope=table), "type"), (lambda: sm.qk_rope(pos, x.half(), x.half(), rope=table), "type"),
            (lambda: sm.qk_rope(pos, x, x.bfloat16(), rope=table), "type"), (lambda: sm.qk_rope(pos, x, x[:2], rope=table), "2 rows"),
            (lambda: sm.qk_rope(pos, x, x[:, :1], rope=table), "shape"), (lambda: sm.qk_rope(pos, x.flatten(1), x, rope=table), "head_dim"),
            (lambda: sm.qk_rope(pos, x, x, rope=table.half()), "type"), (lambda: sm.qk_rope(pos, x, x, q_norm=x[0, 0, :60]), "shape"),
            (lambda: sm.qk_rope(pos, x, x, rope=torch.zeros(9, 66, device=dev)), "rope_dim 66"),
            (lambda: sm.qk_rope(pos, x, x, rope=table.cpu()), "on cpu"), (lambda: sm.qk_rope(pos, x, x, q_norm=x[0, 0], eps=0), "eps"),
            (lambda: sm.rope_table_op(table.half(), 1e4), "type"), (lambda: sm.rope_table_op(table, 1e4, "yarn"), "no RopeScaling"),
            (lambda: sm.rope_table_op(table, 1e4, sm.RopeScaling("yarn", 2))(), "original")):
        with pytest.raises(sm.SparkmvError, match=text):
            call()
