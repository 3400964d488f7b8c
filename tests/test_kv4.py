"""CPU tests of the paged 4-bit cache and of head norms with the rotation: what the
entry points refuse, before any launch, and the oracle's own rules."""
import ctypes

import numpy as np
import pytest

import paged4
from test_kv import BATCHES, P, batch, query, ref, refused


def cache(sm, **kw):
    a = dict(kv_heads=2, head_dim=64, npages=4, nslots=2, max_pages=2, data=P, pages=P)
    a.update(kw)
    return sm.Kv4Cache(**a)


def turn(sm, **kw):
    a = dict(rope=P, rope_rows=128, rope_dim=64, interleaved=0, q_norm=P, k_norm=P, eps=1e-6)
    a.update(kw)
    return sm.HeadTurn(**a)


TURN = ("rope", "rope_rows", "rope_dim", "q_norm", "k_norm", "eps")


def new(sm, **kw):
    a = dict(q=P, k=P, v=P, ldq=256, ldk=128, ldv=128, x_dtype=1, heads=4, q_out=P, ldqo=256)
    a.update({k: v for k, v in kw.items() if k not in TURN})
    return sm.Kv4New(turn=turn(sm, **{k: v for k, v in kw.items() if k in TURN}), **a)


def qk(sm, **kw):
    a = dict(q=P, k=P, q_out=P, k_out=P, ldq=256, ldk=128, ldqo=256, ldko=128, x_dtype=1, heads=4, kv_heads=2, head_dim=64,
             ntok=3, pos=P)
    a.update(kw)
    return sm.QkRows(**a)


@pytest.mark.parametrize("bad,text", [
    ({"kv_heads": 0}, "kv_heads"), ({"kv_heads": 1025}, "kv_heads"), ({"head_dim": 96}, "head_dim 96"), ({"npages": 0}, "0 pages"),
    ({"nslots": 0}, "0 slots"), ({"max_pages": 0}, "slots of 0 pages"), ({"max_pages": 1 << 25}, "max_pages"),
    ({"data": None}, "null array"), ({"pages": None}, "null array"), ({"data": P + 8}, "not 16-byte aligned")])
def test_bad_caches(sm, bad, text):
    c, b, n, q = cache(sm, **bad), batch(sm), new(sm), query(sm)
    L = sm.lib()
    refused(sm, L.sparkmv_kv4_append(ref(c), ref(b), ref(n), None), text)
    refused(sm, L.sparkmv_kv4_attend(ref(c), ref(b), ref(q), None), text)
    refused(sm, L.sparkmv_kv4_read(ref(c), 1, None, P, 1, P, P, 1, None), text)
    assert L.sparkmv_kv4_attend_work(ref(c), ref(b), 4) == 0


@pytest.mark.parametrize("bad,text", BATCHES)
def test_bad_batches(sm, bad, text):
    c, b, n, q = cache(sm), batch(sm, **bad), new(sm), query(sm)
    L = sm.lib()
    refused(sm, L.sparkmv_kv4_append(ref(c), ref(b), ref(n), None), text)
    refused(sm, L.sparkmv_kv4_attend(ref(c), ref(b), ref(q), None), text)


@pytest.mark.parametrize("bad,text", [
    ({"x_dtype": 2}, "unknown type 2"), ({"heads": 0}, "do not agree"), ({"q": None}, "do not agree"),
    ({"q_out": None}, "do not agree"), ({"heads": -1}, "do not agree"), ({"rope_dim": 63}, "rope_dim 63"),
    ({"rope_dim": 66}, "rope_dim 66"), ({"rope_dim": -2}, "rope_dim -2"), ({"rope": None}, "rope table is null"),
    ({"rope_rows": 127}, "does not cover 128"), ({"k": None}, "keys is null"), ({"v": None}, "values is null"),
    ({"ldk": 127}, "holds no 128"), ({"ldv": 130}, "16-byte aligned"), ({"v": P + 4}, "16-byte aligned"),
    ({"ldqo": 260}, "two row strides"), ({"ldq": 255, "q": 2 * P}, "holds no 256"),
    ({"ldqo": 258, "q": 2 * P}, "16-byte aligned"), ({"q_out": P + 2}, "16-byte aligned"), ({"eps": 0.0}, "eps"),
    ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"eps": float("inf")}, "eps"), ({"heads": 65537}, "65537")])
def test_bad_new_rows(sm, bad, text):
    refused(sm, sm.lib().sparkmv_kv4_append(ref(cache(sm)), ref(batch(sm)), ref(new(sm, **bad)), None), text)


@pytest.mark.parametrize("bad,text", [
    ({"q_dtype": 2}, "unknown type 2"), ({"out_dtype": -1}, "unknown type -1"), ({"heads": 0}, "query heads"),
    ({"heads": 3}, "query heads"), ({"heads": 34, "ldq": 4096, "ldo": 4096}, "query heads"), ({"window": -1}, "window"),
    ({"scale": float("nan")}, "not finite"), ({"scale": float("inf")}, "not finite"), ({"q": None}, "queries is null"),
    ({"out": None}, "output is null"), ({"ldq": 255}, "holds no 256"), ({"ldo": 258}, "16-byte aligned"),
    ({"out": P + 8}, "16-byte aligned"), ({"gate": P, "ldg": 3}, "holds no 4 heads"), ({"work": None}, "workspace"),
    ({"work": P + 16}, "workspace"), ({"work_bytes": 16}, "workspace")])
def test_bad_queries(sm, bad, text):
    refused(sm, sm.lib().sparkmv_kv4_attend(ref(cache(sm)), ref(batch(sm, max_len=4000)), ref(query(sm, **bad)), None), text)


def test_sizes_too_large_for_one_call(sm):
    L = sm.lib()
    c = cache(sm, max_pages=1 << 24, kv_heads=64)
    q = query(sm, heads=64, ldq=4096, ldo=4096)
    refused(sm, L.sparkmv_kv4_attend(ref(c), ref(batch(sm)), ref(q), None), "too many for one call")
    big = batch(sm, nseq=1, ntok=0x7fffffff, qstart=P, max_q=0x7fffffff)
    refused(sm, L.sparkmv_kv4_append(ref(cache(sm)), ref(big), ref(new(sm, ldq=256)), None), "too much for one call")
    refused(sm, L.sparkmv_kv4_read(ref(cache(sm)), 4096, None, P, 0x7fffffff, P, P, 1, None), "too much for one call")
    refused(sm, L.sparkmv_kv4_read(ref(cache(sm)), 4097, None, P, 1, P, P, 1, None), "4097 sequences")


def test_calls_of_nothing(sm):
    L = sm.lib()
    assert L.sparkmv_kv4_append(ref(cache(sm)), ref(batch(sm, nseq=0, ntok=0, pos=None)), ref(new(sm)), None) == 0
    assert L.sparkmv_kv4_attend(ref(cache(sm)), ref(batch(sm, nseq=0, ntok=0, pos=None)), ref(query(sm)), None) == 0
    assert L.sparkmv_kv4_read(ref(cache(sm)), 0, None, None, 5, P, P, 1, None) == 0
    assert L.sparkmv_qk_rope(ref(qk(sm, ntok=0)), ref(turn(sm)), None) == 0
    assert L.sparkmv_kv4_bytes(2, 128, 3) == 3 * 2 * 68 * 128 and L.sparkmv_kv4_bytes(0, 128, 3) == 0


@pytest.mark.parametrize("bad,text", [
    ({"x_dtype": 5}, "unknown type 5"), ({"head_dim": 66}, "head_dim 66"), ({"head_dim": 260}, "head_dim 260"),
    ({"head_dim": 0}, "head_dim 0"), ({"ntok": -1}, "-1 tokens"), ({"heads": -1}, "outside"), ({"kv_heads": 70000}, "outside"),
    ({"q": None}, "do not agree"), ({"k_out": None}, "do not agree"), ({"heads": 0}, "do not agree"), ({"pos": None}, "no positions"),
    ({"ldq": 255, "q_out": 2 * P}, "holds no 256"), ({"ldk": 130, "k_out": 2 * P}, "16-byte aligned"), ({"k": P + 8}, "16-byte aligned"),
    ({"ldqo": 512}, "two row strides"), ({"ldk": 512}, "two row strides"), ({"ntok": 0x7fffffff}, "too much")])
def test_bad_qk_rows(sm, bad, text):
    refused(sm, sm.lib().sparkmv_qk_rope(ref(qk(sm, **bad)), ref(turn(sm)), None), text)


@pytest.mark.parametrize("bad,text", [({"rope_dim": 66}, "rope_dim 66"), ({"rope_dim": 7}, "rope_dim 7"), ({"rope": None}, "table is null"),
                                      ({"rope_rows": 0}, "does not cover"), ({"eps": 0.0}, "eps")])
def test_bad_turns(sm, bad, text):
    refused(sm, sm.lib().sparkmv_qk_rope(ref(qk(sm)), ref(turn(sm, **bad)), None), text)


def scaling(sm, **kw):
    a = dict(kind=3, factor=4.0, original=4096.0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0, attention=0.0)
    a.update(kw)
    return sm.RopeScalingC(**a)


@pytest.mark.parametrize("bad,text", [
    ({"kind": 5}, "unknown rope scaling"), ({"kind": -1}, "unknown rope scaling"), ({"factor": 0.5}, "1 or more"),
    ({"factor": float("nan")}, "1 or more"), ({"original": 0.0}, "original context"), ({"kind": 4, "original": -1.0}, "original context"),
    ({"attention": -1.0}, "attention"), ({"beta_slow": 0.0}, "beta_slow"), ({"beta_fast": 0.5}, "beta_slow"),
    ({"kind": 4, "low": 4.0}, "low < high"), ({"kind": 4, "low": 0.0}, "low < high")])
def test_bad_scalings(sm, bad, text):
    refused(sm, sm.lib().sparkmv_rope_table_scaled(P, 10, 64, 1e4, ref(scaling(sm, **bad)), None), text)


@pytest.mark.parametrize("args,text", [
    ((None, 10, 64, 1e4), "null"), ((P, 0, 64, 1e4), "0 rows"), ((P, 10, 63, 1e4), "63 values"), ((P, 10, 258, 1e4), "258 values"),
    ((P, 10, 64, 0.0), "theta"), ((P, 10, 64, float("nan")), "theta"), ((P, 10, 64, 1.0), "theta above 1")])
def test_bad_tables(sm, args, text):
    refused(sm, sm.lib().sparkmv_rope_table_scaled(*args, ref(scaling(sm)), None), text)


def test_scaling_of_the_binding(sm):
    for bad in (dict(kind="other"), dict(kind="yarn", attention=0.0), dict(kind="yarn", attention=-2.0)):
        with pytest.raises(sm.SparkmvError):
            sm.RopeScaling(**bad)
    c = sm.RopeScaling("bands", 8, 8192, low=2).c
    assert (c.kind, c.factor, c.original, c.low, c.high, c.attention) == (4, 8.0, 8192.0, 2.0, 4.0, 0.0)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_page_holds_every_element_once(hd):
    off = paged4.offsets(hd)
    codes = [off[w][:, ::2] for w in (0, 2)]
    scales = [off[w][:, ::32] for w in (1, 3)]
    every = np.concatenate([x.ravel() for x in codes + scales])
    assert sorted(every) == list(range(68 * hd))
    for w in (0, 2):
        assert np.array_equal(off[w][:, ::2], off[w][:, 1::2])
        assert np.array_equal(off[w + 1], np.repeat(off[w + 1][:, ::32], 32, 1))


def test_held_values():
    """The nearest of the sixteen values under the smallest scale that covers 7 times
    it, from every candidate, ties to the even code."""
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((200, 32)) * np.exp(rng.standard_normal((200, 1)) * 4)).astype(np.float32).astype(np.float64)
    x[:40] = rng.integers(-28, 29, (40, 32)) / 4.0        # halves and quarters: ties
    x[40] = 0.0
    code, byte = paged4.held(x)
    for r in range(len(x)):
        e = int(byte[r, 0]) - 127
        most = np.abs(x[r]).max()
        assert e == -120 if most == 0 else (most <= 7 * 2.0 ** e and most > 7 * 2.0 ** (e - 1))
        for v, c in zip(x[r], code[r]):
            away = np.abs(paged4.LEVELS * 2.0 ** e - abs(v))
            best = np.flatnonzero(away == away.min())
            assert (c & 7) == (best[0] if len(best) == 1 else best[best % 2 == 0][0])
            assert (c > 7) == np.signbit(v)
    assert paged4.held(np.full(32, np.inf))[1] == 255 and paged4.held(np.full(32, 3e38))[1] == 252
