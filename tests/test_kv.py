"""CPU tests of the paged 8-bit cache and the log probabilities: what the
entry points refuse, before any launch, and the oracle's own rules."""
import ctypes

import numpy as np
import pytest

import paged

P = 1 << 20      # a pointer that no refused call follows


def cache(sm, **kw):
    a = dict(kv_heads=2, head_dim=64, npages=4, nslots=2, max_pages=2, k=P, v=P, k_scale=P, v_scale=P, pages=P)
    a.update(kw)
    return sm.KvCache(**a)


def batch(sm, **kw):
    a = dict(nseq=2, ntok=2, max_q=1, max_len=10, pos=P)
    a.update(kw)
    return sm.KvBatch(**a)


def new(sm, **kw):
    a = dict(q=P, k=P, v=P, ldq=256, ldk=128, ldv=128, x_dtype=1, heads=4, rope=P, rope_rows=128, rope_dim=64, q_out=P,
             ldqo=256)
    a.update(kw)
    return sm.KvNew(**a)


def query(sm, **kw):
    a = dict(q=P, ldq=256, q_dtype=1, heads=4, scale=0.1, window=0, out=P, ldo=256, out_dtype=1, work=P, work_bytes=1 << 30)
    a.update(kw)
    return sm.KvQuery(**a)


def ref(x):
    return ctypes.byref(x)


def refused(sm, rc, text):
    assert rc == -1
    assert text in sm.last_error(), sm.last_error()


CACHES = [({"kv_heads": 0}, "kv_heads"), ({"head_dim": 96}, "head_dim 96"), ({"npages": 0}, "0 pages"),
          ({"nslots": 0}, "0 slots"), ({"max_pages": 0}, "slots of 0 pages"), ({"max_pages": 1 << 25}, "max_pages"),
          ({"k": None}, "null array"), ({"v_scale": None}, "null array"), ({"pages": None}, "null array"),
          ({"v": P + 8}, "not 16-byte aligned")]
BATCHES = [({"nseq": -1}, "sequences"), ({"nseq": 4097, "ntok": 4097}, "4097 sequences"), ({"ntok": -1}, "-1 tokens"),
           ({"pos": None}, "no positions"), ({"max_q": 0}, "max_q"), ({"ntok": 1}, "one token each")]


@pytest.mark.parametrize("bad,text", CACHES)
def test_bad_caches(sm, bad, text):
    c, b, n, q = cache(sm, **bad), batch(sm), new(sm), query(sm)
    L = sm.lib()
    refused(sm, L.sparkmv_kv_append(ref(c), ref(b), ref(n), None), text)
    refused(sm, L.sparkmv_kv_attend(ref(c), ref(b), ref(q), None), text)
    refused(sm, L.sparkmv_kv_read(ref(c), 1, None, P, 1, P, P, 1, None), text)


@pytest.mark.parametrize("bad,text", BATCHES)
def test_bad_batches(sm, bad, text):
    c, b, n, q = cache(sm), batch(sm, **bad), new(sm), query(sm)
    L = sm.lib()
    refused(sm, L.sparkmv_kv_append(ref(c), ref(b), ref(n), None), text)
    refused(sm, L.sparkmv_kv_attend(ref(c), ref(b), ref(q), None), text)


@pytest.mark.parametrize("bad,text", [
    ({"x_dtype": 2}, "unknown type 2"), ({"heads": 0}, "do not agree"), ({"q": None}, "do not agree"),
    ({"q_out": None}, "do not agree"), ({"heads": -1}, "do not agree"), ({"rope_dim": 63}, "rope_dim 63"),
    ({"rope_dim": 66}, "rope_dim 66"), ({"rope_dim": -2}, "rope_dim -2"), ({"rope": None}, "rope table is null"),
    ({"rope_rows": 127}, "does not cover 128"), ({"k": None}, "keys is null"), ({"v": None}, "values is null"),
    ({"ldk": 127}, "holds no 128"), ({"ldv": 130}, "16-byte aligned"), ({"v": P + 4}, "16-byte aligned"),
    ({"ldqo": 260}, "two row strides"), ({"ldq": 255, "q": 2 * P}, "holds no 256"), ({"ldqo": 258, "q": 2 * P}, "16-byte aligned"), ({"q_out": P + 2}, "16-byte aligned")])
def test_bad_new_rows(sm, bad, text):
    refused(sm, sm.lib().sparkmv_kv_append(ref(cache(sm)), ref(batch(sm)), ref(new(sm, **bad)), None), text)


@pytest.mark.parametrize("bad,text", [
    ({"q_dtype": 3}, "unknown type 3"), ({"out_dtype": -1}, "unknown type -1"), ({"heads": 3}, "3 query heads"),
    ({"heads": 0}, "0 query heads"), ({"heads": 34}, "34 query heads"), ({"window": -1}, "window -1"),
    ({"scale": float("nan")}, "not finite"), ({"scale": float("inf")}, "not finite"), ({"q": None}, "queries is null"),
    ({"out": None}, "output is null"), ({"ldq": 252}, "holds no 256"), ({"ldo": 257}, "16-byte aligned"),
    ({"out": P + 8}, "16-byte aligned"), ({"gate": P, "ldg": 3}, "gate")])
def test_bad_queries(sm, bad, text):
    refused(sm, sm.lib().sparkmv_kv_attend(ref(cache(sm)), ref(batch(sm)), ref(query(sm, **bad)), None), text)


def test_workspace(sm):
    L = sm.lib()
    c = cache(sm)
    for b, heads in ((batch(sm), 4), (batch(sm, nseq=1, ntok=300, qstart=P, max_q=300, max_len=128), 4), (batch(sm), 32)):
        need = L.sparkmv_kv_attend_work(ref(c), ref(b), heads)
        rows = dict(heads=heads, ldq=64 * heads, ldo=64 * heads)
        if need:
            for w in (dict(work=None, work_bytes=need), dict(work=P, work_bytes=need - 1), dict(work=P + 128, work_bytes=need)):
                refused(sm, L.sparkmv_kv_attend(ref(c), ref(b), ref(query(sm, **rows, **w)), None), "workspace")
    assert L.sparkmv_kv_attend_work(ref(c), ref(batch(sm)), 4) > 0
    # the count of pages has to fit a 32-bit number
    big = cache(sm, kv_heads=64, max_pages=1 << 20)
    refused(sm, L.sparkmv_kv_attend(ref(big), ref(batch(sm, nseq=64, ntok=64)), ref(query(sm, heads=64, ldq=4096, ldo=4096)), None),
            "too many for one call")


def test_more_tiles_than_a_launch_holds(sm):
    """2^30 tokens of 64 x 16 heads: 2^28 tiles of 64 columns, each on 64 kv heads."""
    rows = query(sm, heads=1024, ldq=1 << 16, ldo=1 << 16)
    refused(sm, sm.lib().sparkmv_kv_attend(ref(cache(sm, kv_heads=64)), ref(batch(sm, ntok=1 << 30, qstart=P, max_q=64)), ref(rows), None),
            "too much for one call")


def test_null_structures_and_empty_calls(sm):
    L = sm.lib()
    c, b, n, q = cache(sm), batch(sm), new(sm), query(sm)
    refused(sm, L.sparkmv_kv_append(None, ref(b), ref(n), None), "cache is null")
    refused(sm, L.sparkmv_kv_append(ref(c), None, ref(n), None), "batch is null")
    refused(sm, L.sparkmv_kv_append(ref(c), ref(b), None, None), "rows are null")
    refused(sm, L.sparkmv_kv_attend(ref(c), ref(b), None, None), "query is null")
    # nothing to do is no error and launches nothing (there is no GPU here)
    for e in (batch(sm, nseq=0, ntok=0, pos=None), batch(sm, nseq=1, ntok=0, qstart=P)):
        assert L.sparkmv_kv_append(ref(c), ref(e), ref(n), None) == 0
        assert L.sparkmv_kv_attend(ref(c), ref(e), ref(q), None) == 0
    assert L.sparkmv_kv_read(ref(c), 0, None, None, 5, P, P, 1, None) == 0
    assert L.sparkmv_kv_read(ref(c), 3, None, P, 0, P, P, 1, None) == 0
    refused(sm, L.sparkmv_kv_read(ref(c), 3, None, None, 1, P, P, 1, None), "no positions")
    refused(sm, L.sparkmv_kv_read(ref(c), 5000, None, P, 1, P, P, 1, None), "5000 sequences")
    refused(sm, L.sparkmv_kv_read(ref(c), 3, None, P, -1, P, P, 1, None), "-1 positions")
    refused(sm, L.sparkmv_kv_read(ref(c), 3, None, P, 1, P + 4, P, 1, None), "16-byte aligned")
    refused(sm, L.sparkmv_kv_read(ref(c), 3, None, P, 1, P, P, 7, None), "unknown type 7")


@pytest.mark.parametrize("args,text", [
    ((None, 4, 64, 1e4), "null"), ((P, 0, 64, 1e4), "0 rows"), ((P, 4, 63, 1e4), "63 values"), ((P, 4, 0, 1e4), "0 values"),
    ((P, 4, 64, 0.0), "theta"), ((P, 4, 64, float("nan")), "theta")])
def test_bad_rope_tables(sm, args, text):
    refused(sm, sm.lib().sparkmv_rope_table(*args, None), text)


@pytest.mark.parametrize("bad,text", [
    ({"x_dtype": 9}, "unknown type 9"), ({"rows": -1}, "-1 rows"), ({"n": 0}, "0 logits"), ({"n": 524289, "ld": 524289}, "above 524288"),
    ({"rows": 65536}, "above 65535"), ({"work": None}, "workspace"), ({"work_bytes": 63}, "workspace"), ({"work": P + 16}, "workspace"),
     ({"k": 33}, "33 alternatives"),
    ({"k": -1}, "-1 alternatives"), ({"logits": None}, "logits are null"), ({"ld": 9}, "holds no 10"),
    ({"tokens": None}, "do not agree"), ({"logprob": None}, "do not agree"), ({"top_id": None}, "without room"),
    ({"top_logprob": None}, "without room")])
def test_bad_logprobs(sm, bad, text):
    a = dict(logits=P, x_dtype=1, rows=2, n=10, ld=10, tokens=P, k=3, logprob=P, entropy=P, top_id=P, top_logprob=P, work=P,
             work_bytes=1 << 30)
    a.update(bad)
    refused(sm, sm.lib().sparkmv_logprobs(*a.values(), None), text)


def test_no_rows_of_logits(sm):
    assert sm.lib().sparkmv_logprobs(None, 1, 0, 10, 10, None, 0, None, None, None, None, None, 0, None) == 0


def test_layout_is_a_permutation():
    for hd in (64, 128, 256):
        for off in paged.offsets(hd):
            assert np.array_equal(np.sort(off.ravel()), np.arange(64 * hd))


def test_oracle_rounding_bound():
    """Appended one at a time with magnitudes that keep growing, every value
    stays within 3 steps of the page's last scale: each growth but the one
    that fills the page multiplies the scale by 1.25 at least, so the half steps
    of all roundings add up to at most s / 2 / (1 - 1 / 1.25) + s / 2."""
    rng = np.random.default_rng(3)
    hd = 64
    c = {"k": np.zeros((1, 1, 64 * hd), np.int8), "v": np.zeros((1, 1, 64 * hd), np.int8),
         "k_scale": np.zeros((1, 1), np.float32), "v_scale": np.zeros((1, 1), np.float32), "pages": np.zeros((1, 1), np.int32)}
    x = (rng.standard_normal((64, 1, hd)) * (1.3 ** np.arange(64))[:, None, None]).astype(np.float32).astype(np.float64)
    for p in range(64):
        paged.append(c, None, x[p:p + 1], x[p:p + 1], None, [p])
    for p in range(64):
        k, v = paged.read(c, 0, p, hd)
        assert np.abs(k - x[p]).max() <= 3 * c["k_scale"][0, 0] * (1 + 1e-6)
        assert np.array_equal(k, v)
