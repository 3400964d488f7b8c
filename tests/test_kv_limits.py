"""CPU tests of sizes next to the limits of the paged cache's calls: refused
before any launch."""
from test_kv import P, batch, cache, new, query, ref, refused


def test_page_counts_next_to_the_32_bit_limit(sm):
    """4095 sequences of 524408 pages count 128 less than 2^31; the shares of 512
    workgroups round up past it."""
    L = sm.lib()
    rows = dict(heads=4, ldq=256, ldo=256)
    c = cache(sm, kv_heads=1, max_pages=524408)
    assert 0 < 2 ** 31 - 4095 * (524408 + 8) <= 512
    refused(sm, L.sparkmv_kv_attend(ref(c), ref(batch(sm, nseq=4095, ntok=4095)), ref(query(sm, **rows)), None),
            "too many for one call")


def test_more_rows_than_a_launch_holds(sm):
    """2^31 - 1 rows: counts of pages and workgroups do not wrap."""
    L = sm.lib()
    most = 2 ** 31 - 1
    b = batch(sm, nseq=1, ntok=most, max_q=most, qstart=P)
    refused(sm, L.sparkmv_kv_append(ref(cache(sm)), ref(b), ref(new(sm)), None), "too much for one call")
    refused(sm, L.sparkmv_kv_read(ref(cache(sm)), 1, None, P, most, P, P, 1, None), "too much for one call")
    refused(sm, L.sparkmv_rope_table(P, most, 64, 1e4, None), "too large")
