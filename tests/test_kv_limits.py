"""CPU tests of sizes next to the limits of the paged cache's calls: refused
before any launch."""
from test_kv import batch, cache, query, ref, refused


def test_page_counts_next_to_the_32_bit_limit(sm):
    """4095 sequences of 524408 pages count 128 less than 2^31; the shares of 512
    workgroups round up past it."""
    L = sm.lib()
    rows = dict(heads=4, ldq=256, ldo=256)
    c = cache(sm, kv_heads=1, max_pages=524408)
    assert 0 < 2 ** 31 - 4095 * (524408 + 8) <= 512
    refused(sm, L.sparkmv_kv_attend(ref(c), ref(batch(sm, nseq=4095, ntok=4095)), ref(query(sm, **rows)), None),
            "too many for one call")
