"""CPU and GPU tests of calls over the paged caches, and of head norms with the
rotation, that have no rows."""
import pytest

import test_kv
from test_kv import P, batch, query, ref, refused
from test_kv4 import cache, new, qk, turn


def test_calls_of_no_rows(sm):
    """An array of no rows may be null, heads or not: a tensor of none has no address."""
    L = sm.lib()
    none = dict(q=None, k=None, v=None, q_out=None)
    for b in (batch(sm, nseq=0, ntok=0, pos=None), batch(sm, nseq=2, ntok=0, qstart=P)):
        assert L.sparkmv_kv4_append(ref(cache(sm)), ref(b), ref(new(sm, **none)), None) == 0, sm.last_error()
        assert L.sparkmv_kv_append(ref(test_kv.cache(sm)), ref(b), ref(test_kv.new(sm, **none)), None) == 0, sm.last_error()
        assert L.sparkmv_kv4_attend(ref(cache(sm)), ref(b), ref(query(sm, q=None, out=None, work=None)), None) == 0, sm.last_error()
    assert L.sparkmv_qk_rope(ref(qk(sm, q=None, k=None, q_out=None, k_out=None, ntok=0)), ref(turn(sm)), None) == 0, sm.last_error()
    refused(sm, L.sparkmv_qk_rope(ref(qk(sm, heads=-1, ntok=0)), ref(turn(sm)), None), "outside")
    refused(sm, L.sparkmv_kv4_append(ref(cache(sm)), ref(batch(sm, nseq=0, ntok=0, pos=None)), ref(new(sm, heads=-1)), None), "do not agree")


@pytest.mark.gpu
def test_calls_of_empty_tensors(sm, dev):
    import torch
    q, k, w = (torch.empty(0, h, 64, device=dev) for h in (4, 2, 1))
    none, w = torch.empty(0, dtype=torch.int32, device=dev), torch.ones(64, device=dev)
    table = sm.rope_table(128, 64, 1e4, dev)
    sm.qk_rope(none, q, q, k, k, table, False, w, w)
    starts = torch.zeros(3, dtype=torch.int32, device=dev)
    for kv in (sm.PagedKV(2, 64, 4, 2, 2, device=dev), sm.PagedKV4(2, 64, 4, 2, 2, device=dev)):
        for b in (sm.KVBatch(none), sm.KVBatch(starts[:2], 0, starts)):
            kv.append(b, q, k, k, table, q)
            kv.attend(b, q, torch.empty_like(q))
        kv.read(none, torch.empty(0, 5, 2, 64, device=dev))
    torch.cuda.synchronize()
