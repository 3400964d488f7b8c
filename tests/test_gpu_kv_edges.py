"""GPU tests of calls over the paged cache at the edges of what their arguments
allow: row starts that fall or wrap, bounds far above the call's rows, the
largest window, workspaces on other streams."""
import numpy as np
import pytest

from test_gpu_kv import Case, check_attention, rows, types
import paged

pytestmark = pytest.mark.gpu

LOW = -(1 << 31)


@pytest.mark.parametrize("group,max_q", [(1, 4), (4, None), (4, 2)])
def test_row_starts_that_fall(sm, dev, group, max_q):
    """A sequence whose rows end before they begin is left out, however far
    before: its rows and pages stay as they were, the others are served."""
    import torch
    kvh, hd, ntok = 2, 64, 14
    qstart = [0, 4, LOW, 4, 10, LOW + 3, 10, 12, 5]
    pos = [60, 5, 6, 100, 7, 8, 62, 9]
    c = Case(sm, dev, kvh, hd, len(pos), 2, 91)
    q, qf = rows(dev, c.rng.standard_normal((ntok, kvh * group, hd)), torch.float32)
    k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.float32)
    b = c.batch(pos, ntok, qstart, max_q=max_q)
    turned, out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    table = sm.rope_table(128, 64, 1e4, dev)
    c.kv.append(b, q, k, k, table, turned)
    most = 1 << 30 if max_q is None else max_q
    want = paged.append(c.host, qf, kf, kf, table.cpu().numpy(), pos, qstart, None, most)
    c.same()
    got = turned.double().cpu().numpy()
    assert np.array_equal(got, np.where(np.isnan(want), 7.0, want).astype(np.float32).astype(np.float64))
    c.kv.attend(b, q, out)
    check_attention(c, q, qf, out, 0.125, 0, None, pos, qstart, None, most, f"group {group} max_q {max_q}")
